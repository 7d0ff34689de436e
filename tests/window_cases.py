"""Seeded inputs, references and tolerances of the windowed-attention and 4-bit-cache tests."""

from __future__ import annotations

import numpy as np
import torch

from oracle import window as ow
from pagelora_amd.window_attention import WindowAttention

BF16, F16 = torch.bfloat16, torch.float16


def case(lens, hq, hkv, head_dim, page_size, dtype, device, *, bits=16, new=None, window=0, sinks=0, seed=0, q_scale=1.0,
         poison=True, extra=3):
    """Requests of ``lens`` tokens, the last ``new`` of each with queries (default: one, none of an empty request's).
    With ``poison`` all that no query sees is NaN: the tails of pages, unused pages, what a window leaves out."""
    gen = torch.Generator().manual_seed(seed)
    prompts, new = new is not None, [1] * len(lens) if new is None else new
    pages = [-(-n // page_size) for n in lens]
    pool = sum(pages) + extra
    ids = torch.randperm(pool, generator=gen)[: sum(pages)].int()
    indptr = torch.tensor([0, *np.cumsum(pages)], dtype=torch.int32)
    last = torch.tensor([n - (p - 1) * page_size if p else 0 for n, p in zip(lens, pages)], dtype=torch.int32)
    cache = torch.randn((pool, 2, page_size, hkv, head_dim), generator=gen).to(dtype)
    q = (torch.randn((sum(new), hq, head_dim), generator=gen) * q_scale).to(dtype)
    if poison:
        seen = torch.zeros((pool, page_size), dtype=torch.bool)
        for r, n in enumerate(lens):
            for i in range(min(new[r], n)):
                at = torch.from_numpy(ow.sees(n - min(new[r], n) + i, n, window, sinks))
                seen[ids[indptr[r] + at // page_size].long(), at % page_size] = True
        cache[~seen[:, None].expand(-1, 2, -1)] = float("nan")
    out = {"q": q.to(device), "q_host": q, "indptr": indptr, "indices": ids, "last": last, "lens": list(lens), "new": list(new),
           "qo_indptr": torch.tensor([0, *np.cumsum(new)], dtype=torch.int32), "heads": (hq, hkv), "head_dim": head_dim,
           "page_size": page_size, "dtype": dtype, "bits": bits, "window": window, "sinks": sinks, "device": device, "prefill": prompts}
    set_cache(out, cache)
    return out


def set_cache(c, cache):
    """Makes ``cache`` (16 bits, host) the case's, in its bits."""
    if c["bits"] == 16:
        c["cache_host"] = cache.double().numpy()
        c["cache"] = cache.to(c["device"])
        return
    x = cache.double().numpy()
    (kc, ks), (vc, vs) = ow.quantize(x[:, 0]), ow.quantize(x[:, 1])
    c["cache_host"] = np.stack([ow.values(kc, ks), ow.values(vc, vs)], 1)
    c["cache"] = torch.from_numpy(ow.pack_pages(kc, ks, vc, vs)).to(c["device"])


def tables(c, device=None):
    t = {"paged_kv_indptr": c["indptr"], "paged_kv_indices": c["indices"], "paged_kv_last_page_len": c["last"]}
    return t if device is None else {k: v.to(device) for k, v in t.items()}


def attention(c):
    return WindowAttention(device=c["device"], num_qo_heads=c["heads"][0], num_kv_heads=c["heads"][1], head_dim=c["head_dim"],
                           page_size=c["page_size"], window=c["window"], sinks=c["sinks"])


def reference(c, sm_scale=None, window=None):
    """(o, lse, how far an output may be off) in 64 bits, packed by queries.

    Half a step of the output's type (eps / 2 of the value; below the normal range of fp16, 2^-25), and of the weighted
    mean of |v|: twice (numerator and denominator) what the weights are off by: a score's D products and their sum in
    32 bits, 2^-24 D of sum |q||k| s; its exponent, x up to twice the largest score times log2 e held to 2^-24, and 2^-22
    of the conversion; the two planes (bf16 2^-7 left, of which 2^-8: 2^-15; fp16 2^-11 twice: 2^-22; prompts of bf16 over 4
    bits have one fp16 plane: 2^-11); the sum over the tokens in 32 bits, 2^-24 each.  And of the largest |v|, per token, what falls below a plane's range: in bf16 weights
    are held with the row's largest at 2^-32 or more, and the second plane ends at the smallest normal number, 2^-126: 2^-94 of
    the largest; in fp16 with the largest at 2^11 or more, and half of 2^-24 is lost: 2^-36.
    """
    (hq, hkv), d, outs = c["heads"], c["head_dim"], []
    sm_scale = d ** -0.5 if sm_scale is None else sm_scale
    ptr, qo = c["indptr"].tolist(), c["qo_indptr"].tolist()
    for r, n in enumerate(c["lens"]):
        kv = c["cache_host"][c["indices"][ptr[r]: ptr[r + 1]].long().numpy()]
        k, v = (kv[:, i].reshape(-1, hkv, d)[:n] for i in (0, 1))
        q = c["q_host"][qo[r]: qo[r + 1]].double().numpy()
        if n == 0:  # rows without tokens
            outs.append((np.zeros(q.shape), np.full(q.shape[:2], -np.inf), np.zeros(q.shape), np.zeros(q.shape[:2])))
        else:
            outs.append(ow.attend(q, k, v, c["window"] if window is None else window, c["sinks"], sm_scale))
    o, lse, spread, reach = (np.concatenate(x) for x in zip(*outs))
    most = np.nan_to_num(np.abs(c["cache_host"]), nan=0.0, posinf=0.0).max(initial=0.0)
    eps = torch.finfo(c["dtype"]).eps
    # past the type's largest by half a step, an output rounds to an infinity
    with np.errstate(invalid="ignore"):
        o = np.where(np.abs(o) >= torch.finfo(c["dtype"]).max * (1 + eps / 4), np.copysign(np.inf, o), o)
    half = c["dtype"] == F16 if c["bits"] == 16 else c.get("prefill", False)  # probabilities in fp16
    planes = 2.0 ** -15 if not half else 2.0 ** -22 if c["dtype"] == F16 else 2.0 ** -11
    weight = 2 * (2.0 ** -24 * d * reach + 2.0 ** -24 * 2 * 1.4427 * reach + 2.0 ** -22) + planes + 2.0 ** -24 * max(c["lens"], default=0)
    with np.errstate(invalid="ignore"):
        tol = eps / 2 * np.abs(o) + weight[..., None] * spread * (1 + eps) + (2.0 ** -25 if c["dtype"] == F16 else 0)
        tol += (2.0 ** -36 if half else 2.0 ** -94) * max(c["lens"], default=0) * most
    return o, lse, tol, weight


def check(c, got, lse=None, sm_scale=None, window=None):
    """``got`` (and ``lse``) against :func:`reference`: infinities and NaN where it has them, the rest within its bounds."""
    o, want_lse, tol, weight = reference(c, sm_scale, window)
    got = got.double().cpu().numpy()
    assert got.shape == o.shape
    assert (np.isnan(got) == np.isnan(o)).all(), "NaN in other places"
    inf = np.isinf(o)
    assert (np.isinf(got) == inf).all() and (got[inf] == o[inf]).all(), "infinities in other places"
    live = np.isfinite(o)
    off = np.abs(got - o)[live] - tol[live]
    assert off.size == 0 or off.max() <= 0, f"off by {off.max()} more than it may be"
    if lse is not None:
        lse = lse.double().cpu().numpy()
        empty = want_lse == -np.inf
        assert (lse[empty] == -np.inf).all()
        # the weights' bound, and the two roundings of a number of this size
        bound = weight + 2.0 ** -22 * (1 + np.abs(np.where(empty, 0, want_lse)))
        assert (np.abs(lse - want_lse)[~empty] <= bound[~empty]).all()


def decode(c, **kw):
    attn = attention(c)
    attn.plan_decode(**tables(c, kw.get("tables_on")))
    out = torch.empty_like(c["q"])
    lse = torch.empty(c["q"].shape[:2], dtype=torch.float32, device=c["q"].device)
    attn.run_decode_into(c["q"], c["cache"], out, lse)
    torch.cuda.synchronize()
    return out, lse


def prefill(c):
    attn = attention(c)
    attn.plan_prefill(qo_indptr=c["qo_indptr"], **tables(c))
    out = attn.run_prefill(c["q"], c["cache"])
    torch.cuda.synchronize()
    return out
