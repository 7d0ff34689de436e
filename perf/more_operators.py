"""The operators of long contexts held in little memory, as timed cases.

A serving engine keeps long sequences either in 4 bits per value, or by reading
only the last tokens of them and a few first ones (sinks), or both:

* ``kv4``: tokens quantized into a paged 4-bit cache and read back from it,
* ``decode4`` / ``decode``: one layer's attention of single tokens over a 4-bit
  and a 16-bit paged cache, with or without a window,
* ``prefill4`` / ``prefill``: the same of prompts, whole or behind what the
  cache holds already.

A query at position p sees position t <= p where t > p - window (window 0: no
bound) or t < sinks.

The 4-bit cache holds each 32 values along head_dim as codes e2m1 (sign, two
bits of exponent, one of mantissa: 0, 0.5, 1, 1.5, 2, 3, 4, 6) and one byte s:
a power of two 2^(s - 127), the least at which the largest magnitude is at most
6; 255 marks a group that held a NaN or an infinity.  A layer is uint8
[pages, 2, kv heads, page * (dim / 2 + dim / 32)], K at 0 and V at 1 of dim 2:
codes, then scales.  K token t's codes are bytes t * dim / 2 on, its scales
t * dim / 32 on.  V goes by four tokens: codes [t / 4][d / 8][t % 4][4 bytes],
scales [t / 4][d / 32][t % 4].  The lower nibble is the lower dim.

``own`` False computes them from elementary torch operations, True through the
package's entry points.
"""

from __future__ import annotations

import math

import torch

own = False

# (q heads, kv heads): the GQA ratios and the MHA that the other timed cases have
HEADS = {"gqa4": (32, 8), "mha": (32, 32), "gqa7": (28, 4)}
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
GROUP = 32
LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _attn(name, kind, heads, requests, new, lens, dtype, window=0, sinks=0, page=16, dim=128):
    """``new``, ``lens``: (fewest, most) queries of a request, and tokens before them."""
    return {"name": name, "kind": kind, "heads": heads, "requests": requests, "min_new": new[0], "max_new": new[1],
            "min_len": lens[0], "max_len": lens[1], "window": window, "sinks": sinks, "page": page, "dim": dim,
            "dtype": dtype}


def listed():
    return [
        # one decode step's new tokens of a full batch; a long prompt's tokens without GQA
        {"name": "kv4_64_gqa4_bf16", "kind": "kv4", "heads": "gqa4", "tokens": 64, "page": 16, "dim": 128, "dtype": "bf16"},
        {"name": "kv4_8192_mha_fp16", "kind": "kv4", "heads": "mha", "tokens": 8192, "page": 16, "dim": 128, "dtype": "fp16"},
        # one chat: latency and launches
        _attn("decode4_1x2048_gqa4_bf16", "decode4", "gqa4", 1, (1, 1), (2047, 2047), "bf16"),
        # one very long document: the work split over the kv axis
        _attn("decode4_1x131072_gqa4_bf16", "decode4", "gqa4", 1, (1, 1), (131071, 131071), "bf16"),
        # a medium batch of ragged chats, some longer than the window; a GQA ratio that is no power of two
        _attn("decode4_23_w1000_gqa7_fp16", "decode4", "gqa7", 23, (1, 1), (33, 4099), "fp16", window=1000, sinks=4),
        # a full batch of long chats, the most cache
        _attn("decode4_64x16384_gqa4_bf16", "decode4", "gqa4", 64, (1, 1), (4095, 16383), "bf16"),
        # a full batch that reads the last 1024 tokens and 4 sinks of a 16-bit cache
        _attn("decode_64x8192_w1024_gqa4_bf16", "decode", "gqa4", 64, (1, 1), (2047, 8191), "bf16", window=1024, sinks=4),
        # one long context, no GQA, a wider window
        _attn("decode_1x32768_w4096_mha_fp16", "decode", "mha", 1, (1, 1), (32767, 32767), "fp16", window=4096, sinks=16),
        # a prompt over the 4-bit cache that holds it; a later part of a long one
        _attn("prefill4_2048_gqa4_bf16", "prefill4", "gqa4", 1, (2048, 2048), (0, 0), "bf16"),
        _attn("prefill4_512_of_16896_gqa7_fp16", "prefill4", "gqa7", 1, (512, 512), (16384, 16384), "fp16"),
        # a long prompt under a window, the most products
        _attn("prefill_8192_w1024_gqa4_bf16", "prefill", "gqa4", 1, (8192, 8192), (0, 0), "bf16", window=1024, sinks=4),
        # ragged prompts and continuations of a small batch under a narrow window
        _attn("prefill_5_w512_mha_fp16", "prefill", "mha", 5, (1, 701), (0, 3001), "fp16", window=512, sinks=16),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(("kv4", "decode4", "decode4", "decode", "prefill4", "prefill"))
    heads, dtype, dim = rng.choice(sorted(HEADS)), rng.choice(sorted(DTYPES)), rng.choice((128, 128, 128, 64))
    hq, hkv = HEADS[heads]
    page = rng.choice((16, 16, 16, 32, 8))
    if kind == "kv4":
        return {"kind": kind, "heads": heads, "tokens": _log_int(rng, 1, 8192), "page": page, "dim": dim, "dtype": dtype}
    window, sinks = rng.choice((0, 1)) * _log_int(rng, 16, 8192), rng.choice((0, 1, 4, 16, 64))
    least = rng.choice((1, 2, 16))
    if kind.startswith("decode"):
        requests, hi = _log_int(rng, 1, 64), _log_int(rng, 1, 131072)
        # no more cache, held and read, than the largest listed calls
        hi = max(1, min(hi, 64 * 10240 * 8 // (requests * hkv * (1 if kind == "decode4" else 4))))
        return _drawn(kind, heads, requests, (1, 1), (hi // least, hi), dtype, window, sinks, page, dim)
    requests, new, hi = _log_int(rng, 1, 6), _log_int(rng, 2, 4096), _log_int(rng, 1, 16384)
    # no more scores than the largest listed call has
    new = max(1, min(new, 8192 * 8192 * 32 // (requests * hq * (hi + 4096))))
    return _drawn(kind, heads, requests, (max(1, new // least), new), (hi // rng.choice((1, 3, 20000)), hi), dtype, window,
                  sinks, page, dim)


def _drawn(*args):
    case = _attn("", *args)
    del case["name"]
    return case


# ------------------------------------------------------------------- inputs
def _spread(n, lo, hi):
    """n whole numbers evenly over lo .. hi, in no order."""
    at = sorted(range(n), key=lambda i: (i * 7919 + 13) % (n + 1))
    return [lo + (hi - lo) * i // max(1, n - 1) if n > 1 else hi for i in at]


def _sizes(case):
    """(queries, tokens before them) of each request."""
    n = case["requests"]
    return _spread(n, case["min_new"], case["max_new"]), _spread(n, case["min_len"], case["max_len"])[::-1]


def prepare(case, seed):
    gen = torch.Generator().manual_seed(seed)
    dev = torch.Generator(device="cuda").manual_seed(seed)
    (hq, hkv), dtype = HEADS[case["heads"]], DTYPES[case["dtype"]]
    dim, page = case["dim"], case["page"]
    if case["kind"] == "kv4":
        n = case["tokens"]
        pool = -(-n // page) + 3
        slots = torch.randperm(pool * page, generator=gen)[:n].cuda()
        k, v = (torch.randn((n, hkv, dim), dtype=dtype, device="cuda", generator=dev) for _ in range(2))
        # K has channels of larger values
        k *= 1 + 7 * (torch.rand((1, hkv, dim), device="cuda", generator=dev) < 0.05).to(dtype)
        cache = torch.zeros((pool, 2, hkv, page * (dim // 2 + dim // GROUP)), dtype=torch.uint8, device="cuda")
        return {"kind": "kv4", "k": k, "v": v, "cache": cache, "page_id": slots // page, "page_offset": slots % page,
                "page": page}
    new, lens = _sizes(case)
    totals = torch.tensor([a + b for a, b in zip(new, lens)])
    pages = (totals + page - 1) // page
    pool = int(pages.sum()) + 3
    zero = torch.zeros(1, dtype=torch.int64)
    tables = {"paged_kv_indptr": torch.cat((zero, pages.cumsum(0))).int(),
              "paged_kv_indices": torch.randperm(pool, generator=gen)[: pool - 3].int(),
              "paged_kv_last_page_len": (totals - (pages - 1) * page).int()}
    qo_indptr = torch.cat((zero, torch.tensor(new).cumsum(0))).int()
    q = torch.randn((sum(new), hq, dim), dtype=dtype, device="cuda", generator=dev)
    four = case["kind"].endswith("4")
    if four:
        cache = torch.empty((pool, 2, hkv, page * (dim // 2 + dim // GROUP)), dtype=torch.uint8, device="cuda")
        step = max(1, (1 << 26) // (page * hkv * dim))
        for first in range(0, pool, step):
            part = cache[first: first + step]
            for i in (0, 1):
                x = torch.randn((part.shape[0] * page, hkv, dim), device="cuda", generator=dev)
                at = torch.arange(x.shape[0], device="cuda")
                _plain_append(part, i, x, at // page, at % page, page)
    else:
        cache = torch.randn((pool, 2, page, hkv, dim), dtype=dtype, device="cuda", generator=dev)
    decode = case["kind"].startswith("decode")
    state = {"kind": "decode" if decode else "prefill", "four": four, "q": q, "cache": cache, "heads": (hq, hkv),
             "page": page, "qo_indptr": qo_indptr.cuda(), "tables": {k: v.cuda() for k, v in tables.items()},
             "window": case["window"], "sinks": case["sinks"], "most_new": max(new), "most": int(totals.max()),
             "span": max(_span(a, b, case["window"]) for a, b in zip(new, lens))}
    if own:
        # the step's plan, which all layers of a model share
        from pagelora_amd.window_attention import WindowAttention

        attn = state["attn"] = WindowAttention(device="cuda", num_qo_heads=hq, num_kv_heads=hkv, head_dim=dim,
                                               page_size=page, window=case["window"], sinks=case["sinks"])
        if decode:
            attn.plan_decode(**state["tables"])
        else:
            attn.plan_prefill(qo_indptr=qo_indptr, **tables)
    return state


def _span(new, before, window):
    """Positions from the first that some query's window holds to the last."""
    return new + min(before, window - 1 if window else before)


# --------------------------------------------------------------------- runs
def run(state):
    if state["kind"] == "kv4":
        return _run_kv4(state)
    if own:
        return (state["attn"].run_decode if state["kind"] == "decode" else state["attn"].run_prefill)(state["q"], state["cache"])
    return _plain_attention(state)


def _run_kv4(s):
    (n, hkv, dim), page = s["k"].shape, s["page"]
    if own:
        from pagelora_amd.kv4 import kv4_append, kv4_read

        sizes = {"num_kv_heads": hkv, "head_dim": dim, "page_size": page}
        kv4_append(s["cache"], s["k"], s["v"], s["page_id"], s["page_offset"], **sizes)
        return kv4_read(s["cache"], s["page_id"], s["page_offset"], dtype=s["k"].dtype, **sizes)
    for i, x in enumerate((s["k"], s["v"])):
        _plain_append(s["cache"], i, x.float(), s["page_id"], s["page_offset"], page)
    return tuple(_plain_values(s["cache"], i, s["page_id"], s["page_offset"], page, dim).to(s["k"].dtype) for i in (0, 1))


def _places(cache, i, page, dim):
    """Views of K's (i 0) or V's part of a 4-bit layer: codes and scales, and how a token's place in a page indexes them."""
    part, cut = cache[:, i], page * dim // 2
    codes, scales = part[..., :cut], part[..., cut:]
    if i == 0:
        return codes.unflatten(2, (page, dim // 2)), scales.unflatten(2, (page, dim // GROUP)), None
    return codes.unflatten(2, (page // 4, dim // 8, 4, 4)), scales.unflatten(2, (page // 4, dim // GROUP, 4)), 4


def _plain_append(cache, i, x, page_id, offset, page):
    dim = x.shape[2]
    groups = x.unflatten(2, (dim // GROUP, GROUP))
    top = groups.abs().amax(3).view(torch.int32)
    held = top < 255 << 23
    scale = ((top >> 23) - 2 + ((top & 0x7FFFFF) > 0x400000).int()).clamp(2, 252)
    y = groups * ((254 - scale) << 23).view(torch.float32)[..., None]
    a = y.abs()
    # to the nearest of LEVELS, halfway to the one with an even mantissa
    code = (a > 0.25).to(torch.uint8)
    for border, up in ((0.75, True), (1.25, False), (1.75, True), (2.5, False), (3.5, True), (5.0, False)):
        code += (a >= border) if up else (a > border)
    code = torch.where(held[..., None], code + 8 * torch.signbit(y).to(torch.uint8), 0).flatten(2)
    packed = code[..., 0::2] + 16 * code[..., 1::2]
    scale = torch.where(held, scale, 255).to(torch.uint8)
    codes, scales, quad = _places(cache, i, page, dim)
    if quad is None:
        codes[page_id, :, offset] = packed
        scales[page_id, :, offset] = scale
    else:
        codes[page_id, :, offset // 4, :, offset % 4] = packed.unflatten(2, (dim // 8, 4))
        scales[page_id, :, offset // 4, :, offset % 4] = scale


def _plain_values(cache, i, page_id, offset, page, dim):
    """fp32 values of the tokens at these places: [..., kv heads, dim]."""
    codes, scales, quad = _places(cache, i, page, dim)
    if quad is None:
        c, s = codes[page_id, :, offset], scales[page_id, :, offset]
    else:
        c, s = codes[page_id, :, offset // 4, :, offset % 4].flatten(-2), scales[page_id, :, offset // 4, :, offset % 4]
    table = torch.tensor(LEVELS + tuple(-x for x in LEVELS), device=cache.device)
    values = torch.stack((table[(c & 15).int()], table[(c >> 4).int()]), -1).flatten(-2)
    power = torch.where(s == 255, math.nan, (s.int() << 23).view(torch.float32))
    return (values.unflatten(-1, (dim // GROUP, GROUP)) * power[..., None]).flatten(-2)


def _plain_attention(state):
    q, cache, t, page = state["q"], state["cache"], state["tables"], state["page"]
    (hq, hkv), window, sinks, dim = state["heads"], state["window"], state["sinks"], q.shape[2]
    starts, pages = t["paged_kv_indptr"][:-1].long(), t["paged_kv_indptr"].diff().long()
    total = (pages - 1) * page + t["paged_kv_last_page_len"]
    first, new = state["qo_indptr"][:-1].long(), state["qo_indptr"].diff().long()
    before = total - new
    # the positions that some query of a request sees, side by side: sinks, then from the first window on
    lo = (before - window + 1).clamp(min=0) if window else torch.zeros_like(before)
    sink = torch.arange(min(sinks, state["most"]) if window else 0, device=q.device).expand(lo.numel(), -1)
    pos = torch.cat((sink, lo[:, None] + torch.arange(state["span"], device=q.device)), 1)
    there = (pos < total[:, None]) & torch.cat((sink < lo[:, None], torch.ones_like(pos[:, sink.shape[1]:], dtype=torch.bool)), 1)
    at = torch.minimum(pos, total[:, None] - 1)
    ids, offset = t["paged_kv_indices"].long()[starts[:, None] + at // page], at % page
    if state["four"]:
        k, v = (_plain_values(cache, i, ids, offset, page, dim).transpose(1, 2) for i in (0, 1))
    else:
        k, v = (cache[ids, i, offset].transpose(1, 2).float() for i in (0, 1))
    # the queries padded to the most: [requests, kv heads, queries x group, dim]
    width, g = state["most_new"], hq // hkv
    j = torch.arange(width, device=q.device)
    inside = j < new[:, None]
    rows = (first[:, None] + j).clamp(max=q.shape[0] - 1)
    qs = q[rows].float().unflatten(2, (hkv, g)).permute(0, 2, 1, 3, 4).flatten(2, 3)
    scores = torch.matmul(qs, k.transpose(2, 3).contiguous()) / math.sqrt(dim)
    p = (before[:, None] + j)[:, :, None]
    sees = there[:, None] & (pos[:, None] <= p)
    if window:
        sees &= (pos[:, None] > p - window) | (pos[:, None] < sinks)
    scores = scores.unflatten(2, (width, g)).masked_fill_(~sees[:, None, :, None], -math.inf).flatten(2, 3)
    scores = torch.exp(scores.sub_(scores.amax(3, keepdim=True).clamp(min=-3e38)))
    out = torch.matmul(scores, v) / scores.sum(3, keepdim=True).clamp(min=1e-38)
    return out.unflatten(2, (width, g)).permute(0, 2, 1, 3, 4).flatten(2, 3)[inside].to(q.dtype)


# --------------------------------------------------------------------- work
def work(case):
    (hq, hkv), dim = HEADS[case["heads"]], case["dim"]
    four = 2 * hkv * (dim // 2 + dim // GROUP)  # bytes of a token in 4 bits, and in 16
    wide = 2 * hkv * dim * 2
    if case["kind"] == "kv4":
        return {"bytes": case["tokens"] * 2 * (wide + four), "flops": 0}
    new, lens = _sizes(case)
    window, sinks = case["window"], case["sinks"]
    read = pairs = 0
    for n, b in zip(new, lens):
        lo = max(0, b - window + 1) if window else 0
        read += n + b - lo + min(sinks, lo)
        for p in range(b, b + n):
            low = max(0, p - window + 1) if window else 0
            pairs += p + 1 - low + min(sinks, low)
    return {"bytes": read * (four if case["kind"].endswith("4") else wide) + 4 * sum(new) * hq * dim,
            "flops": 4 * pairs * hq * dim}


# -------------------------------------------------------------------- exact
def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "kv4":
        return tuple(_exact_quantized(x.double()) for x in (s["k"], s["v"]))
    t = {k: v.tolist() for k, v in s["tables"].items()}
    (hq, hkv), page, dim, outs = s["heads"], s["page"], case["dim"], []
    qo = s["qo_indptr"].tolist()
    for r, last in enumerate(t["paged_kv_last_page_len"]):
        ids = torch.tensor(t["paged_kv_indices"][t["paged_kv_indptr"][r]: t["paged_kv_indptr"][r + 1]], device="cuda")
        total = (len(ids) - 1) * page + last
        if s["four"]:
            k, v = _exact_pages(s["cache"][ids], page, dim)
        else:
            k, v = s["cache"][ids].double().transpose(0, 1).flatten(1, 2)
        q = s["q"][qo[r]: qo[r + 1]].double()
        p = torch.arange(total - q.shape[0], total, device="cuda")[:, None]
        pos = torch.arange(total, device="cuda")[None, :]
        hidden = pos > p
        if s["window"]:
            hidden |= (p - pos >= s["window"]) & (pos >= s["sinks"])
        heads = []
        for h in range(hq):
            x = q[:, h] @ k[:total, h // (hq // hkv)].T.contiguous() * dim ** -0.5
            heads.append(torch.softmax(x.masked_fill_(hidden, -math.inf), 1) @ v[:total, h // (hq // hkv)])
        outs.append(torch.stack(heads, 1))
    return torch.cat(outs)


def _exact_quantized(x):
    """Every 32 values at the nearest multiple of a step that doubles at 2 and 4 times their power of two."""
    y = x.unflatten(2, (x.shape[2] // GROUP, GROUP))
    e = torch.ceil(torch.log2(y.abs().amax(3, keepdim=True) / 6)).clamp(-125, 125)
    unit = torch.pow(2.0, e)
    a = y.abs() / unit
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    return (torch.sign(y) * (torch.round(a / step) * step).clamp(max=6) * unit).flatten(2)


def _exact_pages(pages, page, dim):
    """K and V of whole pages in 64 bits: [tokens, kv heads, dim]."""
    n, _, hkv, _ = pages.shape
    codes, scales = pages.split((page * dim // 2, page * dim // GROUP), 3)
    kc, vc = codes.unbind(1)
    ks, vs = scales.unbind(1)
    kc = kc.reshape(n, hkv, page, dim // 2)
    vc = vc.reshape(n, hkv, page // 4, dim // 8, 4, 4).transpose(3, 4).reshape(n, hkv, page, dim // 2)
    ks = ks.reshape(n, hkv, page, dim // GROUP)
    vs = vs.reshape(n, hkv, page // 4, dim // GROUP, 4).transpose(3, 4).reshape(n, hkv, page, dim // GROUP)
    out = []
    for c, s in ((kc, ks), (vc, vs)):
        c = torch.stack((c & 15, c >> 4), 4).flatten(3).double()
        sign, c = torch.where(c >= 8, -1.0, 1.0), c % 8
        e, m = torch.floor(c / 2), c % 2
        x = sign * torch.where(e > 0, (1 + m / 2) * torch.pow(2.0, e - 1), m / 2)
        x = x * torch.pow(2.0, s.double() - 127).repeat_interleave(GROUP, 3)
        out.append(x.transpose(1, 2).flatten(0, 1))
    return out
