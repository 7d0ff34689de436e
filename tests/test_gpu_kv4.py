"""Tokens into a 4-bit paged cache and back: every byte against the format's definition in 64 bits."""

import numpy as np
import pytest
import torch

from oracle import window as ow
from pagelora_amd.kv4 import kv4_append, kv4_page_shape, kv4_read
from pagelora_amd.kv_pool import PagedKVPool, Request, kv_copy_pages
from pagelora_amd import fused_ops
from tests.window_cases import BF16, F16, check
from pagelora_amd.window_attention import WindowAttention

pytestmark = pytest.mark.gpu


def sizes(hkv, head_dim, page):
    return {"num_kv_heads": hkv, "head_dim": head_dim, "page_size": page}


def empty(pages, hkv, head_dim, page, device, fill=0):
    return torch.full((pages, *kv4_page_shape(**sizes(hkv, head_dim, page))), fill, dtype=torch.uint8, device=device)


def expected(layer, k, v, page_id, offset, page):
    """``layer`` (host) with the tokens written, and their values."""
    hkv, d = k.shape[1:]
    out = layer.numpy().copy()
    (kc, ks), (vc, vs) = (ow.quantize(x.double().cpu().numpy()) for x in (k, v))
    cut = page * d // 2
    kcodes = out[:, 0, :, :cut].reshape(-1, hkv, page, d // 2)
    kscale = out[:, 0, :, cut:].reshape(-1, hkv, page, d // 32)
    vcodes = out[:, 1, :, :cut].reshape(-1, hkv, page // 4, d // 8, 4, 4)
    vscale = out[:, 1, :, cut:].reshape(-1, hkv, page // 4, d // 32, 4)
    pair = lambda c: c[..., 0::2] | (c[..., 1::2] << 4)  # noqa: E731
    for i, (p, o) in enumerate(zip(page_id.tolist(), offset.tolist())):
        if not (0 <= p < out.shape[0] and 0 <= o < page):
            continue
        kcodes[p, :, o], kscale[p, :, o] = pair(kc[i]), ks[i]
        vcodes[p, :, o // 4, :, o % 4], vscale[p, :, o // 4, :, o % 4] = pair(vc[i]).reshape(hkv, d // 8, 4), vs[i]
    whole = np.stack([np.concatenate([kcodes.reshape(-1, hkv, cut), kscale.reshape(out.shape[0], hkv, -1)], 2),
                      np.concatenate([vcodes.reshape(-1, hkv, cut), vscale.reshape(out.shape[0], hkv, -1)], 2)], 1)
    return whole, ow.values(kc, ks), ow.values(vc, vs)


def places(n, pages, page, seed):
    at = torch.randperm(pages * page, generator=torch.Generator().manual_seed(seed))[:n]
    return at // page, at % page


def run(k, v, page_id, offset, page, pages, device, fill=0):
    layer = empty(pages, *k.shape[1:], page, device, fill)
    where = page_id.to(device), offset.to(device)
    kv4_append(layer, k.to(device), v.to(device), *where, **sizes(*k.shape[1:], page))
    back = kv4_read(layer, *where, dtype=k.dtype, **sizes(*k.shape[1:], page))
    torch.cuda.synchronize()
    return layer.cpu().numpy(), [x.cpu() for x in back]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("tokens", [1, 2, 5, 64, 700])
@pytest.mark.parametrize("hkv,head_dim,page", [(1, 64, 8), (3, 64, 16), (8, 128, 16), (1, 128, 8), (2, 128, 40), (33, 64, 64)])
def test_bytes_and_values(gpu_device, dtype, tokens, hkv, head_dim, page):
    gen = torch.Generator().manual_seed(tokens + hkv)
    k, v = (torch.randn((tokens, hkv, head_dim), generator=gen).to(dtype) for _ in range(2))
    pages = -(-tokens // page) + 2
    where = places(tokens, pages, page, 1)
    layer, back = run(k, v, *where, page, pages, gpu_device, fill=0xA5)
    want, kv, vv = expected(torch.full(layer.shape, 0xA5, dtype=torch.uint8), k, v, *where, page)
    assert (layer == want).all()
    for got, value in zip(back, (kv, vv)):
        assert torch.equal(got, torch.from_numpy(value).to(dtype))


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_borders(gpu_device, dtype):
    """Groups of one magnitude after another, so that the largest passes every power's border, and values halfway between two levels;
    the smallest and largest of the type; zeros of both signs."""
    tiny = torch.finfo(dtype).smallest_normal
    tops = [6.0, 6.03125, 5.96875, 3.0, 3.015625, 4.0, 1.0, 0.75, 48.0, 0.0, -0.0, tiny, tiny / 8, -tiny, torch.finfo(dtype).max,
            -torch.finfo(dtype).max, 448.0, 1e-4]
    level = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 0.2421875, 0.2578125, 4.96875, 5.03125, 0.0, -0.0, 1.0, 2.0, 0.5])
    x = torch.zeros((len(tops), 1, 128), dtype=torch.float64)
    for i, top in enumerate(tops):
        unit = abs(top) / 6 if top else 1.0
        x[i, 0] = torch.cat((level, -level)).repeat(4).double() * unit
        x[i, 0, ::32] = top
    x = x.to(dtype)
    where = places(len(tops), 3, 16, 2)
    layer, back = run(x, x.flip(0), *where, 16, 3, gpu_device)
    want, kv, vv = expected(torch.zeros(layer.shape, dtype=torch.uint8), x, x.flip(0), *where, 16)
    assert (layer == want).all()
    for got, value in zip(back, (kv, vv)):
        assert torch.equal(got, torch.from_numpy(value).to(dtype))


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_error_of_a_value(gpu_device, dtype):
    """Half the distance of the levels around it.  With the largest magnitude in (3, 6] powers of two: in (3, 4] no two levels
    are more than 1 apart, 0.5 <= a sixth of it; above, the levels 4 and 6 give up to 1 for values of 5 and more, and below
    5 the distance to 4 is under a fifth of it: a fifth in all.  Of a value of one power and more, halfway at 1.25, 2.5 and
    5: a fifth of the value."""
    x = torch.randn((256, 2, 128), generator=torch.Generator().manual_seed(4)).to(dtype)
    _, (k, _) = run(x, x, *places(256, 16, 16, 3), 16, 16, gpu_device)
    groups, got = x.double().unflatten(2, (4, 32)), k.double().unflatten(2, (4, 32))
    top = groups.abs().amax(3, keepdim=True)
    off = (groups - got).abs()
    assert (off <= top / 5).all()
    assert (off <= groups.abs() / 5)[groups.abs() * 3 >= top].all()


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_groups_of_zeros(gpu_device, dtype):
    """Scale 127, that of 4 to 6, whatever stands beside them."""
    x = torch.randn((9, 2, 64), generator=torch.Generator().manual_seed(8)).to(dtype)
    x[..., 32:] = 0.0
    x[1, :, 40] = -0.0
    where = places(9, 2, 8, 5)
    layer, back = run(x, x, *where, 8, 2, gpu_device, fill=0xA5)
    scales = torch.from_numpy(layer)[..., 8 * 32:]
    k = scales[:, 0].unflatten(2, (8, 2))[where[0], :, where[1]]
    v = scales[:, 1].unflatten(2, (2, 2, 4))[where[0], :, where[1] // 4, :, where[1] % 4]
    assert (k[..., 1] == 127).all() and (v[..., 1] == 127).all() and (k[..., 0] != 127).any()
    assert torch.equal(back[0][..., 32:], x[..., 32:]) and torch.equal(back[1][..., 32:], x[..., 32:])


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_what_is_not_finite_marks_its_group(gpu_device, dtype, bad):
    x = torch.randn((6, 2, 128), generator=torch.Generator().manual_seed(5)).to(dtype)
    y = x.clone()
    y[2, 1, 37] = bad
    y[4, 0, 127] = bad
    where = places(6, 2, 16, 4)
    layer, (k, v) = run(y, x, *where, 16, 2, gpu_device)
    assert (layer == expected(torch.zeros(layer.shape, dtype=torch.uint8), y, x, *where, 16)[0]).all()
    want = torch.zeros(k.shape, dtype=torch.bool)
    want[2, 1, 32:64] = True
    want[4, 0, 96:] = True
    assert torch.equal(k.isnan(), want) and not v.isnan().any()


def test_places_outside_the_pool(gpu_device):
    x = torch.randn((6, 2, 128), generator=torch.Generator().manual_seed(6)).to(BF16)
    ids, offs = torch.tensor([0, -1, 2, 1, 1, 2**40]), torch.tensor([3, 0, 0, 16, -1, 0])
    layer, (k, v) = run(x, x, ids, offs, 16, 2, gpu_device, fill=7)
    assert (layer == expected(torch.full(layer.shape, 7, dtype=torch.uint8), x, x, ids, offs, 16)[0]).all()
    assert k[1:].isnan().all() and v[1:].isnan().all() and k[0].isfinite().all()


def test_strides_and_large_pools(gpu_device):
    """K and V as slices of a packed projection, a pool past 4 GiB, K and V halves of pages apart."""
    x = torch.randn((9, 12, 128), generator=torch.Generator().manual_seed(7)).to(BF16).to(gpu_device)
    shape = kv4_page_shape(**sizes(2, 128, 16))
    apart = (1 << 30) // 16 * 16
    memory = torch.zeros(5 * apart + 2 * 2 * shape[2], dtype=torch.uint8, device=gpu_device)
    layer = memory.as_strided((6, *shape), (apart, 2 * shape[2], shape[2], 1))
    ids, offs = torch.tensor([5, 4, 3, 2, 1, 0, 5, 5, 0]), torch.arange(9)
    where = ids.to(gpu_device), offs.to(gpu_device)
    kv4_append(layer, x[:, 8:10], x[:, 10:], *where, **sizes(2, 128, 16))
    want, kv, vv = expected(torch.zeros(layer.shape, dtype=torch.uint8), x[:, 8:10], x[:, 10:], ids, offs, 16)
    assert (layer.cpu().numpy() == want).all()
    for got, value in zip(kv4_read(layer, *where, **sizes(2, 128, 16)), (kv, vv)):
        assert torch.equal(got.cpu(), torch.from_numpy(value).to(BF16))


def test_capture(gpu_device):
    x = torch.randn((5, 2, 128), generator=torch.Generator().manual_seed(8)).to(BF16).to(gpu_device)
    layer = empty(2, 2, 128, 16, gpu_device)
    ids, offs = (t.to(gpu_device) for t in places(5, 2, 16, 5))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kv4_append(layer, x, x, ids, offs, **sizes(2, 128, 16))
        k, v = kv4_read(layer, ids, offs, **sizes(2, 128, 16))
    for i in range(3):
        x.mul_(-1.5)
        layer.zero_()
        graph.replay()
        torch.cuda.synchronize()
        _, kv, vv = expected(torch.zeros(layer.shape, dtype=torch.uint8), x, x, ids, offs, 16)
        assert torch.equal(k.cpu(), torch.from_numpy(kv).to(BF16)) and torch.equal(v.cpu(), torch.from_numpy(vv).to(BF16))


def test_pages_of_a_4_bit_pool_are_copied(gpu_device):
    pool = PagedKVPool(num_layers=3, capacity_pages=12, page_size=8, num_kv_heads=3, head_dim=64, dtype=BF16, device=gpu_device, kv_bits=4)
    pool.cache.random_(0, 256)
    before = pool.cache.clone()
    pool.copy_pages([2, 5, 2], [7, 1, 0])
    want = before.clone()
    for s, d in ((2, 7), (5, 1), (2, 0)):
        want[:, d] = before[:, s]
    assert torch.equal(pool.cache, want)
    kv_copy_pages(pool.cache[1], [3], [4])
    want[1, 4] = want[1, 3]
    assert torch.equal(pool.cache, want)
    request = Request()
    pool.reserve(request, 20)
    fork, = pool.fork([request])
    assert fork.own_pages[:2] == request.own_pages[:2] and fork.own_pages[2] != request.own_pages[2]
    assert torch.equal(pool.cache[:, fork.own_pages[2]], pool.cache[:, request.own_pages[2]])
    pool.reserve(request, 200)  # grows
    assert torch.equal(pool.cache[1, 4], want[1, 4])


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("window,sinks", [(0, 0), (24, 4)])
def test_a_request_from_prompt_to_fork(gpu_device, dtype, window, sinks):
    """What a server does: two layers' prompts rotated and quantized, attended in two parts, decoded token by token in one
    graph (append, plan, attention), forked, and both continuations decoded."""
    hq, hkv, d, page, layers = 8, 2, 128, 16, 2
    pool = PagedKVPool(num_layers=layers, capacity_pages=40, page_size=page, num_kv_heads=hkv, head_dim=d, dtype=dtype,
                       device=gpu_device, kv_bits=4)
    attn = WindowAttention(device=gpu_device, num_qo_heads=hq, num_kv_heads=hkv, head_dim=d, page_size=page, window=window,
                           sinks=sinks)
    size = sizes(hkv, d, page)
    gen = torch.Generator(device=gpu_device).manual_seed(9)
    norm = torch.ones(d, dtype=dtype, device=gpu_device)
    history = {}  # (request, layer) -> K and V as the cache holds them

    def rotated(tokens, positions):
        """q, k, v of new tokens, through the framework's norm and rotation into a scratch cache of one token a page."""
        qkv = torch.randn((tokens, (hq + 2 * hkv) * d), generator=gen, device=gpu_device).to(dtype)
        scratch = torch.empty((tokens, 2, 1, hkv, d), dtype=dtype, device=gpu_device)
        at = torch.arange(tokens, device=gpu_device)
        q = fused_ops.qk_norm_rope_append(qkv, norm, norm, positions, at, torch.zeros_like(at), scratch, num_qo_heads=hq,
                                          num_kv_heads=hkv, head_dim=d, page_size=1, eps=1e-6, rope_theta=1e4)
        return q.view(tokens, hq, d), scratch[:, 0, 0], scratch[:, 1, 0]

    def keep(name, layer, k, v):
        held = [torch.from_numpy(ow.values(*ow.quantize(x.double().cpu().numpy()))) for x in (k, v)]
        old = history.get((name, layer))
        history[name, layer] = held if old is None else [torch.cat(x) for x in zip(old, held)]

    def verify(names, new, layer, q, out):
        lens = [history[n, layer][0].shape[0] for n in names]
        pages = [-(-n // page) for n in lens]
        cache = np.zeros((sum(pages), 2, page, hkv, d))
        first = 0
        for n, ln, p in zip(names, lens, pages):
            for i in (0, 1):
                cache[first: first + p, i].reshape(p * page, hkv, d)
                flat = np.zeros((p * page, hkv, d))
                flat[:ln] = history[n, layer][i].numpy()
                cache[first: first + p, i] = flat.reshape(p, page, hkv, d)
            first += p
        c = {"heads": (hq, hkv), "head_dim": d, "dtype": dtype, "bits": 4, "window": window, "sinks": sinks, "lens": lens,
             "indptr": torch.tensor([0, *np.cumsum(pages)]), "indices": torch.arange(sum(pages)), "cache_host": cache,
             "qo_indptr": torch.tensor([0, *np.cumsum(new)]), "q_host": q.cpu(), "prefill": max(new) > 1}
        check(c, out)

    def slots(request, positions):
        where = [request.slot(p, page) for p in positions]
        return (torch.tensor([w[i] for w in where], device=gpu_device) for i in (0, 1))

    def tables(requests):
        names = ("paged_kv_indptr", "paged_kv_indices", "paged_kv_last_page_len")
        return {n: torch.from_numpy(t) for n, t in zip(names, pool.tables(requests))}

    a = Request()
    for part in (37, 14):  # the prompt in two parts
        start = a.length
        pool.reserve(a, part)
        ids, offs = slots(a, range(start, a.length))
        attn.plan_prefill(qo_indptr=torch.tensor([0, part], dtype=torch.int32), **tables([a]))
        for layer in range(layers):
            q, k, v = rotated(part, torch.arange(start, a.length, device=gpu_device))
            kv4_append(pool.cache[layer], k, v, ids, offs, **size)
            keep("a", layer, k, v)
            verify(["a"], [part], layer, q, attn.run_prefill(q, pool.cache[layer]))
    requests, names = [a], ["a"]
    for turn in range(2):
        graph = None
        room = max(len(r.pages()) for r in requests) + 3
        static = {"paged_kv_indptr": torch.zeros(len(requests) + 1, dtype=torch.int32, device=gpu_device),
                  "paged_kv_indices": torch.zeros(room * len(requests), dtype=torch.int32, device=gpu_device),
                  "paged_kv_last_page_len": torch.zeros(len(requests), dtype=torch.int32, device=gpu_device)}
        n = len(requests)
        qs = torch.zeros((layers, n, hq, d), dtype=dtype, device=gpu_device)
        ks, vs = (torch.zeros((layers, n, hkv, d), dtype=dtype, device=gpu_device) for _ in range(2))
        ids, offs = (torch.zeros(n, dtype=torch.int64, device=gpu_device) for _ in range(2))
        for step in range(18):
            for r in requests:
                pool.reserve(r, 1)
            where = [r.slot(r.length - 1, page) for r in requests]
            ids.copy_(torch.tensor([w[0] for w in where]))
            offs.copy_(torch.tensor([w[1] for w in where]))
            for name, t in tables(requests).items():
                static[name][: t.numel()].copy_(t)
            for layer in range(layers):
                q, k, v = rotated(n, torch.tensor([r.length - 1 for r in requests], device=gpu_device))
                qs[layer].copy_(q), ks[layer].copy_(k), vs[layer].copy_(v)
                for i, name in enumerate(names):
                    keep(name, layer, k[i: i + 1], v[i: i + 1])
            if graph is None:
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph):
                    attn.plan_decode(**static)
                    outs = []
                    for layer in range(layers):
                        kv4_append(pool.cache[layer], ks[layer], vs[layer], ids, offs, **size)
                        outs.append(attn.run_decode(qs[layer], pool.cache[layer]))
            graph.replay()
            torch.cuda.synchronize()
            for layer in range(layers):
                verify(names, [1] * n, layer, qs[layer], outs[layer])
        if turn == 0:
            requests += pool.fork([a])
            names.append("b")
            for layer in range(layers):
                history["b", layer] = [x.clone() for x in history["a", layer]]
