"""Decode attention under a window with sinks, over 16-bit and 4-bit caches, against 64 bits."""

import numpy as np
import pytest
import torch

from tests.window_cases import BF16, F16, attention, case, check, decode, reference, set_cache, tables

pytestmark = pytest.mark.gpu

RAGGED = [0, 1, 3, 15, 16, 17, 31, 32, 33, 64, 127, 128, 129, 300, 1000, 1, 0]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("heads", [(1, 1), (8, 2), (14, 2), (2, 2), (33, 1), (48, 3)])
@pytest.mark.parametrize("head_dim", [64, 128])
def test_heads(gpu_device, dtype, bits, heads, head_dim):
    """One head, GQA of powers of two and not, no GQA, groups over one and two blocks of 16 heads."""
    c = case(RAGGED, *heads, head_dim, 16, dtype, gpu_device, bits=bits, window=100, sinks=5, seed=3)
    check(c, *decode(c))


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("window,sinks", [(0, 0), (0, 7), (1, 0), (1, 1), (5, 0), (31, 4), (32, 32), (33, 33), (64, 100),
                                          (500, 1), (1000, 16), (2**31 - 1, 2**31 - 1), (7, 2**31 - 1)])
def test_windows(gpu_device, bits, window, sinks):
    """Windows of one token, of whole tiles and one more, longer than the sequences; sinks that meet the window."""
    c = case(RAGGED, 8, 2, 128, 16, BF16, gpu_device, bits=bits, window=window, sinks=sinks, seed=window % 97)
    check(c, *decode(c))


@pytest.mark.parametrize("bits,page", [(16, 1), (16, 3), (16, 4), (16, 7), (16, 32), (16, 48), (16, 1024), (4, 8), (4, 24),
                                       (4, 32), (4, 40), (4, 48), (4, 1024)])
@pytest.mark.parametrize("head_dim", [64, 128])
def test_pages(gpu_device, bits, page, head_dim):
    c = case(RAGGED, 8, 2, head_dim, page, F16, gpu_device, bits=bits, window=70, sinks=33, seed=page)
    check(c, *decode(c))


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("lens", [[1], [4097], [20000], [9000, 1, 2500], [700] * 70])
def test_lengths(gpu_device, bits, lens):
    """One request cut into many items, several, a large batch."""
    c = case(lens, 4, 1, 128, 16, BF16, gpu_device, bits=bits, seed=len(lens))
    check(c, *decode(c))


@pytest.mark.parametrize("dtype,bits", [(BF16, 16), (F16, 16), (BF16, 4), (F16, 4)])
def test_scores_far_apart(gpu_device, dtype, bits):
    """Peaked rows, whose maxima rise along the sequence."""
    c = case([40, 513, 2000], 8, 2, 128, 16, dtype, gpu_device, bits=bits, seed=8, q_scale=30.0)
    check(c, *decode(c))


def test_large_values_stay_finite(gpu_device):
    """bf16 V near the type's largest: their mean is finite, their sums in 32 bits need not be."""
    for bits in (16, 4):
        c = case([500], 4, 1, 128, 16, BF16, gpu_device, bits=bits, seed=2, poison=False)
        cache = torch.randn((c["indices"].numel() + 3, 2, 16, 1, 128), generator=torch.Generator().manual_seed(1))
        cache[:, 1] = 2.5e38
        set_cache(c, cache.to(BF16))
        check(c, *decode(c))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("where", [0, 1, 17, 600, 998, 999])
def test_infinities_and_nan_in_v(gpu_device, dtype, where):
    """What a row sees of them is its output, in their dims alone; in every place of the cut."""
    c = case([1000, 40], 8, 2, 128, 16, dtype, gpu_device, seed=5, poison=False)
    cache = torch.from_numpy(c["cache_host"]).to(dtype)
    page, off = int(c["indices"][where // 16]), where % 16
    cache[page, 1, off, 0, 3] = float("inf")
    cache[page, 1, off, 0, 40] = -float("inf")
    cache[page, 1, off, 1, 7] = float("nan")
    cache[page, 1, off, 1, 8] = float("inf")
    cache[int(c["indices"][31]), 1, 4, 1, 8] = -float("inf")
    set_cache(c, cache)
    assert np.isinf(reference(c)[0]).any() and np.isnan(reference(c)[0]).any()
    check(c, *decode(c))


@pytest.mark.parametrize("where", [0, 17, 999])
def test_nan_groups_of_a_4_bit_cache(gpu_device, where):
    c = case([1000, 40], 8, 2, 128, 16, BF16, gpu_device, seed=5, bits=4, poison=False)
    cache = torch.randn((c["indices"].numel() + 3, 2, 16, 2, 128), generator=torch.Generator().manual_seed(1)).to(BF16)
    cache[int(c["indices"][where // 16]), 1, where % 16, 0, 33] = float("nan")
    set_cache(c, cache)
    nan = np.isnan(reference(c)[0])
    assert nan[0, :4, 32:64].all() and nan.sum() == 4 * 32
    check(c, *decode(c))


@pytest.mark.parametrize("dtype,bits", [(BF16, 16), (F16, 4)])
def test_nan_in_k_and_q(gpu_device, dtype, bits):
    """A NaN score makes its row NaN, and no other."""
    c = case([300, 40, 50], 8, 2, 128, 16, dtype, gpu_device, bits=bits, seed=5, poison=False)
    cache = torch.randn((c["indices"].numel() + 3, 2, 16, 2, 128), generator=torch.Generator().manual_seed(1)).to(dtype)
    cache[int(c["indices"][3]), 0, 5, 1, 9] = float("nan")
    set_cache(c, cache)
    c["q_host"][1, 2, 3] = float("nan")
    c["q"] = c["q_host"].to(gpu_device)
    got, _ = decode(c)
    want = torch.zeros(3, 8, dtype=torch.bool)
    want[0, 4:] = True
    want[1, 2] = True
    nan = got.isnan().cpu()
    assert (nan.all(2) == want).all() and (nan.any(2) == want).all()


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("scale", [-0.2, 0.0, 3.0])
def test_softmax_scale(gpu_device, bits, scale):
    c = case([40, 300], 8, 2, 128, 16, F16, gpu_device, bits=bits, window=64, sinks=4, seed=11)
    attn = attention(c)
    attn.sm_scale = scale
    attn.plan_decode(**tables(c))
    check(c, attn.run_decode(c["q"], c["cache"]), sm_scale=scale)


@pytest.mark.parametrize("bits", [16, 4])
def test_strides(gpu_device, bits):
    """q and out as slices of wider rows, pages and heads of a pool at other distances, K and V apart."""
    c = case([1, 40, 300], 8, 2, 128, 16, BF16, gpu_device, bits=bits, window=64, sinks=4, seed=12)
    attn = attention(c)
    attn.plan_decode(**tables(c, gpu_device))
    wide = torch.full((3, 12, 136), float("nan"), dtype=BF16, device=gpu_device)
    wide[:, 2:10, :128] = c["q"]
    out = torch.full((3, 20, 128), 7.0, dtype=BF16, device=gpu_device)
    caches = []
    if bits == 16:
        k, v = c["cache"].unbind(1)
        caches.append((k.clone(), v.clone()))
        hnd = torch.empty((k.shape[0], 2, 2, 16, 128), dtype=BF16, device=gpu_device).transpose(2, 3)
        hnd.copy_(c["cache"])
        caches.append(hnd)
    big = torch.zeros((4, *c["cache"].shape), dtype=c["cache"].dtype, device=gpu_device)
    big[2] = c["cache"]
    caches.append(big.transpose(0, 1).contiguous()[:, 2])
    for cache in caches:
        out.fill_(7.0)
        attn.run_decode_into(wide[:, 2:10, :128], cache, out[:, 5:13])
        check(c, out[:, 5:13])
        assert (out[:, :5] == 7).all() and (out[:, 13:] == 7).all()
    assert attn.run_decode(c["q"][:, :, None], c["cache"]).shape == (3, 8, 1, 128)


@pytest.mark.parametrize("bits", [16, 4])
def test_pool_past_4_gib(gpu_device, bits):
    c = case([100, 33], 8, 2, 128, 16, BF16, gpu_device, bits=bits, seed=13, extra=0)
    n, per = c["cache"].shape[0], c["cache"][0].numel()
    apart = (5 << 30) // c["cache"].element_size() // n // 64 * 64
    memory = torch.empty(apart * n + per, dtype=c["cache"].dtype, device=gpu_device)
    cache = memory.as_strided(c["cache"].shape, (apart, *c["cache"].stride()[1:]))
    cache.copy_(c["cache"])
    c["cache"] = cache
    check(c, *decode(c))


def test_tokens_far_apart(gpu_device):
    """A page's 16 tokens over more than 4 GiB."""
    c = case([30], 4, 2, 128, 16, BF16, gpu_device, seed=13, extra=0)
    apart = 150 << 20  # values
    memory = torch.empty(16 * apart, dtype=BF16, device=gpu_device)
    cache = memory.as_strided(c["cache"].shape, (1024, 512, apart, 128, 1))
    cache.copy_(c["cache"])
    c["cache"] = cache
    check(c, *decode(c))


@pytest.mark.parametrize("bits", [16, 4])
def test_pages_that_nobody_sees_may_be_any(gpu_device, bits):
    """Page ids of what the window has left behind are not read: a freed page's, or none's."""
    c = case([500], 8, 2, 128, 16, BF16, gpu_device, bits=bits, window=64, sinks=4, seed=14)
    c["indices"][1:27] = 2**31 - 1
    attn = attention(c)
    attn.plan_decode(**tables(c, gpu_device))
    got = attn.run_decode(c["q"], c["cache"])
    c["indices"][1:27] = 0
    check(c, got)


@pytest.mark.parametrize("bits,page", [(16, 16), (16, 3), (4, 16), (4, 8)])
def test_device_tables_are_clamped(gpu_device, bits, page):
    """Bad tables on the device give some finite output, and touch nothing outside the pool."""
    c = case([40, 100, 70], 8, 2, 128, page, BF16, gpu_device, bits=bits, seed=15, poison=False)
    for name, value in (("indices", [2**31 - 1, -5] * 200), ("indptr", [-3, 1000, 2, 2**31 - 1]), ("last", [-1, 999, 2**31 - 1])):
        t = tables(c, gpu_device)
        key = {"indices": "paged_kv_indices", "indptr": "paged_kv_indptr", "last": "paged_kv_last_page_len"}[name]
        t[key] = torch.tensor(value, dtype=torch.int32, device=gpu_device)[: t[key].numel()]
        attn = attention(c)
        attn.plan_decode(**t)
        assert attn.run_decode(c["q"], c["cache"]).isfinite().all()


def test_batch_of_none(gpu_device):
    c = case([], 8, 2, 128, 16, BF16, gpu_device, seed=1)
    for on in (None, gpu_device):
        attn = attention(c)
        attn.plan_decode(**tables(c, on))
        assert attn.run_decode(c["q"], c["cache"]).shape == (0, 8, 128)


@pytest.mark.parametrize("bits", [16, 4])
def test_same_bits_every_time(gpu_device, bits):
    c = case([3000, 100, 5], 8, 2, 128, 16, BF16, gpu_device, bits=bits, seed=16)
    first = decode(c)
    for _ in range(3):
        again = decode(c)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


@pytest.mark.parametrize("bits", [16, 4])
def test_other_stream(gpu_device, bits):
    """A plan of one stream, runs on others; the plan's tables change at once afterwards."""
    c = case([300, 40], 8, 2, 128, 16, BF16, gpu_device, bits=bits, seed=17)
    attn = attention(c)
    t = tables(c, gpu_device)
    side, third = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)
        attn.plan_decode(**t)
        for x in t.values():
            x.zero_()
    with torch.cuda.stream(third):
        got = attn.run_decode(c["q"], c["cache"])
    torch.cuda.synchronize()
    check(c, got)


@pytest.mark.parametrize("bits", [16, 4])
def test_captured_plan_follows_its_tables(gpu_device, bits):
    """Plan and run in one graph: replays with longer sequences, eager work in between."""
    full = case([700, 90], 8, 2, 128, 16, BF16, gpu_device, bits=bits, window=50, sinks=3, seed=18, poison=False)
    attn = attention(full)
    t = tables(full, gpu_device)
    static = {k: v.clone() for k, v in t.items()}
    q = full["q"].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        attn.plan_decode(**static)
        out = attn.run_decode(q, full["cache"])
    with pytest.raises(RuntimeError, match="captured"):
        attn.run_decode(q, full["cache"])
    ids, ptr = full["indices"].tolist(), full["indptr"].tolist()
    for lens in ([700, 90], [1, 33], [650, 64], [0, 1], [700, 90]):
        pages = [-(-n // 16) for n in lens]
        rows = [ids[ptr[r]: ptr[r] + pages[r]] for r in range(2)]
        part = {**full, "lens": lens, "indptr": torch.tensor([0, pages[0], sum(pages)], dtype=torch.int32),
                "indices": torch.tensor(rows[0] + rows[1] + [0] * (len(ids) - sum(pages)), dtype=torch.int32),
                "last": torch.tensor([n - 16 * (p - 1) if p else 0 for n, p in zip(lens, pages)], dtype=torch.int32)}
        for k, v in tables(part).items():
            static[k].copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        check(part, out)
        eager = attention(part)
        eager.plan_decode(**tables(part, gpu_device))
        assert torch.equal(out, eager.run_decode(q, part["cache"]))


@pytest.mark.parametrize("bits", [16, 4])
def test_captured_runs_keep_their_plan(gpu_device, bits):
    """Two graphs on eager plans, other plans in between: each replays on its own."""
    a = case([300, 40], 8, 2, 128, 16, BF16, gpu_device, bits=bits, seed=19)
    b = case([77, 1000], 8, 2, 128, 16, BF16, gpu_device, bits=bits, seed=20)
    attn = attention(a)
    graphs = []
    for c in (a, b):
        attn.plan_decode(**tables(c))
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            graphs.append((c, g, attn.run_decode(c["q"], c["cache"])))
    for _ in range(3):
        for c, g, out in graphs:
            g.replay()
            attn.plan_decode(**tables(b))
            attn.run_decode(b["q"], b["cache"])
        torch.cuda.synchronize()
        for c, _, out in graphs:
            check(c, out)


def test_refusals(gpu_device):
    c = case([40, 30], 8, 2, 128, 16, BF16, gpu_device, seed=21)
    attn = attention(c)
    with pytest.raises(RuntimeError, match="plan_decode"):
        attn.run_decode(c["q"], c["cache"])
    attn.plan_decode(**tables(c))
    for q, cache, error in ((c["q"][:1], c["cache"], ValueError), (c["q"].float(), c["cache"], NotImplementedError),
                            (c["q"].half(), c["cache"], ValueError), (c["q"][:, :4], c["cache"], ValueError),
                            (c["q"], c["cache"][:, :1], ValueError), (c["q"], c["cache"][:4], ValueError),
                            (c["q"], c["cache"].view(torch.uint8), ValueError), (c["q"], c["cache"].cpu(), RuntimeError),
                            (c["q"].cpu(), c["cache"], RuntimeError)):
        with pytest.raises(error):
            attn.run_decode(q, cache)
    with pytest.raises(ValueError, match="lse"):
        attn.run_decode_into(c["q"], c["cache"], torch.empty_like(c["q"]), torch.empty(2, 8, dtype=BF16, device=gpu_device))
    with pytest.raises(ValueError, match="16 bytes"):
        attn.run_decode(torch.empty(2, 8, 132, dtype=BF16, device=gpu_device)[:, :, :128], c["cache"])
