"""Prefill attention under a window with sinks, over 16-bit and 4-bit caches, against 64 bits."""

import numpy as np
import pytest
import torch

from tests.window_cases import BF16, F16, attention, case, check, prefill, reference, set_cache, tables

pytestmark = pytest.mark.gpu

# (tokens, queries) of each request
RAGGED = [(1, 1), (0, 0), (5, 0), (17, 17), (40, 3), (64, 64), (65, 1), (130, 129), (300, 33)]


def ragged(requests, *args, **kw):
    return case([n for n, _ in requests], *args, new=[m for _, m in requests], **kw)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("heads", [(1, 1), (8, 2), (7, 1), (33, 1)])
@pytest.mark.parametrize("head_dim", [64, 128])
def test_heads(gpu_device, dtype, bits, heads, head_dim):
    c = ragged(RAGGED, *heads, head_dim, 16, dtype, gpu_device, bits=bits, window=50, sinks=5, seed=3)
    check(c, prefill(c))


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("window,sinks", [(0, 0), (0, 7), (1, 0), (1, 1), (5, 0), (63, 4), (64, 64), (65, 65), (100, 200),
                                          (200, 1), (2**31 - 1, 2**31 - 1), (7, 2**31 - 1)])
def test_windows(gpu_device, bits, window, sinks):
    c = ragged(RAGGED + [(400, 200)], 4, 2, 128, 16, BF16, gpu_device, bits=bits, window=window, sinks=sinks, seed=window % 97)
    check(c, prefill(c))


@pytest.mark.parametrize("bits,page", [(16, 1), (16, 3), (16, 4), (16, 7), (16, 32), (16, 48), (16, 1024), (4, 8), (4, 24),
                                       (4, 32), (4, 40), (4, 48), (4, 1024)])
@pytest.mark.parametrize("head_dim", [64, 128])
def test_pages(gpu_device, bits, page, head_dim):
    c = ragged(RAGGED, 4, 2, head_dim, page, F16, gpu_device, bits=bits, window=70, sinks=33, seed=page)
    check(c, prefill(c))


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("requests,window,sinks", [([(3000, 5)], 0, 0), ([(3000, 40), (700, 3)], 0, 0), ([(4000, 9)], 2500, 70),
                                                   ([(1500, 2)] * 3, 0, 0)])
def test_split_ranges(gpu_device, bits, requests, window, sinks):
    """Few queries behind many tokens: the kv ranges are cut and joined."""
    c = ragged(requests, 4, 1, 128, 16, BF16, gpu_device, bits=bits, window=window, sinks=sinks, seed=7)
    check(c, prefill(c))


@pytest.mark.parametrize("dtype,bits", [(BF16, 16), (F16, 16), (BF16, 4), (F16, 4)])
def test_scores_far_apart(gpu_device, dtype, bits):
    c = ragged([(300, 260)], 2, 1, 128, 16, dtype, gpu_device, bits=bits, seed=8, q_scale=30.0)
    check(c, prefill(c))


def test_large_values_stay_finite(gpu_device):
    for bits in (16, 4):
        c = ragged([(300, 20)], 4, 1, 128, 16, BF16, gpu_device, bits=bits, seed=2, poison=False)
        cache = torch.randn((c["indices"].numel() + 3, 2, 16, 1, 128), generator=torch.Generator().manual_seed(1))
        cache[:, 1] = 2.5e38
        set_cache(c, cache.to(BF16))
        check(c, prefill(c))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("window,sinks", [(0, 0), (30, 2)])
@pytest.mark.parametrize("requests", [[(200, 150)], [(2000, 6)]])
def test_infinities_and_nan_in_v(gpu_device, dtype, window, sinks, requests):
    """In tokens that some of the rows of a tile see and others do not: theirs alone, with their sign."""
    n, new = requests[0]
    c = ragged(requests, 4, 2, 128, 16, dtype, gpu_device, window=window, sinks=sinks, seed=5, poison=False)
    cache = torch.from_numpy(c["cache_host"]).to(dtype)
    for i, t in enumerate([0, 1, n - new // 2 - 40, n - new // 2, n - 2, n - 1]):
        page, off = int(c["indices"][t // 16]), t % 16
        cache[page, 1, off, 0, 3 + i] = float("inf")
        cache[page, 1, off, 0, 40 + i] = -float("inf")
        cache[page, 1, off, 1, 60] = float("inf") if i % 2 else -float("inf")
        cache[page, 1, off, 1, 100 + i] = float("nan")
    set_cache(c, cache)
    o = reference(c)[0]
    assert np.isinf(o).any() and np.isnan(o).any() and np.isfinite(o).any()
    check(c, prefill(c))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("requests", [[(200, 150), (70, 70)], [(2000, 6)]])
@pytest.mark.parametrize("k_power,v_power", [(0, -30), (0, 20), (0, -100), (0, 100), (0, 3), (0, -17), (-17, 0), (-30, 0), (12, 0)])
def test_scales_of_a_4_bit_cache(gpu_device, dtype, requests, k_power, v_power):
    """K or V of a few tokens, or of a dim group of all, far outside fp16's range and about its ends: as exact as others."""
    c = ragged(requests, 4, 2, 128, 16, dtype, gpu_device, bits=4, seed=6, poison=False)
    cache = torch.randn((c["indices"].numel() + 3, 2, 16, 2, 128), generator=torch.Generator().manual_seed(1))
    cache[:, 0, :, :, 64:96] *= 2.0 ** k_power
    cache[:, 1, :, 1, 32:64] *= 2.0 ** v_power
    cache[int(c["indices"][2]), 1, 3, 0] *= 2.0 ** v_power
    set_cache(c, cache.to(BF16))
    if k_power > 0:  # (scores of a usual size)
        c["q_host"][..., 64:96] /= 2.0 ** k_power
        c["q"] = c["q_host"].to(gpu_device)
    check(c, prefill(c))


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_head_dims_that_only_pad(gpu_device, dtype):
    """96 dims in 128: groups of zeros in q, K and V, and a V token of zeros."""
    c = ragged([(200, 150), (2000, 6)], 4, 2, 128, 16, dtype, gpu_device, bits=4, seed=6, poison=False)
    cache = torch.randn((c["indices"].numel() + 3, 2, 16, 2, 128), generator=torch.Generator().manual_seed(1))
    cache[..., 96:] = 0.0
    cache[int(c["indices"][2]), 1, 3] = 0.0
    set_cache(c, cache.to(BF16))
    out = prefill(c)
    check(c, out)
    assert (out[..., 96:] == 0).all()


@pytest.mark.parametrize("window,sinks", [(0, 0), (30, 2)])
def test_nan_groups_of_a_4_bit_cache(gpu_device, window, sinks):
    c = ragged([(200, 150)], 4, 2, 128, 16, BF16, gpu_device, bits=4, window=window, sinks=sinks, seed=5, poison=False)
    cache = torch.randn((c["indices"].numel() + 3, 2, 16, 2, 128), generator=torch.Generator().manual_seed(1)).to(BF16)
    for t in (0, 100, 199):
        cache[int(c["indices"][t // 16]), 1, t % 16, 1, 33] = float("nan")
    set_cache(c, cache)
    nan = np.isnan(reference(c)[0])
    assert nan.any() and not nan.all()
    check(c, prefill(c))


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("scale", [-0.2, 0.0, 3.0])
def test_softmax_scale(gpu_device, bits, scale):
    c = ragged(RAGGED, 4, 2, 128, 16, F16, gpu_device, bits=bits, window=64, sinks=4, seed=11)
    attn = attention(c)
    attn.sm_scale = scale
    attn.plan_prefill(qo_indptr=c["qo_indptr"], **tables(c, gpu_device))
    check(c, attn.run_prefill(c["q"], c["cache"]), sm_scale=scale)


@pytest.mark.parametrize("bits", [16, 4])
def test_strides(gpu_device, bits):
    c = ragged([(40, 7), (300, 130)], 8, 2, 128, 16, BF16, gpu_device, bits=bits, window=64, sinks=4, seed=12)
    attn = attention(c)
    attn.plan_prefill(qo_indptr=c["qo_indptr"], **tables(c))
    n = c["q"].shape[0]
    wide = torch.full((n, 12, 136), float("nan"), dtype=BF16, device=gpu_device)
    wide[:, 2:10, :128] = c["q"]
    out = torch.full((n, 20, 128), 7.0, dtype=BF16, device=gpu_device)
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
        attn.run_prefill_into(wide[:, 2:10, :128], cache, out[:, 5:13])
        check(c, out[:, 5:13])
        assert (out[:, :5] == 7).all() and (out[:, 13:] == 7).all()


@pytest.mark.parametrize("bits", [16, 4])
def test_pool_past_4_gib(gpu_device, bits):
    c = ragged([(100, 40)], 4, 2, 128, 16, BF16, gpu_device, bits=bits, seed=13, extra=0)
    n, per = c["cache"].shape[0], c["cache"][0].numel()
    apart = (5 << 30) // c["cache"].element_size() // n // 64 * 64
    memory = torch.empty(apart * n + per, dtype=c["cache"].dtype, device=gpu_device)
    cache = memory.as_strided(c["cache"].shape, (apart, *c["cache"].stride()[1:]))
    cache.copy_(c["cache"])
    c["cache"] = cache
    check(c, prefill(c))


def test_tokens_far_apart(gpu_device):
    """A page's 16 tokens over more than 4 GiB."""
    c = ragged([(30, 20)], 4, 2, 128, 16, BF16, gpu_device, seed=13, extra=0)
    apart = 150 << 20  # values
    memory = torch.empty(16 * apart, dtype=BF16, device=gpu_device)
    cache = memory.as_strided(c["cache"].shape, (1024, 512, apart, 128, 1))
    cache.copy_(c["cache"])
    c["cache"] = cache
    check(c, prefill(c))


def test_many_requests(gpu_device):
    """More records than a plan has room for at first."""
    c = ragged([(3, 1), (20, 2)] * 600, 1, 1, 64, 16, BF16, gpu_device, bits=4, window=9, sinks=1, seed=3)
    check(c, prefill(c))


def test_no_queries(gpu_device):
    for requests in ([], [(5, 0), (0, 0)]):
        c = ragged(requests, 8, 2, 128, 16, BF16, gpu_device, seed=1)
        assert prefill(c).shape == (0, 8, 128)


@pytest.mark.parametrize("bits", [16, 4])
def test_agrees_with_decode(gpu_device, bits):
    """The last queries of prompts, alone and among the others."""
    c = ragged([(70, 70), (300, 2), (1, 1)], 8, 2, 128, 16, BF16, gpu_device, bits=bits, window=40, sinks=4, seed=14, poison=False)
    out = prefill(c)
    attn = attention(c)
    attn.plan_decode(**tables(c))
    ends = c["qo_indptr"][1:].long() - 1
    got = attn.run_decode(c["q"][ends.to(gpu_device)], c["cache"])
    tol = reference(c)[2] + reference({**c, "prefill": False})[2]
    assert (np.abs((out[ends.to(gpu_device)].double() - got.double()).cpu().numpy()) <= tol[ends.numpy()]).all()


@pytest.mark.parametrize("bits", [16, 4])
def test_streams_and_capture(gpu_device, bits):
    c = ragged([(300, 129), (2000, 3)], 4, 1, 128, 16, BF16, gpu_device, bits=bits, seed=15)
    attn = attention(c)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)
        attn.plan_prefill(qo_indptr=c["qo_indptr"], **tables(c))
    got = attn.run_prefill(c["q"], c["cache"])
    torch.cuda.synchronize()
    check(c, got)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = attn.run_prefill(c["q"], c["cache"])
    other = ragged([(64, 64)], 4, 1, 128, 16, BF16, gpu_device, bits=bits, seed=16)
    attn.plan_prefill(qo_indptr=other["qo_indptr"], **tables(other))
    for _ in range(3):
        out.zero_()
        check(other, attn.run_prefill(other["q"], other["cache"]))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, got)


def test_refusals(gpu_device):
    c = ragged([(40, 3)], 8, 2, 128, 16, BF16, gpu_device, seed=21)
    attn = attention(c)
    with pytest.raises(RuntimeError, match="plan_prefill"):
        attn.run_prefill(c["q"], c["cache"])
    attn.plan_prefill(qo_indptr=c["qo_indptr"], **tables(c))
    for q, cache, error in ((c["q"][:1], c["cache"], ValueError), (c["q"].float(), c["cache"], NotImplementedError),
                            (c["q"].half(), c["cache"], ValueError), (c["q"][:, :4], c["cache"], ValueError),
                            (c["q"], c["cache"][:, :1], ValueError), (c["q"], c["cache"][:3], ValueError),
                            (c["q"], c["cache"].cpu(), RuntimeError), (c["q"].cpu(), c["cache"], RuntimeError)):
        with pytest.raises(error):
            attn.run_prefill(q, cache)
