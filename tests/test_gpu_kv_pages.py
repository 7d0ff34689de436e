"""Pages copied in every layer, bit for bit; forks, cuts and compaction of requests on the device."""

import pytest
import torch

from pagelora_amd import _lib
from pagelora_amd.kv_pool import PagedKVPool, Request, kv_copy_pages

pytestmark = pytest.mark.gpu


def random_cache(layers, pages, page, hkv, dim, dtype, device, seed=0):
    gen = torch.Generator(device=device).manual_seed(seed)
    return torch.randn((layers, pages, 2, page, hkv, dim), device=device, generator=gen).to(dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("page,hkv,dim", [(16, 8, 128), (1, 1, 8), (5, 3, 24), (64, 8, 128)])
@pytest.mark.parametrize("n", [1, 7, 449, 1000])
def test_copy(gpu_device, dtype, page, hkv, dim, n):
    """Pages of less than one workgroup's bytes and of many, more pages than one launch names, sources listed twice."""
    if n > 7 and page == 64:
        n = 30
    cache = random_cache(3, 2 * n + 1, page, hkv, dim, dtype, gpu_device)
    ids = torch.randperm(2 * n + 1, generator=torch.Generator().manual_seed(n)).tolist()
    src, dst = ids[:n], ids[n: 2 * n]
    src[-1] = src[0]
    want = cache.clone()
    want[:, dst] = cache[:, src]
    kv_copy_pages(cache, src, dst)
    torch.cuda.synchronize()
    assert torch.equal(cache, want)


def test_copy_in_views_and_graphs(gpu_device):
    """A pool that is a slice of layers and pages of a larger one; one layer; a captured copy names its pages itself."""
    room = random_cache(4, 40, 16, 2, 64, torch.bfloat16, gpu_device)
    want = room.clone()
    view = room[1:3, 5:30]
    kv_copy_pages(view, [3, 4], [20, 0])
    want[1:3, 25], want[1:3, 5] = want[1:3, 8], want[1:3, 9]
    assert torch.equal(room, want)
    kv_copy_pages(room[0], (1,), (2,))
    want[0, 2] = want[0, 1]
    assert torch.equal(room, want)
    src, dst = [7, 8, 9], [17, 18, 19]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kv_copy_pages(room, src, dst)
    src[:], dst[:] = [0, 0, 0], [1, 1, 1]
    for i in range(3):
        room[:, 7:10].normal_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(room[:, 17:20], room[:, 7:10]), i


def test_copy_past_4_gib(gpu_device):
    pages = 2**32 // (2 * 16 * 8 * 128 * 2) + 5
    cache = torch.zeros((1, pages, 2, 16, 8, 128), dtype=torch.bfloat16, device=gpu_device)
    cache[0, pages - 1].normal_()
    kv_copy_pages(cache, [pages - 1, 0], [1, pages - 2])
    assert torch.equal(cache[0, 1], cache[0, pages - 1]) and not cache[0, pages - 2].any() and not cache[0, 2].any()


def test_refusals(gpu_device):
    cache = random_cache(2, 8, 16, 2, 64, torch.bfloat16, gpu_device)
    before = cache.clone()
    for src, dst, what in (([1], [1], "also a source"), ([1, 2], [3, 3], "written twice"), ([1, 2], [2, 3], "also a source"),
                           ([8], [1], "outside the 8-page"), ([1], [-1], "outside the 8-page"), ([1], [2**40], "integers"), ([1, 2], [3], "destination"),
                           ([1.0], [2.0], "integers")):
        with pytest.raises(ValueError, match=what):
            kv_copy_pages(cache, src, dst)
    with pytest.raises(ValueError, match="contiguous"):
        kv_copy_pages(cache.transpose(3, 4), [1], [2])
    with pytest.raises(ValueError, match="cache must be"):
        kv_copy_pages(cache[0, 0], [1], [2])
    with pytest.raises(NotImplementedError):
        kv_copy_pages(cache.double(), [1], [2])
    many = list(range(1, 60))
    big = random_cache(1, 130, 1, 1, 8, torch.bfloat16, gpu_device)
    for dst, what in ((many, "also a source"), ([60 + i // 2 for i in range(59)], "written twice")):
        with pytest.raises(ValueError, match=what):
            kv_copy_pages(big, many, dst)
    kv_copy_pages(cache, [], [])
    torch.cuda.synchronize()
    assert torch.equal(cache, before)


def test_fork_truncate_compact(gpu_device):
    """Every request's tokens read back through its page list stay what they were."""
    pool = PagedKVPool(num_layers=3, capacity_pages=40, page_size=4, num_kv_heads=2, head_dim=8, dtype=torch.float32,
                       device=gpu_device)
    pool.cache.normal_()
    prefix = pool.allocator.allocate(2)
    a, b = Request(list(prefix), 8, [], 8), Request()
    pool.reserve(a, 9)
    pool.reserve(b, 12)
    c, d, e = pool.fork([a, b, a])

    def read(r):
        pages = torch.tensor(r.pages(), device=gpu_device)
        return pool.cache[:, pages].transpose(2, 3).flatten(1, 2)[:, : r.length].clone()

    text = {id(r): read(r) for r in (a, b, c, d, e)}
    assert torch.equal(text[id(a)], text[id(c)]) and torch.equal(text[id(b)], text[id(d)])
    assert len({a.own_pages[-1], c.own_pages[-1], e.own_pages[-1]}) == 3 and d.own_pages == b.own_pages
    pool.truncate(d, 6)   # its last page was shared with b
    assert d.own_pages[0] == b.own_pages[0] and d.own_pages[1] != b.own_pages[1] and len(d.own_pages) == 2
    assert torch.equal(read(d), text[id(b)][:, :6]) and torch.equal(read(b), text[id(b)])
    pool.reserve(d, 3)
    pages = torch.tensor(d.pages(), device=gpu_device)
    pool.cache[:, pages[1]] = 7.0
    assert torch.equal(read(b), text[id(b)])
    pool.release(a)
    others = {id(r): read(r) for r in (b, c, d, e)}
    assert torch.equal(others[id(c)], text[id(c)])
    moved = pool.compact([b, c, d, e])
    assert moved and all(new < old for old, new in moved.items())
    for r in (b, c, d, e):
        assert torch.equal(read(r), others[id(r)])
    assert c.prefix_pages == prefix
    for r in (b, c, d, e):
        pool.release(r)
    pool.allocator.free(prefix)
    assert sorted(pool.allocator._free) == list(range(1, 40)) and not pool.allocator._more


def test_c_entry_refuses_what_it_cannot_copy(gpu_device):
    lib = _lib.load()
    cache = random_cache(1, 4, 16, 2, 64, torch.bfloat16, gpu_device)
    import numpy as np

    src, dst = np.array([1], np.int32), np.array([9], np.int32)
    call = lambda ps, n: lib.pl_kv_copy_pages(cache.data_ptr(), cache.stride(0), ps, cache.stride(1), 1, 4,  # noqa: E731
                                              src.ctypes.data, dst.ctypes.data, n, _lib.PL_DTYPE_BF16, None)
    assert call(cache.stride(1), 1) == _lib.PL_ERR_INVALID and "outside" in _lib.last_error()
    assert call(cache.stride(1) // 2, 1) == _lib.PL_ERR_INVALID and "overlap" in _lib.last_error()
    assert call(cache.stride(1), -1) == _lib.PL_ERR_INVALID
