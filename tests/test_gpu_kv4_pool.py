"""Requests of a 4-bit pool are cut back and moved, and read as they did."""

import pytest
import torch

from pagelora_amd.kv4 import kv4_append, kv4_read
from pagelora_amd.kv_pool import PagedKVPool, Request

pytestmark = pytest.mark.gpu

SIZE = dict(num_kv_heads=2, head_dim=64, page_size=8)


def a_pool(device, capacity=24):
    pool = PagedKVPool(num_layers=2, capacity_pages=capacity, dtype=torch.bfloat16, device=device, kv_bits=4, **SIZE)
    pool.cache.random_(0, 256)
    return pool


def slots(pool, request, start=0):
    where = [request.slot(p, 8) for p in range(start, request.length)]
    return (torch.tensor([w[i] for w in where], dtype=torch.int64, device=pool.cache.device) for i in (0, 1))


def append(pool, request, tokens, gen):
    start = request.length
    pool.reserve(request, tokens)
    for layer in range(2):
        k, v = (torch.randn((tokens, 2, 64), generator=gen).to(pool.cache.device, torch.bfloat16) for _ in range(2))
        kv4_append(pool.cache[layer], k, v, *slots(pool, request, start), **SIZE)


def read(pool, request):
    return [x for layer in range(2) for x in kv4_read(pool.cache[layer], *slots(pool, request), **SIZE)]


def same(a, b, tokens):
    return all(torch.equal(x[:tokens], y[:tokens]) for x, y in zip(a, b))


@pytest.mark.parametrize("length", [30, 24, 17, 1])
def test_truncate(gpu_device, length):
    """A fork cut back and appended to writes to a page of its own, also within a group of four tokens."""
    pool, gen = a_pool(gpu_device), torch.Generator().manual_seed(length)
    a = Request()
    append(pool, a, 30, gen)
    before = read(pool, a)
    assert not any(x.isnan().any() for x in before)
    b, = pool.fork([a])
    pool.truncate(b, length)
    assert same(read(pool, b), before, length) and len(b.own_pages) == -(-length // 8)
    append(pool, b, 11, gen)
    after = read(pool, b)
    assert same(after, before, length) and not any(x.isnan().any() for x in after)
    assert same(read(pool, a), before, 30)
    append(pool, a, 5, gen)
    assert same(read(pool, b), after, length + 11) and same(read(pool, a), before, 30)


def test_compact(gpu_device):
    """Pages go to the lowest ids, a shared one once for both holders."""
    pool, gen = a_pool(gpu_device), torch.Generator().manual_seed(2)
    requests = [Request() for _ in range(4)]
    for turn in range(3):
        for r in requests:
            append(pool, r, 9 + turn, gen)
    fork, = pool.fork([requests[3]])
    append(pool, fork, 3, gen)
    left = [requests[1], requests[3], fork]
    before = [read(pool, r) for r in left]
    pool.release(requests[0])
    pool.release(requests[2])
    moved = pool.compact(left)
    pages = {p for r in left for p in r.own_pages}
    assert moved and max(pages) == len(pages)  # (page 0 is never handed out)
    assert all(same(read(pool, r), b, r.length) for r, b in zip(left, before))
    for r in left:
        append(pool, r, 4, gen)
    assert all(same(read(pool, r), b, r.length - 4) for r, b in zip(left, before))
