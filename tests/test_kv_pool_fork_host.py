"""Forks, cuts and compaction of requests: the page lists and holders (host logic; the copies are recorded)."""

import pytest
import torch

from pagelora_amd.kv_pool import PageAllocator, PagedKVPool, Request, kv_copy_pages


@pytest.fixture
def pool(monkeypatch):
    p = PagedKVPool(num_layers=1, capacity_pages=20, page_size=4, num_kv_heads=1, head_dim=8, dtype=torch.float32,
                    device="cpu", max_pages=None)
    p.copies = []
    monkeypatch.setattr(p, "copy_pages", lambda src, dst: p.copies.extend(zip(src, dst)))
    return p


def request(pool, n, prefix=()):
    r = Request(list(prefix), len(prefix) * 4, [], len(prefix) * 4)
    pool.reserve(r, n)
    return r


def test_fork_shares_full_pages_and_copies_the_partial_one(pool):
    r = request(pool, 10)
    f, g = pool.fork([r, r])
    assert f.own_pages[:2] == g.own_pages[:2] == r.own_pages[:2] and f.length == 10
    assert len({r.own_pages[2], f.own_pages[2], g.own_pages[2]}) == 3
    assert pool.copies == [(r.own_pages[2], f.own_pages[2]), (r.own_pages[2], g.own_pages[2])]
    assert [pool.allocator.holders(p) for p in r.own_pages] == [3, 3, 1]


def test_fork_at_a_page_border_copies_nothing(pool):
    r = request(pool, 8)
    (f,) = pool.fork([r])
    assert f.own_pages == r.own_pages and f.own_pages is not r.own_pages and not pool.copies
    pool.reserve(f, 1)
    assert len(f.own_pages) == 3 and len(r.own_pages) == 2


def test_fork_of_nothing_and_of_a_prefix_alone(pool):
    prefix = pool.allocator.allocate(2)
    empty, only = pool.fork([Request(), Request(list(prefix), 8, [], 8)])
    assert empty.pages() == [] and only.pages() == prefix and only.prefix_len == 8 and not pool.copies


def test_a_page_is_free_with_its_last_holder(pool):
    r = request(pool, 8)
    free = pool.allocator.free_pages
    (f,) = pool.fork([r])
    pages = list(r.own_pages)
    pool.release(r)
    assert pool.allocator.free_pages == free and pool.allocator.holders(pages[0]) == 1
    pool.release(f)
    assert pool.allocator.free_pages == free + 2 and not pool.allocator._more


def test_fork_without_room_changes_nothing(pool):
    r = request(pool, 4 * 18 + 1)  # all 19 pages
    with pytest.raises(RuntimeError, match="exhausted"):
        pool.fork([r])
    assert pool.allocator.holders(r.own_pages[0]) == 1 and not pool.copies


def test_fork_whose_copy_fails_gives_its_pages_back(pool, monkeypatch):
    r = request(pool, 6)
    free = pool.allocator.free_pages
    monkeypatch.setattr(pool, "copy_pages", lambda s, d: kv_copy_pages(pool.cache, s, d))
    with pytest.raises(RuntimeError, match="ROCm device"):
        pool.fork([r])
    assert pool.allocator.free_pages == free and pool.allocator.holders(r.own_pages[0]) == 1


def test_truncate_frees_the_pages_behind(pool):
    r = request(pool, 15)
    pages, free = list(r.own_pages), pool.allocator.free_pages
    pool.truncate(r, 15)
    assert r.own_pages == pages
    pool.truncate(r, 5)
    assert r.own_pages == pages[:2] and r.length == 5 and pool.allocator.free_pages == free + 2 and not pool.copies
    pool.truncate(r, 0)
    assert r.own_pages == [] and pool.allocator.free_pages == free + 4


def test_truncate_copies_a_shared_page_it_will_write_to(pool):
    r = request(pool, 8)
    (f,) = pool.fork([r])
    pool.truncate(f, 6)
    assert f.own_pages[0] == r.own_pages[0] and f.own_pages[1] != r.own_pages[1]
    assert pool.copies == [(r.own_pages[1], f.own_pages[1])]
    assert pool.allocator.holders(r.own_pages[1]) == 1 and pool.allocator.holders(r.own_pages[0]) == 2
    pool.truncate(f, 4)  # a full page may stay shared
    assert f.own_pages == r.own_pages[:1] and len(pool.copies) == 1


def test_truncate_refuses_other_lengths(pool):
    prefix = pool.allocator.allocate(1)
    r = request(pool, 3, prefix)
    for n in (8, 3, -1):
        with pytest.raises(ValueError, match="outside"):
            pool.truncate(r, n)


def test_compact_moves_pages_down_and_keeps_foreign_holders_in_place(pool):
    a, b, c = request(pool, 8), request(pool, 8), request(pool, 8)  # pages 1..6
    (d,) = pool.fork([c])                                          # holds 5, 6 too
    shared = Request(list(b.own_pages), 8, [], 8)                  # b's pages as its prefix
    pool.release(a)
    moved = pool.compact([b, shared, c])                            # c's pages have a holder (d) that is not named
    assert moved == {4: 1, 3: 2} and pool.copies == [(4, 1), (3, 2)]
    assert b.own_pages == [2, 1] and shared.prefix_pages == [2, 1] and c.own_pages == d.own_pages == [5, 6]
    moved = pool.compact([b, shared, c, d, c])
    assert moved == {6: 3, 5: 4} and c.own_pages == d.own_pages == [4, 3] and pool.allocator.holders(3) == 2
    assert pool.allocator.allocate(1) == [5]
    assert pool.compact([b, c, d]) == {}


def test_allocator_free_without_share_is_as_before():
    a = PageAllocator(4)
    first = a.allocate(3)
    a.free(first)
    assert sorted(a._free) == [1, 2, 3] and a.holders(2) == 1
