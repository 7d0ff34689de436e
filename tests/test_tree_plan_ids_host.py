"""What pl_tree_plan_ids refuses before any launch (pointers are never read)."""

import pytest

from pagelora_amd import _lib

PTR = 4096  # aligned, never dereferenced


def plan(**kw):
    a = dict(qo=PTR, kv=PTR, ind=PTR, n=3, last=PTR, batch=2, tokens=3, max_tree=2, parents=PTR, mask=None, ld=0, hq=4,
             hkv=2, d=64, page=16, share=0, ids=PTR, cap=16, buf=PTR, size=1 << 30, stream=None)
    return _lib.load().pl_tree_plan_ids(*{**a, **kw}.values())


@pytest.mark.parametrize("kw,status", [
    (dict(n=17), 1), (dict(n=-1), 1), (dict(ids=None), 1), (dict(ids=PTR + 2), 1), (dict(cap=2), 1), (dict(buf=None), 1),
    (dict(buf=PTR + 8), 1), (dict(batch=-1), 1), (dict(d=96), 2), (dict(mask=PTR, ld=4), 1), (dict(size=64), 3),
])
def test_pl_tree_plan_ids_refuses(kw, status):
    assert plan(**kw) == status and _lib.last_error()


def test_a_plan_buffer_of_no_ids_is_the_same_for_every_length():
    lib = _lib.load()
    size = lib.pl_tree_plan_size(2, 3, 2, 0, 4, 2, 64)
    assert plan(size=size - 1) == 3 and lib.pl_tree_plan_size(2, 3, 2, 1000, 4, 2, 64) >= size + 4000


def test_pl_tree_plan_ids_of_nothing():
    assert plan(batch=0, qo=None, buf=None) == 0 and plan(tokens=0, max_tree=0, buf=None) == 0
