"""What plan_tree and the tree's C entries refuse before any launch (host checks only; pointers are never read)."""

import ctypes

import pytest
import torch

from pagelora_amd import _lib
from pagelora_amd.attention_backend import PagedDecodeAttention

PTR = 4096  # aligned, never dereferenced


def i32(*x):
    return torch.tensor(x, dtype=torch.int32)


def good():
    return dict(qo_indptr=i32(0, 2, 3), paged_kv_indptr=i32(0, 1, 3), paged_kv_indices=i32(4, 2, 7),
                paged_kv_last_page_len=i32(5, 1), tree_parents=i32(-1, 0, -1))


@pytest.mark.parametrize("name,value,what", [
    ("qo_indptr", i32(0, 2), "batch \\+ 1"), ("qo_indptr", i32(1, 2, 3), "qo_indptr"), ("qo_indptr", i32(0, 3, 2), "qo_indptr"),
    ("qo_indptr", i32(0, 2, 2), "ends at"), ("qo_indptr", i32(0, 2, 3).long(), "int32"),
    ("paged_kv_indptr", i32(0, 2, 1), "non-decreasing"), ("paged_kv_indptr", i32(0, 1, 4), "exceeds"),
    ("paged_kv_indptr", i32(0, 0, 2), "exceeds its 0 tokens"), ("paged_kv_indices", i32(4, -2, 7), "negative"),
    ("paged_kv_last_page_len", i32(1, 1), "exceeds its 1 tokens"), ("paged_kv_last_page_len", i32(5, 17), "outside"),
    ("tree_parents", i32(-1, 1, -1), "earlier nodes"), ("tree_parents", i32(-1, 0, 0), "earlier nodes"),
    ("tree_parents", i32(-2, 0, -1), "earlier nodes"), ("tree_parents", None, "not both"),
    ("tree_parents", torch.zeros((3, 1), dtype=torch.int32), "1-D"), ("tree_mask", torch.ones((3, 2), dtype=torch.bool), "not both"),
    ("max_tree", 1, "exceeds max_tree"),
])
def test_plan_tree_refuses(name, value, what):
    be = PagedDecodeAttention(device="cpu", workspace_mb=1, num_qo_heads=4, num_kv_heads=2, head_dim=64, page_size=16)
    with pytest.raises(ValueError, match=what):
        be.plan_tree(**{**good(), name: value})


@pytest.mark.parametrize("mask,what", [
    (torch.ones(3, dtype=torch.bool), "2-D"), (torch.ones((3, 2)), "bool or uint8"),
    (torch.ones((3, 1), dtype=torch.bool), "columns"), (torch.ones((2, 2), dtype=torch.bool), "ends at"),
])
def test_plan_tree_refuses_masks(mask, what):
    be = PagedDecodeAttention(device="cpu", workspace_mb=1, num_qo_heads=4, num_kv_heads=2, head_dim=64, page_size=16)
    with pytest.raises(ValueError, match=what):
        be.plan_tree(**{**good(), "tree_parents": None}, tree_mask=mask)


def test_plan_tree_needs_a_device():
    be = PagedDecodeAttention(device="cpu", workspace_mb=1, num_qo_heads=4, num_kv_heads=2, head_dim=64, page_size=16)
    with pytest.raises(RuntimeError, match="ROCm device"):
        be.plan_tree(**good())


def plan(**kw):
    a = dict(qo=PTR, kv=PTR, ind=PTR, n=3, last=PTR, batch=2, tokens=3, max_tree=2, parents=PTR, mask=None, ld=0, hq=4,
             hkv=2, d=64, page=16, share=0, cap=16, buf=PTR, size=1 << 30, stream=None)
    return _lib.load().pl_tree_plan(*{**a, **kw}.values())


@pytest.mark.parametrize("kw,status", [
    (dict(batch=-1), 1), (dict(tokens=-1), 1), (dict(hkv=3), 1), (dict(hkv=0), 1), (dict(d=96), 2), (dict(page=0), 1),
    (dict(page=65537), 1), (dict(batch=4097), 2), (dict(max_tree=4), 1), (dict(tokens=1 << 27, hq=4), 2), (dict(n=17), 1),
    (dict(n=-1), 1), (dict(qo=None), 1), (dict(buf=None), 1), (dict(ind=None), 1), (dict(mask=PTR, ld=4), 1),
    (dict(parents=None), 1), (dict(parents=None, mask=PTR, ld=1), 1), (dict(share=-1), 1),
    (dict(buf=PTR + 8), 1), (dict(size=64), 3),
])
def test_pl_tree_plan_refuses(kw, status):
    assert plan(**kw) == status and _lib.last_error()


def test_pl_tree_plan_of_nothing():
    assert plan(batch=0, qo=None, buf=None) == 0 and plan(tokens=0, max_tree=0, buf=None) == 0


def run(**kw):
    a = dict(q=PTR, qt=256, qh=64, k=PTR, v=PTR, ps=4096, ts=128, hs=64, pages=9, o=PTR, ot=256, oh=64, lse=None, batch=2,
             tokens=3, max_tree=2, hq=4, hkv=2, d=64, page=16, scale=0.125, dtype=2, plan=PTR, pbytes=1 << 30, cap=16,
             ws=PTR, wbytes=1 << 34, stream=None)
    return _lib.load().pl_tree_run(*{**a, **kw}.values())


@pytest.mark.parametrize("kw,status", [
    (dict(dtype=0), 2), (dict(dtype=9), 2), (dict(d=32), 2), (dict(q=None), 1), (dict(o=None), 1), (dict(plan=None), 1),
    (dict(ws=None), 1), (dict(pages=0), 1), (dict(qt=252), 1), (dict(hs=4), 1), (dict(ot=254), 1), (dict(q=PTR + 8), 1),
    (dict(o=PTR + 4), 1), (dict(pbytes=64), 3), (dict(wbytes=64), 3), (dict(batch=-1), 1),
])
def test_pl_tree_run_refuses(kw, status):
    assert run(**kw) == status and _lib.last_error()


def test_pl_tree_run_of_nothing():
    assert run(batch=0, q=None) == 0 and run(tokens=0, max_tree=0, q=None) == 0


def test_sizes_hold_what_is_planned():
    lib = _lib.load()
    # header, masks and indices at the least; two partial results of each of 256 slots
    assert lib.pl_tree_plan_size(64, 1024, 16, 40000, 32, 8, 128) >= 64 + 1024 * 8 + 40000 * 4
    assert lib.pl_tree_workspace_size(1, 8, 8, 32, 8, 128) >= 2 * 256 * 32 * 130 * 4
    assert lib.pl_tree_plan_size(1, 8, 8, 16, 32, 8, 96) == 0 and lib.pl_tree_workspace_size(1, 8, 9, 32, 8, 128) == 0


def accept(**kw):
    a = dict(tokens=PTR, parents=PTR, picks=PTR, qo=PTR, batch=2, n=3, max_path=4, path=PTR, count=PTR, kept=PTR, stream=None)
    return _lib.load().pl_tree_accept(*{**a, **kw}.values())


def test_pl_tree_accept_refuses():
    for kw in (dict(batch=-1), dict(n=-1), dict(max_path=0), dict(tokens=None), dict(path=None), dict(qo=None)):
        assert accept(**kw) == _lib.PL_ERR_INVALID and _lib.last_error()
    assert accept(batch=0, qo=None) == 0


def commit(**kw):
    a = dict(k=PTR, v=PTR, ls=1 << 20, ps=4096, ts=128, hs=64, layers=2, pages=9, qo=PTR, kv=PTR, ind=PTR, n=3, last=PTR,
             path=PTR, count=PTR, batch=2, max_path=4, hkv=2, d=64, page=16, dtype=2, stream=None)
    return _lib.load().pl_tree_commit(*{**a, **kw}.values())


def test_pl_tree_commit_refuses():
    for kw in (dict(batch=-1), dict(layers=-1), dict(hkv=0), dict(d=4), dict(max_path=0), dict(pages=0), dict(page=0),
               dict(k=None), dict(path=None), dict(ts=4), dict(k=PTR + 8)):
        assert commit(**kw) == _lib.PL_ERR_INVALID and _lib.last_error()
    assert commit(dtype=7) == _lib.PL_ERR_UNSUPPORTED and commit(batch=65536) == _lib.PL_ERR_UNSUPPORTED
    assert commit(batch=0, qo=None) == 0 and commit(layers=0, k=None) == 0


def test_pl_kv_copy_pages_refuses():
    src, dst = (ctypes.c_int32 * 1)(1), (ctypes.c_int32 * 1)(2)
    for layers, elements, stride in ((65536, 1024, 1024), (1, 1 << 29, 1 << 29), (1, 1 << 50, 1 << 50)):
        assert _lib.load().pl_kv_copy_pages(PTR, 0, stride, elements, layers, 9, ctypes.addressof(src),
                                            ctypes.addressof(dst), 1, 2, None) == _lib.PL_ERR_UNSUPPORTED
