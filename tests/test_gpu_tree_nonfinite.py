"""Infinities in V that a row of a tree sees: the definition's infinity, wherever the work is cut."""

import numpy as np
import pytest
import torch

from tests.test_gpu_tree_attention import backend, oracle, tables, tree_case

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16
INF = float("inf")


def slot(case, pos, page_size=16):
    return case["indices"].tolist()[case["indptr"].tolist()[0] + pos // page_size], pos % page_size


def compare(case, got, dtype):
    """Infinities with their sign and NaN (both signs in one dim) where the definition has them; the rest within the
    output's rounding and 1e-3, which weights off by 2^-13 make of values of up to 5 (theirs are off by less)."""
    ref = oracle(case)[0]
    got = got.double().cpu().numpy()
    assert (np.isnan(got) == np.isnan(ref)).all()
    inf = np.isinf(ref)
    assert inf.any() and (got[inf] == ref[inf]).all() and not np.isinf(got[~inf]).any()
    live = np.isfinite(ref)
    assert (np.abs(got - ref)[live] <= torch.finfo(dtype).eps / 2 * np.abs(ref[live]) + 1e-3).all()


def run(case, heads, head_dim, device, **kw):
    be = backend(*heads, head_dim, 16, device)
    be.plan_tree(**tables(case), tree_parents=case["parents"], **kw)
    out = be.run_tree(case["q"], case["cache"])
    torch.cuda.synchronize()
    return out


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("heads,head_dim", [((1, 1), 128), ((4, 1), 128), ((4, 1), 64), ((4, 1), 256)])
@pytest.mark.parametrize("tree,prefix,where", [(4, 0, "node")] + [
    (tree, prefix, where) for tree, prefix in ((4, 44), (20, 44), (30, 700), (70, 1500))
    for where in ("node", "committed", "both")])
def test_infinite_v(gpu_device, dtype, heads, head_dim, tree, prefix, where):
    """In nodes and in committed tokens, both signs, in the first block of a wave and in later ones, 16 to 64 rows of a
    row block, every kv range cut in several ways."""
    case = tree_case([tree], [prefix + tree], *heads, head_dim, 16, dtype, gpu_device, seed=tree + prefix)
    at = ([prefix, prefix + tree // 2, prefix + tree - 1] if where != "committed" else []) + \
         ([0, prefix // 2, prefix - 1] if where != "node" else [])
    for n, pos in enumerate(at):
        page, off = slot(case, pos)
        case["cache_host"][page, 1, off, 0, 5 + n] = INF
        case["cache_host"][page, 1, off, 0, 30 + n] = -INF
        case["cache_host"][page, 1, off, 0, 50] = INF if n % 2 else -INF
    case["cache"] = case["cache_host"].to(gpu_device)
    for share in (0, 1, 3):
        compare(case, run(case, heads, head_dim, gpu_device, min_share=share), dtype)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("head_dim", [64, 128, 256])
@pytest.mark.parametrize("tree", [1, 20, 64])
@pytest.mark.parametrize("far", [60.0, 190.0])
@pytest.mark.parametrize("high", [0, 210, 399])
def test_infinite_v_far_below_the_maximum(gpu_device, dtype, head_dim, tree, far, high):
    """The infinite V lies in tokens whose score is `far` (in e's) below the row's maximum, before and after it, a
    weight of e^-190 among them, which fp32 does not hold: still an infinity, however the range is cut."""
    case = tree_case([tree], [400 + tree], 1, 1, head_dim, 16, dtype, gpu_device, seed=tree)
    q, cache = torch.zeros_like(case["q_host"]), torch.nan_to_num(case["cache_host"])
    q[:, :, 0] = 4.0
    cache[:, 0] = 0.0
    page, off = slot(case, high)
    cache[page, 0, off, 0, 0] = far * head_dim**0.5 / 4
    for n, pos in enumerate((5, 130, 300, 398)):
        page, off = slot(case, pos)
        cache[page, 1, off, 0, 9 + n] = -INF
    case.update(q_host=q, cache_host=cache, q=q.to(gpu_device), cache=cache.to(gpu_device))
    for share in (0, 1, 2):
        compare(case, run(case, (1, 1), head_dim, gpu_device, min_share=share), dtype)


def test_an_infinite_v_leaves_other_requests_and_rows_their_bits(gpu_device):
    """Rows that do not see it, of its own request and of others in the same workgroup, come out as without it."""
    trees, lens = [24] + [3] * 40, [200] + [20 + i for i in range(40)]
    case = tree_case(trees, lens, 2, 1, 64, 16, BF16, gpu_device, seed=4)
    clean = run(case, (2, 1), 64, gpu_device)
    page, off = slot(case, 176 + 7)
    case["cache"][page, 1, off, 0, 3] = INF
    got = run(case, (2, 1), 64, gpu_device)
    sees = torch.from_numpy(case["sees"][0][:, 7].copy()).to(gpu_device)
    assert torch.equal(got[24:], clean[24:]) and torch.equal(got[:24][~sees], clean[:24][~sees])
    assert (got[:24][sees][:, :, 3] == INF).all()
    rest = torch.arange(64, device=gpu_device) != 3
    assert torch.equal(got[:24][sees][:, :, rest], clean[:24][sees][:, :, rest])


@pytest.mark.parametrize("page_size", [1, 5, 48])
@pytest.mark.parametrize("tree,prefix", [(30, 300), (200, 90)])
def test_infinite_v_in_any_pages_and_wide_trees(gpu_device, page_size, tree, prefix):
    """Pages that end inside blocks, nodes past the first word of the masks, heads of their own."""
    case = tree_case([3, tree], [50, prefix + tree], 4, 2, 128, page_size, BF16, gpu_device, seed=tree + page_size)
    ip, ind = case["indptr"].tolist(), case["indices"].tolist()
    for n, pos in enumerate((0, prefix - 1, prefix, prefix + 17, prefix + tree - 3)):
        case["cache_host"][ind[ip[1] + pos // page_size], 1, pos % page_size, n % 2, 4 + n] = -INF
    case["cache"] = case["cache_host"].to(gpu_device)
    be = backend(4, 2, 128, page_size, gpu_device)
    for share in (0, 1):
        be.plan_tree(**tables(case), tree_parents=case["parents"], min_share=share)
        compare(case, be.run_tree(case["q"], case["cache"]), BF16)


def test_nan_and_infinite_k_stay_nan(gpu_device):
    """NaN in V, both signs in one dim of a row, V infinite where K is (a weight of exactly 0): NaN in that dim alone."""
    case = tree_case([5], [300], 1, 1, 64, 16, F16, gpu_device, seed=2)
    q, cache = case["q_host"].abs(), torch.nan_to_num(case["cache_host"])
    (p0, o0), (p1, o1), (p2, o2), (p3, o3) = (slot(case, n) for n in (3, 150, 200, 201))
    cache[p0, 1, o0, 0, 7] = float("nan")
    cache[p0, 1, o0, 0, 11] = cache[p3, 1, o3, 0, 11] = INF
    cache[p1, 1, o1, 0, 11] = -INF
    cache[p2, 0, o2, 0, :] = -INF  # q > 0: a score of -inf
    cache[p2, 1, o2, 0, 13] = INF
    cache[p1, 1, o1, 0, 20] = -INF
    case.update(q_host=q, cache_host=cache, q=q.to(gpu_device), cache=cache.to(gpu_device))
    for share in (0, 1, 2):
        got = run(case, (1, 1), 64, gpu_device, min_share=share)
        compare(case, got, F16)
        assert torch.isnan(got[:, 0, [7, 11, 13]]).all() and (got[:, 0, 20] == -INF).all()
