"""Forms of the tree's calls that ordinary decoding seldom makes: zero scales, caches of other orders, far offsets, bad tables."""

import numpy as np
import pytest
import torch

from oracle import tree as otree
from pagelora_amd.speculative import commit_tree
from tests.test_gpu_tree_attention import backend, oracle, tables, tree_case
from tests.test_gpu_tree_commit import commit_args, commit_case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("head_dim", [64, 128, 256])
def test_a_softmax_scale_of_zero_is_a_mean(gpu_device, dtype, head_dim):
    case = tree_case([11, 3], [400, 30], 8, 2, head_dim, 16, dtype, gpu_device, seed=5)
    be = backend(8, 2, head_dim, 16, gpu_device)
    for scale in (0.0, -0.0):
        be.sm_scale = scale
        be.plan_tree(**tables(case), tree_parents=case["parents"])
        out = torch.empty_like(case["q"])
        lse = torch.empty(out.shape[:2], device=gpu_device)
        be.run_tree_into(case["q"], case["cache"], out, lse)
        ref, ref_lse = oracle(case, 0.0)
        err = np.abs(out.double().cpu().numpy() - ref)
        # sums of 400 values of up to 5 in fp32, then half a step
        assert (err <= torch.finfo(dtype).eps / 2 * np.abs(ref) + 400 * 2.0**-24 * 5).all()
        # the sum of up to 411 weights, each addition off by 2^-24 of it at most: its logarithm by 411 x 2^-24.  fp16 sums
        # weights of 2^14, up to 2^23 in all, whose binary logarithm lies in [16, 32): a step is 2^-19, times ln 2
        assert (np.abs(lse.double().cpu().numpy() - ref_lse) <= 411 * 2.0**-24 + 2.0**-19).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_commit_in_strided_caches(gpu_device, dtype):
    """A pool ordered by heads, and every other page and layer of a larger one: what is not moved stays."""
    cache, *rest = commit_case([9, 20, 1], [5, 33, 16], 16, 3, 2, 64, dtype, seed=3, max_path=9)
    want = otree.commit(cache.float().numpy(), *rest)
    args, kw = commit_args(gpu_device, *rest)
    hnd = cache.to(gpu_device).transpose(3, 4).contiguous()
    commit_tree(hnd.transpose(3, 4), *args, **kw)
    assert np.array_equal(hnd.transpose(3, 4).float().cpu().numpy(), want)
    room = torch.full((6, 2 * cache.shape[1] + 1, 2, 16, 3, 80), 7.0, dtype=dtype, device=gpu_device)
    view = room[1::2, 1::2, :, :, 1:, 8:72]
    view.copy_(cache)
    commit_tree(view, *args, **kw)
    assert np.array_equal(view.float().cpu().numpy(), want)
    view.fill_(7.0)
    assert (room == 7).all()


def test_commit_past_4_gib(gpu_device):
    """Pages whose byte offsets pass 2^32, a layer whose offset does."""
    cache, qo, kv, ids, last, path, count = commit_case([30], [50], 16, 2, 8, 128, torch.bfloat16, seed=1, max_path=12)
    pages = 2**32 // (2 * 16 * 8 * 128 * 2) + 20
    room = torch.zeros((2, pages, 2, 16, 8, 128), dtype=torch.bfloat16, device=gpu_device)
    n = cache.shape[1]
    room[:, pages - n:] = cache.to(gpu_device)
    want = otree.commit(cache.float().numpy(), qo, kv, ids, last, path, count)
    args, kw = commit_args(gpu_device, qo, kv, [i + pages - n for i in ids], last, path, count)
    commit_tree(room, *args, **kw)
    assert np.array_equal(room[:, pages - n:].float().cpu().numpy(), want) and not room[:, : pages - n].any()


def test_commit_by_a_bad_row_pointer_moves_nothing(gpu_device):
    """Rows that begin before the ids, past them, or end before they begin: every request is left alone."""
    cache, qo, kv, ids, last, _, _ = commit_case([8, 8, 8, 8], [20] * 4, 16, 2, 2, 64, torch.bfloat16, 1, max_path=4)
    got = cache.to(gpu_device)
    args, kw = commit_args(gpu_device, qo, kv, ids, last, [[0, 2, 5, 7]] * 4, [4] * 4)
    kw["paged_kv_indptr"] = torch.tensor([-3, 10**8, 10**8, 5, 2], dtype=torch.int32, device=gpu_device)
    commit_tree(got, *args, **kw)
    torch.cuda.synchronize()
    assert torch.equal(got.cpu(), cache)
