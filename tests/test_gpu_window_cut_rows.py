"""Windowed decode of batches in which some rows are cut and most are not."""

import pytest
import torch

from tests.window_cases import BF16, F16, attention, case, check, decode, tables

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits,dtype", [(16, BF16), (4, F16)])
@pytest.mark.parametrize("heads", [(4, 1), (3, 3), (33, 1), (8, 8)])
@pytest.mark.parametrize("lens", [[9000, 1, 2500, 0, 40], [1, 40, 0, 7000, 33] * 3 + [20] * 300, [500] * 40 + [12000], [3000]])
def test_some_rows_are_cut(gpu_device, bits, dtype, heads, lens):
    c = case(lens, *heads, 64, 16, dtype, gpu_device, bits=bits, seed=len(lens))
    check(c, *decode(c))


def test_many_short_rows_need_little_scratch(gpu_device):
    """4096 rows of 32 kv heads: peak memory of a run beyond its output and plan."""
    batch = 4096
    c = case([5] * 8, 32, 32, 128, 16, BF16, gpu_device, seed=1)
    c8 = tables(c, gpu_device)
    t = {"paged_kv_indptr": torch.arange(batch + 1, dtype=torch.int32, device=gpu_device),
         "paged_kv_indices": c8["paged_kv_indices"].repeat(batch // 8), "paged_kv_last_page_len": c8["paged_kv_last_page_len"].repeat(batch // 8)}
    attn = attention(c)
    attn.plan_decode(**t)
    q = c["q"].repeat(batch // 8, 1, 1)
    out = torch.empty_like(q)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    attn.run_decode_into(q, c["cache"], out)
    torch.cuda.synchronize()
    assert torch.cuda.max_memory_allocated() - before <= 40 << 20
    assert torch.equal(out, out[:8].repeat(batch // 8, 1, 1))
    check(c, out[:8])
