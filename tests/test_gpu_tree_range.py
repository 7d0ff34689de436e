"""Tree attention over the whole range of its values: V near the type's largest."""

import math

import numpy as np
import pytest
import torch

from tests.test_gpu_tree_attention import BF16, backend, oracle, tables, tree_case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("head_dim", [64, 128, 256])
@pytest.mark.parametrize("group", [1, 4, 20])
@pytest.mark.parametrize("high", [5, 200, 520])
@pytest.mark.parametrize("above", [0.5, 7.5, 20.0])
def test_large_finite_v_stays_finite(gpu_device, head_dim, group, high, above):
    """One token `above` the others' scores (in powers of two) holds +-2e38, before the others and behind them: no
    weight is above 1, so what the row holds of it is finite."""
    case = tree_case([3], [600], group, 1, head_dim, 16, BF16, gpu_device, seed=high)
    q, cache = torch.zeros_like(case["q_host"]), torch.nan_to_num(case["cache_host"])
    q[:, :, 0] = 4.0
    cache[:, 0] = 0.0
    page, off = case["indices"].tolist()[high // 16], high % 16
    cache[page, 0, off, 0, 0] = above * math.sqrt(head_dim) / 4 / math.log2(math.e)
    cache[page, 1, off, 0, ::2], cache[page, 1, off, 0, 1::2] = 2e38, -2e38
    case.update(q_host=q, cache_host=cache)
    be = backend(group, 1, head_dim, 16, gpu_device)
    for share in (0, 1, 3):
        be.plan_tree(**tables(case), tree_parents=case["parents"], min_share=share)
        got = be.run_tree(q.to(gpu_device), cache.to(gpu_device)).double().cpu().numpy()
        ref = oracle(case)[0]
        # half a step, and weights off by 2^-16: 601 sums in 32 bits, an exponent below 2^5 and its scale's rounding
        assert np.isfinite(got).all() and (np.abs(got - ref) <= (2.0**-8 + 2.0**-15) * np.abs(ref)).all()
