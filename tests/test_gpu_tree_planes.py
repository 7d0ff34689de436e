"""The probabilities of tree attention keep their 32 bits, as a decode step's do: terms that cancel."""

import math

import numpy as np
import pytest
import torch

from tests.test_gpu_tree_attention import backend, oracle, tables, tree_case

pytestmark = pytest.mark.gpu


def cancelling_error(dtype, group, head_dim, device, seed):
    """The relative error of one node behind two committed tokens, whose three terms take each other down to 2^-12."""
    rng = np.random.default_rng(seed)
    case = tree_case([1], [3], group, 1, head_dim, 16, dtype, device, seed=seed)
    page = int(case["indices"][0])
    q, cache = torch.zeros_like(case["q_host"]), torch.zeros_like(case["cache_host"])
    q[:, :, 0] = 8.0
    scores = np.array([0.0, -rng.uniform(0.1, 0.9), -rng.uniform(1.1, 1.9)])  # powers of two
    cache[page, 0, :3, 0, 0] = torch.as_tensor(scores * math.sqrt(head_dim) / 8 / math.log2(math.e)).to(dtype)
    k = cache[page, 0, :3, 0, 0].double().numpy()
    p = np.exp((k - k.max()) * 8.0 / math.sqrt(head_dim))
    cut = lambda x: torch.as_tensor(x, dtype=torch.float64).to(dtype).double().numpy()  # noqa: E731
    v = np.zeros((3, head_dim))
    v[1] = cut(rng.uniform(1, 2, head_dim))
    v[0] = cut(-p[1] * v[1] / p[0])
    left = p[0] * v[0] + p[1] * v[1]
    v[2] = cut(-(left - np.sign(left) * 2.0**-12) / p[2])
    cache[page, 1, :3, 0] = torch.as_tensor(v).to(dtype)
    case.update(q_host=q, cache_host=cache)
    be = backend(group, 1, head_dim, 16, device)
    be.plan_tree(**tables(case), tree_parents=case["parents"])
    got = be.run_tree(q.to(device), cache.to(device)).double().cpu().numpy()
    want = oracle(case)[0]
    return np.linalg.norm(got - want) / np.linalg.norm(want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("group,head_dim", [(1, 64), (4, 128), (40, 128), (7, 256)])
def test_probabilities_keep_their_32_bits(gpu_device, dtype, group, head_dim):
    """In units of 2^-24: a probability is off by 5 of itself (scale and exponent, below 2^1, rounded: 2 x 1.4; the
    exponential: 2), and nine additions of what is below 2 by 18 more.  The terms are up to 2, 1 and 1 in size, so the
    sum, times 1 / 1.75 like its value, is off by 38 of 2^-12 x 2^12: 2^-6.7 of a value of 2^-12.  Two planes
    of bf16 leave 2^-17 of a probability, seven times as much.  The store rounds to half a step."""
    errs = [cancelling_error(dtype, group, head_dim, gpu_device, s) for s in range(8)]
    print(f"[planes] {dtype} {group} heads of {head_dim}: " + " ".join(f"{e:.1e}" for e in errs), flush=True)
    assert max(errs) <= 2.0**-6.7 + torch.finfo(dtype).eps / 2
