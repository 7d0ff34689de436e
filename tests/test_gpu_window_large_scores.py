"""Windowed attention under scores of any finite size: the row's maximum is its exponents' zero, exactly."""

import math

import numpy as np
import pytest
import torch

from tests.window_cases import BF16, F16, case, decode, prefill, set_cache

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,bits,size", [(F16, 16, 2**11), (F16, 4, 2**11), (F16, 4, 2**13), (BF16, 16, 2**11),
                                             (BF16, 4, 2**11), (BF16, 16, 2**14), (BF16, 4, 2**14), (BF16, 16, 2**40), (BF16, 4, 2**40)])
@pytest.mark.parametrize("how", ["decode", "prefill"])
@pytest.mark.parametrize("lens", [[40, 130, 300] * 8, [3000, 2500]])
def test_rows_that_are_one_hot(gpu_device, dtype, bits, size, how, lens):
    """q . k = sum of 128 products that are equal but for signs which cancel: exact, and the largest is shared by three tokens,
    far apart, whose V is averaged; the others are thousands away.  Weights of 1 (2^-22 of two fp16 planes, 2^-23 of an
    exponential of one exponent, alike), five sums and a product: 16 times 2^-22 of the largest |v| holds them."""
    rng = np.random.default_rng(size % 1000 + len(lens) + bits)
    c = case(lens, 4, 2, 128, 16, dtype, gpu_device, bits=bits, seed=3, poison=False,
             new=[1] * len(lens) if how == "prefill" else None)
    cache = torch.randn((c["indices"].numel() + 3, 2, 16, 2, 128), generator=torch.Generator().manual_seed(1)).to(dtype)
    signs = torch.as_tensor(rng.choice([-1.0, 1.0], 128))
    big = torch.as_tensor((1 + rng.integers(0, 128, (len(lens), 4, 1)) / 128) * size).to(dtype)  # eight bits
    c["q_host"][:] = (big.double() * signs).to(dtype)
    c["q"] = c["q_host"].to(gpu_device)
    most = []
    for r, n in enumerate(lens):
        pages = c["indices"][c["indptr"][r]: c["indptr"][r + 1]].long()
        level = np.sort(rng.choice([-1.0, 0.5, 0.75, 1.0], n)) if r % 2 else rng.choice([-1.0, 0.5, 0.75, 1.0], n)
        at = rng.choice(n, 3, replace=False)
        level[at] = 1.5
        most.append(at)
        level = torch.as_tensor(level * size)
        for t in range(n):
            cache[pages[t // 16], 0, t % 16] = (level[t] * signs).to(dtype)
    set_cache(c, cache)
    got = prefill(c) if how == "prefill" else None
    lse = None
    if got is None:
        got, lse = decode(c)
    got = got.double().cpu().numpy()
    for r, n in enumerate(lens):
        kv = c["cache_host"][c["indices"][c["indptr"][r]: c["indptr"][r + 1]].long().numpy()]
        v = kv[:, 1].reshape(-1, 2, 128)[most[r]]
        o = np.repeat(v.mean(0), 2, axis=0)
        bound = torch.finfo(dtype).eps / 2 * np.abs(o) + 16 * 2.0**-22 * np.abs(v).max() + (2.0**-25 if dtype == F16 else 0.0)
        assert (np.abs(got[r] - o) <= bound).all(), f"request {r}: {np.abs(got[r] - o).max()}"
        if lse is not None:  # a product of two roundings and a scale of two
            want = 128 * 1.5 * size * big[r, :, 0].double().numpy() / math.sqrt(128) + math.log(3)
            assert (np.abs(lse[r].double().cpu().numpy() - want) <= 2.0**-21 * want).all()
