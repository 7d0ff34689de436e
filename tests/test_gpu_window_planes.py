"""Windowed attention keeps its weights' bits: terms that cancel, and weights far below a row's largest."""

import math

import numpy as np
import pytest
import torch

from tests.window_cases import BF16, F16, case, decode, prefill, reference, set_cache

pytestmark = pytest.mark.gpu
KINDS = [(BF16, 16), (F16, 16), (BF16, 4), (F16, 4)]


def run(c, how):
    return (prefill(c) if how == "prefill" else decode(c)[0]).double().cpu().numpy()


def one_query(lens, heads, head_dim, dtype, bits, device, seed, how):
    """Requests with one query each, as a decode step or as prompts' last tokens; q, K and V are all zeros."""
    c = case(lens, *heads, head_dim, 16, dtype, device, bits=bits, new=[1] * len(lens) if how == "prefill" else None, seed=seed,
             poison=False)
    c["q_host"].zero_()
    return c, torch.zeros((c["indices"].numel() + 3, 2, 16, heads[1], head_dim), dtype=dtype)


@pytest.mark.parametrize("dtype,bits", KINDS)
@pytest.mark.parametrize("heads,head_dim", [((4, 1), 128), ((2, 2), 64)])
@pytest.mark.parametrize("how", ["decode", "prefill"])
def test_terms_that_cancel(gpu_device, dtype, bits, heads, head_dim, how):
    """Up to eight terms p_t v_t that take each other down under 2^-11 of the first: 1 or 1.5 times a power of two each, which
    a 4-bit cache holds, alike over the 32 dims of a group but for their sign.

    Of a weight, in units of 2^-24: the exponent, under 2 in size, 2.8 (its scale's two roundings) and 1.4 (its own), the
    exponential 2, and in fp16 4 of the planes (2^-11 of 2^-11) and 5.5 of the 11 in the exponent (2^-21 ln 2): 6.2 and 15.7.
    A sum of n terms in k planes is n k additions, each off by 2 of the largest partial sum (cut off, not rounded).  Two planes
    of bf16 leave 256 of a weight, one of fp16 8192.  The store rounds to half a step; q k is one product, exact."""
    requests, rng = 24, np.random.default_rng(head_dim + heads[0])
    c, cache = one_query([8] * requests, heads, head_dim, dtype, bits, gpu_device, 1, how)
    c["q_host"][..., 0] = torch.as_tensor(rng.uniform(0.5, 0.9, (requests, 1)) * math.sqrt(head_dim)).to(dtype)
    c["q"] = c["q_host"].to(gpu_device)
    q0 = c["q_host"][:, 0, 0].double().numpy()
    bound = np.zeros((requests, heads[0], head_dim))
    for r in range(requests):
        page = int(c["indices"][r])
        for h in range(heads[1]):
            k = -rng.permutation([0.0, 0.0625, 0.125, 0.25, 0.375, 0.5, 0.75, 1.0])
            cache[page, 0, :8, h, 0] = torch.as_tensor(k).to(dtype)
            p = np.exp((k - k.max()) * q0[r] / math.sqrt(head_dim))
            for d in range(0, head_dim, 32):
                v, total, size, top = np.zeros(8), 0.0, 0.0, 0.0
                for t in range(8):
                    if t and abs(total) < 2.0**-11 * size:
                        break
                    want = -total / p[t] if t else 1.0 / p[t]
                    levels = np.sign(want) * 2.0 ** np.floor(math.log2(abs(want))) * np.array([1.0, 1.5, 2.0])
                    v[t] = levels[np.abs(levels - want).argmin()]
                    total += p[t] * v[t]
                    size += abs(p[t] * v[t])
                    top = max(top, abs(total))
                n, planes = np.count_nonzero(v), 3 if dtype == BF16 or (bits == 4 and how == "decode") else 2
                sign = rng.choice([-1.0, 1.0], 32)
                cache[page, 1, :8, h, d: d + 32] = torch.as_tensor(v[:, None] * sign).to(dtype)
                g = heads[0] // heads[1]
                units = (6.2 if planes == 3 else 15.7) * size + n * planes * 2 * max(top, 1.0)
                bound[r, h * g: h * g + g, d: d + 32] = units * 2.0**-24 / p.sum()
    set_cache(c, cache)
    got, o = run(c, how), reference(c)[0]
    off = np.abs(got - o) / (bound + torch.finfo(dtype).eps / 2 * np.abs(o) + (2.0**-25 if dtype == F16 else 0.0))
    print(f"[planes] {how} {dtype} {bits} bits {heads} of {head_dim}: {off.max():.2f} of the bound", flush=True)
    assert off.max() <= 1


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("how", ["decode", "prefill"])
@pytest.mark.parametrize("down", [20, 45, 70])
def test_small_weights_count_where_the_large_meet_zeros(gpu_device, bits, how, down):
    """One token of each row has V = 0 and 2^down times the weight of the others.  An exponent of this size is off by 2^-24
    of it thrice, the exponential and the sums of 40 tokens by 44 more of 2^-24."""
    c, cache = one_query([41] * 3, (4, 2), 128, BF16, bits, gpu_device, 2, how)
    c["q_host"][..., 0] = 16.0
    c["q"] = c["q_host"].to(gpu_device)
    k = torch.tensor(down * math.log(2) * math.sqrt(128) / 16).to(BF16)
    k = float(2.0 ** round(math.log2(float(k))))  # (a value that 4 bits hold)
    for r in range(3):
        pages = c["indices"][c["indptr"][r]: c["indptr"][r + 1]].long()
        cache[pages, 1] = 1.5
        cache[pages[1], 0, 5, :, 0] = k
        cache[pages[1], 1, 5] = 0.0
    set_cache(c, cache)
    got, o = run(c, how), reference(c)[0]
    assert (o > 0).all() and o.max() < 2.0 ** (-down / 2)
    x = k * 16 / math.sqrt(128) * math.log2(math.e)
    assert (np.abs(got - o) <= (2.0**-8 + (3 * x + 44) * 2.0**-24) * o).all()
