"""What no query of a prompt sees under a window changes nothing, not a bit of the outputs: prompts over clean and over poisoned caches."""

import numpy as np
import pytest
import torch

from tests.window_cases import BF16, F16, attention, case, check, prefill, set_cache, tables

pytestmark = pytest.mark.gpu

RAGGED = [(1, 1), (17, 17), (40, 3), (130, 129), (300, 33), (400, 200), (1100, 7), (2200, 500)]


def prompts(*args, **kw):
    return case([n for n, _ in RAGGED], *args, new=[m for _, m in RAGGED], **kw)


@pytest.mark.parametrize("dtype,bits", [(BF16, 16), (F16, 16), (BF16, 4), (F16, 4)])
@pytest.mark.parametrize("head_dim,page", [(128, 16), (128, 8), (64, 16), (64, 24), (128, 40)])
@pytest.mark.parametrize("window,sinks", [(70, 5), (33, 0), (200, 70)])
def test_unseen_tokens_change_no_bit(gpu_device, dtype, bits, head_dim, page, window, sinks):
    """NaN groups, or NaN, in the tokens between sinks and window, behind the last one and in unused pages.  In 4 bits a tile
    that holds seen and unseen tokens is worked on in fp16 all the same (another path would round elsewhere)."""
    outs = []
    for poison in (False, True):
        c = prompts(4, 2, head_dim, page, dtype, gpu_device, bits=bits, window=window, sinks=sinks, seed=page, poison=poison)
        outs.append(prefill(c))
        check(c, outs[-1])
    assert torch.equal(*outs)


@pytest.mark.parametrize("dtype,bits", [(BF16, 16), (F16, 16), (BF16, 4), (F16, 4)])
@pytest.mark.parametrize("window,sinks", [(70, 5), (100, 20)])
def test_pages_that_no_query_sees_may_be_any(gpu_device, dtype, bits, window, sinks):
    """Their entries of the table point at a page of NaN."""
    c = prompts(4, 2, 128, 16, dtype, gpu_device, bits=bits, window=window, sinks=sinks, seed=4)
    want = prefill(c)
    check(c, want)
    attn, ids = attention(c), c["indices"].clone()
    nan = int(np.setdiff1d(np.arange(ids.numel() + 3), ids.numpy())[0])  # (unused: poisoned)
    moved = 0
    for (n, new), begin in zip(RAGGED, c["indptr"].tolist()):
        first = max(0, n - new - window + 1)  # of the first query's window
        for page in range(-(-sinks // 16), first // 16):
            ids[begin + page] = nan
            moved += 1
    assert moved > 100
    attn.plan_prefill(qo_indptr=c["qo_indptr"], **{**tables(c), "paged_kv_indices": ids})
    assert torch.equal(attn.run_prefill(c["q"], c["cache"]), want)


@pytest.mark.parametrize("dtype,bits", [(BF16, 16), (F16, 16), (BF16, 4), (F16, 4)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (40, 3)])
def test_nan_in_k_and_q(gpu_device, dtype, bits, window, sinks):
    """A NaN score makes a row NaN, and no row that does not see it."""
    c = case([200, 60], 4, 2, 128, 16, dtype, gpu_device, bits=bits, new=[150, 60], window=window, sinks=sinks, seed=5, poison=False)
    cache = torch.randn((c["indices"].numel() + 3, 2, 16, 2, 128), generator=torch.Generator().manual_seed(1)).to(dtype)
    cache[int(c["indices"][5]), 0, 5, 1, 9] = float("nan")  # position 85 of the first request, kv head 1
    set_cache(c, cache)
    c["q_host"][160, 1, 3] = float("nan")
    c["q"] = c["q_host"].to(gpu_device)
    want = torch.zeros(210, 4, dtype=torch.bool)
    rows = torch.arange(50, 200)
    want[:150, 2:] = ((rows >= 85) & ((rows < 85 + window) if window else True))[:, None]
    want[160, 1] = True
    nan = prefill(c).isnan().cpu()
    assert (nan.all(2) == want).all() and (nan.any(2) == want).all()
