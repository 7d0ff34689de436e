"""Pages copied in pools whose dims of one entry have strides of their own."""

import pytest
import torch

from pagelora_amd.kv_pool import kv_copy_pages

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("page,hkv", [(16, 1), (1, 4), (1, 1)])
def test_dims_of_one_entry(gpu_device, page, hkv):
    """A pool ordered by heads is one ordered by tokens where it has one of either: its pages are contiguous."""
    room = torch.randn((3, 9, 2, hkv, page, 64), device=gpu_device)
    cache = room.transpose(3, 4)
    want = cache.clone()
    want[:, [2, 5]] = cache[:, [7, 7]]
    kv_copy_pages(cache, [7, 7], [2, 5])
    kv_copy_pages(cache[1], [0], [1])
    want[1, 1] = want[1, 0]
    assert torch.equal(cache, want)
    one = torch.randn((6, 2, hkv, page, 8), device=gpu_device).transpose(2, 3)[1:2]  # a pool of one page
    kv_copy_pages(one, [], [])
