"""Paths that read 16 bits refuse a pool of 4 when it is handed over, before they take pages or launch anything."""

import pytest
import torch

from pagelora_amd.decode_graph import BatchDecodeGraphRunner
from pagelora_amd.decoder import DecoderConfig, decode_step_static, prefill
from pagelora_amd.generation import BatchGenerator, prefill_requests
from pagelora_amd.kv_pool import PagedKVPool, Request


class Weights:
    cfg = DecoderConfig(num_layers=1, hidden=256, num_qo_heads=4, num_kv_heads=2, head_dim=64, intermediate=256, vocab=64)


@pytest.mark.parametrize("call", [
    lambda pool: prefill(Weights, pool, Request(length=3), torch.zeros(3, dtype=torch.int64)),
    lambda pool: prefill_requests(Weights, pool, [torch.zeros(3, dtype=torch.int64)]),
    lambda pool: decode_step_static(Weights, pool, None, None),
    lambda pool: BatchDecodeGraphRunner(Weights, pool, None),
    lambda pool: BatchGenerator(Weights, pool),
], ids=["prefill", "prefill_requests", "decode_step_static", "BatchDecodeGraphRunner", "BatchGenerator"])
def test_pools_of_4_bits_are_refused(call):
    pool = PagedKVPool(num_layers=1, capacity_pages=4, page_size=16, num_kv_heads=2, head_dim=64, dtype=torch.bfloat16, device="cpu",
                       kv_bits=4)
    with pytest.raises(NotImplementedError, match="16 bits"):
        call(pool)
    assert pool.allocator.free_pages == 3
