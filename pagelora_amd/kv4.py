"""A paged KV cache of 4 bits per value: its layout, tokens into it and back.

A layer is uint8 ``[P, 2, Hkv, page * (D / 2 + D / 32)]``, K at index 0 and V at
index 1 of dim 2: per page and kv head the codes of its tokens, then their
scales.  Each 32 values of a token along head_dim share a power of two
``2^(s - 127)``, one byte ``s``: the least at which the largest magnitude is at
most 6.  A value is a code of 4 bits times it (e2m1: a sign and 0, 0.5, 1, 1.5,
2, 3, 4 or 6), the nearest one, halfway to the one with an even mantissa: 4.25
bits per value.  ``s`` lies in 2 .. 252, and is 127 in a group of zeros; 255 marks
a group that held a NaN or an infinity, and reads back as NaN.

* K: codes ``[token][D / 2 bytes]``, scales ``[token][D / 32]``;
* V: codes ``[token / 4][d / 8][token % 4][4 bytes]``, scales
  ``[token / 4][d / 32][token % 4]``: as the attention's lanes take them.

The lower nibble of a byte is the lower dim.  Pages hold a multiple of 8 tokens,
head_dim is 64 or 128.  The values are exact in bf16, so that attention over
them (:class:`pagelora_amd.window_attention.WindowAttention`) loses nothing
more.  The reference keeps its cache in 16 bits: it has no counterpart.
"""

from __future__ import annotations

import torch

from . import _lib

KV4_GROUP = 32
_CODES = {torch.bfloat16: _lib.PL_DTYPE_BF16, torch.float16: _lib.PL_DTYPE_F16}


def kv4_page_shape(*, num_kv_heads: int, head_dim: int, page_size: int) -> tuple[int, int, int]:
    """The shape of one page of a 4-bit cache (uint8): ``[2, Hkv, bytes]``."""
    if head_dim not in (64, 128):
        raise NotImplementedError(f"a 4-bit cache needs head_dim 64 or 128, got {head_dim}")
    if page_size < 8 or page_size % 8:
        raise ValueError(f"pages of a 4-bit cache hold a multiple of 8 tokens, got {page_size}")
    return 2, num_kv_heads, page_size * (head_dim // 2 + head_dim // KV4_GROUP)


def kv4_geometry(cache: torch.Tensor, num_kv_heads: int, head_dim: int, page_size: int):
    """A 4-bit layer as numbers: (K and V addresses, page and head stride in bytes, pages, device index)."""
    shape, strides = cache.shape, cache.stride()
    if (cache.dtype != torch.uint8 or len(shape) != 4 or page_size < 8 or page_size % 8 or head_dim not in (64, 128)
            or shape[1:] != (2, num_kv_heads, page_size * (head_dim // 2 + head_dim // KV4_GROUP))):
        page = kv4_page_shape(num_kv_heads=num_kv_heads, head_dim=head_dim, page_size=page_size)
        raise ValueError(f"4-bit KV cache layer must be uint8 [P, {page[0]}, {page[1]}, {page[2]}], got {cache.dtype} "
                         f"{tuple(shape)}")
    if strides[3] != 1:
        raise ValueError("the bytes of a head's page must be contiguous in the KV cache")
    k = cache.data_ptr()
    return k, k + strides[1], strides[0], strides[2], shape[0], cache.get_device()


def _places(page_id: torch.Tensor, page_offset: torch.Tensor, device: int) -> int:
    """How many places these are."""
    n = page_id.shape
    if (page_id.dtype != torch.int64 or page_offset.dtype != torch.int64 or len(n) != 1 or page_offset.shape != n
            or not page_id.is_contiguous() or not page_offset.is_contiguous()):
        raise ValueError("page_id and page_offset must be contiguous 1-D int64 tensors of one length")
    if page_id.get_device() != device or page_offset.get_device() != device:
        raise RuntimeError("page_id and page_offset must be on the cache's device")
    return n[0]


def kv4_append(cache_layer: torch.Tensor, k: torch.Tensor, v: torch.Tensor, page_id: torch.Tensor,
               page_offset: torch.Tensor, *, num_kv_heads: int, head_dim: int, page_size: int) -> None:
    """Quantize tokens into their pages (``pl_kv4_append``), one or a prompt's.

    ``k``, ``v``: bf16 or fp16 ``[tokens, Hkv, D]``, head_dim contiguous;
    ``page_id``, ``page_offset``: int64 ``[tokens]``, each place once.  Tokens
    whose place is outside the pool are dropped, as by
    :func:`~pagelora_amd.attention_backend.kv_append`.  May be captured.
    """

    k_ptr, v_ptr, page_stride, head_stride, num_pages, device = kv4_geometry(cache_layer, num_kv_heads, head_dim, page_size)
    if device < 0:
        raise RuntimeError("kv4_append needs a cache on a ROCm device")
    shape, code = k.shape, _CODES.get(k.dtype)
    if len(shape) != 3 or shape[1] != num_kv_heads or shape[2] != head_dim or v.shape != shape:
        raise ValueError(f"k and v must be [tokens, {num_kv_heads}, {head_dim}]")
    if code is None or v.dtype != k.dtype:
        raise NotImplementedError(f"k and v must be both bfloat16 or both float16, got {k.dtype} and {v.dtype}")
    ks, vs = k.stride(), v.stride()
    if ks[2] != 1 or vs[2] != 1:
        raise ValueError("k and v need a contiguous head_dim")
    if k.get_device() != device or v.get_device() != device:
        raise RuntimeError("k and v must be on the cache's device")
    tokens = _places(page_id, page_offset, device)
    if tokens != shape[0]:
        raise ValueError("page_id / page_offset must have one entry per token")
    if tokens == 0 or num_pages == 0:
        return
    with _lib.on_device(device):
        status = _lib.load().pl_kv4_append(
            k.data_ptr(), v.data_ptr(), ks[0], ks[1], vs[0], vs[1], k_ptr, v_ptr, page_stride, head_stride, num_pages,
            page_size, page_id.data_ptr(), page_offset.data_ptr(), tokens, num_kv_heads, head_dim, code,
            _lib.raw_stream(device))
    if status:
        _lib.check(status, "pl_kv4_append")


def kv4_read(cache_layer: torch.Tensor, page_id: torch.Tensor, page_offset: torch.Tensor, *, num_kv_heads: int,
             head_dim: int, page_size: int, dtype: torch.dtype = torch.bfloat16) -> tuple[torch.Tensor, torch.Tensor]:
    """K and V of the tokens at these places, ``[tokens, Hkv, D]`` each (``pl_kv4_read``).

    bf16 holds the cache's values exactly, fp16 rounds those outside its range.
    Tokens whose place is outside the pool read as NaN.  May be captured.
    """

    k_ptr, v_ptr, page_stride, head_stride, num_pages, device = kv4_geometry(cache_layer, num_kv_heads, head_dim, page_size)
    if device < 0:
        raise RuntimeError("kv4_read needs a cache on a ROCm device")
    code = _CODES.get(dtype)
    if code is None:
        raise NotImplementedError(f"dtype must be bfloat16 or float16, got {dtype}")
    tokens = _places(page_id, page_offset, device)
    k = torch.empty((2, tokens, num_kv_heads, head_dim), dtype=dtype, device=cache_layer.device)
    if num_pages == 0:
        k.fill_(float("nan"))
    elif tokens:
        stride = num_kv_heads * head_dim
        address = k.data_ptr()
        with _lib.on_device(device):
            status = _lib.load().pl_kv4_read(
                k_ptr, v_ptr, page_stride, head_stride, num_pages, page_size, page_id.data_ptr(),
                page_offset.data_ptr(), tokens, num_kv_heads, head_dim, address, address + 2 * tokens * stride, stride,
                head_dim, stride, head_dim, code, _lib.raw_stream(device))
        if status:
            _lib.check(status, "pl_kv4_read")
    return k.unbind(0)
