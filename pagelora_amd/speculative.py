"""Tree-speculative decoding: what follows the attention of a drafted tree.

A drafter proposes a tree of tokens per request; the target model runs its
nodes in one pass (``PagedDecodeAttention.plan_tree`` / ``run_tree``), each
node at the position of its depth, and picks a token after every node.  Then
:func:`accept_tree` keeps the longest path that the picks follow, so that
greedy decoding emits the tokens it would have emitted one by one, and
:func:`commit_tree` moves that path's K/V together behind the committed
tokens.  :meth:`~pagelora_amd.kv_pool.PagedKVPool.truncate` gives back the pages
that the rest of the tree held.

Both run on the device without a read-back and may be captured.  The reference
decodes one token per row and step: it has no counterpart.
"""

from __future__ import annotations

from dataclasses import dataclass

import torch

from . import _lib


@dataclass
class AcceptedTree:
    """The accepted path of each request's tree."""

    path: torch.Tensor    # int32 [B, max_path]: its nodes, then -1
    count: torch.Tensor   # int32 [B]: how many
    tokens: torch.Tensor  # int64 [B, max_path]: the target's picks along it, then -1


def _device_1d(t: torch.Tensor, name: str, dtype: torch.dtype, numel: int | None = None) -> None:
    if t.device.type != "cuda":
        raise RuntimeError(f"{name} must be on a ROCm device")
    if t.dtype != dtype or t.dim() != 1 or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous 1-D {dtype} tensor")
    if numel is not None and t.numel() != numel:
        raise ValueError(f"{name} must have {numel} entries, got {t.numel()}")


def _same_device(*tensors: torch.Tensor) -> None:
    if len({t.device for t in tensors}) > 1:
        raise ValueError("all tensors must be on the same device")


def accept_tree(tokens: torch.Tensor, parents: torch.Tensor, picks: torch.Tensor, qo_indptr: torch.Tensor, *,
                max_path: int, out: AcceptedTree | None = None) -> AcceptedTree:
    """Greedy verification of drafted trees (``pl_tree_accept``).

    ``tokens`` (int64), ``parents`` (int32) and ``picks`` (int64: the target's
    pick after each node, ``fused_ops.greedy_argmax`` of the nodes' logits) hold
    the batch's nodes, request r's at ``qo_indptr[r] .. qo_indptr[r+1]``.  Node
    0 of a tree is its root, the token decided by the step before; from node i
    the path goes on to the lowest-numbered child whose token is ``picks[i]``.
    The result's ``tokens`` are what the step decodes: the accepted drafts, then
    the target's own pick after the last of them.  ``out``: tensors to write to.
    """

    if parents.dim() != 1 or qo_indptr.dim() != 1 or qo_indptr.numel() < 1:
        raise ValueError("parents and qo_indptr must be 1-D, qo_indptr with batch + 1 entries")
    n, batch = parents.numel(), qo_indptr.numel() - 1
    _device_1d(tokens, "tokens", torch.int64, n)
    _device_1d(parents, "parents", torch.int32)
    _device_1d(picks, "picks", torch.int64, n)
    _device_1d(qo_indptr, "qo_indptr", torch.int32)
    max_path = int(max_path)
    if max_path < 1:
        raise ValueError("max_path must be >= 1")
    dev = tokens.device
    if out is None:
        out = AcceptedTree(torch.empty((batch, max_path), dtype=torch.int32, device=dev),
                           torch.empty(batch, dtype=torch.int32, device=dev),
                           torch.empty((batch, max_path), dtype=torch.int64, device=dev))
    else:
        for name, t, dtype, shape in (("path", out.path, torch.int32, (batch, max_path)),
                                      ("count", out.count, torch.int32, (batch,)),
                                      ("tokens", out.tokens, torch.int64, (batch, max_path))):
            if t.dtype != dtype or tuple(t.shape) != shape or not t.is_contiguous():
                raise ValueError(f"out.{name} must be a contiguous {dtype} tensor of shape {shape}")
    _same_device(tokens, parents, picks, qo_indptr, out.path, out.count, out.tokens)
    with _lib.on_device(dev):
        _lib.check(_lib.load().pl_tree_accept(
            tokens.data_ptr(), parents.data_ptr(), picks.data_ptr(), qo_indptr.data_ptr(), batch, n, max_path,
            out.path.data_ptr(), out.count.data_ptr(), out.tokens.data_ptr(), _lib.stream_handle(dev)),
            "pl_tree_accept")
    return out


def commit_tree(cache: torch.Tensor, path: torch.Tensor, count: torch.Tensor, *, qo_indptr: torch.Tensor,
                paged_kv_indptr: torch.Tensor, paged_kv_indices: torch.Tensor,
                paged_kv_last_page_len: torch.Tensor) -> None:
    """Move the accepted paths' K/V together, in every layer (``pl_tree_commit``).

    ``cache``: the pool [layers, P, 2, page, Hkv, D], or one layer of it.  The
    tables are those of the tree's ``plan_tree`` (device tensors), ``path`` and
    ``count`` those of :func:`accept_tree`: K/V of tree node ``path[r, k]`` go to
    position ``k`` behind request r's committed tokens.  Its length is then the
    committed tokens plus ``count[r]``; what lies behind keeps its values.
    Paths ascend: an entry below its own index, or outside the tree, ends one.
    Pages that two requests of the batch share are not written safely.
    """

    if cache.dim() == 5:
        cache = cache.unsqueeze(0)
    if cache.dim() != 6 or cache.shape[2] != 2:
        raise ValueError(f"cache must be [layers, P, 2, page, Hkv, D] or a layer of it, got {tuple(cache.shape)}")
    if cache.device.type != "cuda":
        raise RuntimeError("commit_tree needs a cache on a ROCm device")
    if cache.stride(5) != 1:
        raise ValueError("head_dim must be contiguous in the KV cache")
    layers, num_pages, _, page_size, hkv, head_dim = cache.shape
    if qo_indptr.dim() != 1 or qo_indptr.numel() < 1:
        raise ValueError("qo_indptr must be 1-D with batch + 1 entries")
    batch = qo_indptr.numel() - 1
    _device_1d(qo_indptr, "qo_indptr", torch.int32)
    _device_1d(paged_kv_indptr, "paged_kv_indptr", torch.int32, batch + 1)
    _device_1d(paged_kv_indices, "paged_kv_indices", torch.int32)
    _device_1d(paged_kv_last_page_len, "paged_kv_last_page_len", torch.int32, batch)
    _device_1d(count, "count", torch.int32, batch)
    if path.dtype != torch.int32 or path.dim() != 2 or path.shape[0] != batch or not path.is_contiguous():
        raise ValueError(f"path must be a contiguous int32 [{batch}, max_path] tensor")
    _same_device(cache, path, count, qo_indptr, paged_kv_indptr, paged_kv_indices, paged_kv_last_page_len)
    if path.shape[1] == 0 or num_pages == 0:
        return
    with _lib.on_device(cache.device):
        _lib.check(_lib.load().pl_tree_commit(
            cache.data_ptr(), cache[:, :, 1].data_ptr(), cache.stride(0), cache.stride(1), cache.stride(3),
            cache.stride(4), layers, num_pages, qo_indptr.data_ptr(), paged_kv_indptr.data_ptr(),
            paged_kv_indices.data_ptr(), paged_kv_indices.numel(), paged_kv_last_page_len.data_ptr(), path.data_ptr(),
            count.data_ptr(), batch, path.shape[1], hkv, head_dim, page_size, _lib.dtype_code(cache.dtype),
            _lib.stream_handle(cache.device)), "pl_tree_commit")
