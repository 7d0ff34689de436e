"""Tree-speculative decoding: what follows the attention of a drafted tree.

A drafter proposes a tree of tokens per request; the target model runs its
nodes in one pass (``PagedDecodeAttention.plan_tree`` / ``run_tree``), each
node at the position of its depth, and picks a token after every node.  Then
:func:`accept_tree` keeps the path that the picks follow, so that greedy
decoding emits the tokens it would have emitted one by one, and
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


def _vector(t: torch.Tensor, name: str, dtype: torch.dtype, numel: int, device: int) -> int:
    """The address of a contiguous 1-D tensor of ``numel`` elements on device ``device``."""
    if t.get_device() != device:
        raise RuntimeError(f"{name} must be on the same ROCm device as the others")
    if t.dtype != dtype or t.dim() != 1 or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous 1-D {dtype} tensor")
    if t.numel() != numel:
        raise ValueError(f"{name} must have {numel} entries, got {t.numel()}")
    return t.data_ptr()


def accept_tree(tokens: torch.Tensor, parents: torch.Tensor, picks: torch.Tensor, qo_indptr: torch.Tensor, *,
                max_path: int, out: AcceptedTree | None = None) -> AcceptedTree:
    """Greedy verification of drafted trees (``pl_tree_accept``).

    ``tokens`` (int64), ``parents`` (int32) and ``picks`` (int64: the target's
    pick after each node, ``fused_ops.greedy_argmax`` of the nodes' logits) hold
    the batch's nodes, request r's at ``qo_indptr[r] .. qo_indptr[r+1]``.  Node
    0 of a tree is its root, the token decided by the step before; from node i
    the path goes on to the lowest-numbered child whose token is ``picks[i]``
    (the only one, unless a drafter gives a node two children of one token).
    The result's ``tokens`` are what the step decodes: the accepted drafts, then
    the target's own pick after the last of them.  ``out``: tensors to write to.
    """

    n, batch, device = parents.numel(), qo_indptr.numel() - 1, tokens.get_device()
    if device < 0:
        raise RuntimeError("accept_tree needs tensors on a ROCm device")
    if batch < 0:
        raise ValueError("qo_indptr must have batch + 1 entries")
    max_path = int(max_path)
    if max_path < 1:
        raise ValueError("max_path must be >= 1")
    args = (_vector(tokens, "tokens", torch.int64, n, device), _vector(parents, "parents", torch.int32, n, device),
            _vector(picks, "picks", torch.int64, n, device),
            _vector(qo_indptr, "qo_indptr", torch.int32, batch + 1, device))
    if out is None:
        out = AcceptedTree(parents.new_empty((batch, max_path)), parents.new_empty(batch),
                           tokens.new_empty((batch, max_path)))
    else:
        for name, t, dtype, shape in (("path", out.path, torch.int32, (batch, max_path)),
                                      ("count", out.count, torch.int32, (batch,)),
                                      ("tokens", out.tokens, torch.int64, (batch, max_path))):
            if t.dtype != dtype or t.shape != shape or not t.is_contiguous() or t.get_device() != device:
                raise ValueError(f"out.{name} must be a contiguous {dtype} tensor of shape {shape} on the same device")
    with _lib.on_device(device):
        _lib.check(_lib.load().pl_tree_accept(*args, batch, n, max_path, out.path.data_ptr(), out.count.data_ptr(),
                                              out.tokens.data_ptr(), _lib.raw_stream(device)), "pl_tree_accept")
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

    shape, strides = cache.shape, cache.stride()
    if len(shape) == 5:
        shape, strides = (1, *shape), (0, *strides)
    if len(shape) != 6 or shape[2] != 2:
        raise ValueError(f"cache must be [layers, P, 2, page, Hkv, D] or a layer of it, got {tuple(cache.shape)}")
    device = cache.get_device()
    if device < 0:
        raise RuntimeError("commit_tree needs a cache on a ROCm device")
    if strides[5] != 1:
        raise ValueError("head_dim must be contiguous in the KV cache")
    layers, num_pages, _, page_size, hkv, head_dim = shape
    batch = qo_indptr.numel() - 1
    if batch < 0:
        raise ValueError("qo_indptr must have batch + 1 entries")
    num_indices = paged_kv_indices.numel()
    tables = (_vector(qo_indptr, "qo_indptr", torch.int32, batch + 1, device),
              _vector(paged_kv_indptr, "paged_kv_indptr", torch.int32, batch + 1, device),
              _vector(paged_kv_indices, "paged_kv_indices", torch.int32, num_indices, device), num_indices,
              _vector(paged_kv_last_page_len, "paged_kv_last_page_len", torch.int32, batch, device))
    if path.dtype != torch.int32 or path.dim() != 2 or path.shape[0] != batch or not path.is_contiguous():
        raise ValueError(f"path must be a contiguous int32 [{batch}, max_path] tensor")
    if path.get_device() != device:
        raise RuntimeError("path must be on the same ROCm device as the others")
    counts = _vector(count, "count", torch.int32, batch, device)
    if path.shape[1] == 0 or num_pages == 0:
        return
    base = cache.data_ptr()
    with _lib.on_device(device):
        _lib.check(_lib.load().pl_tree_commit(
            base, base + strides[2] * cache.element_size(), strides[0], strides[1], strides[3], strides[4], layers,
            num_pages, *tables, path.data_ptr(), counts, batch, path.shape[1], hkv, head_dim, page_size,
            _lib.dtype_code(cache.dtype), _lib.raw_stream(device)), "pl_tree_commit")
