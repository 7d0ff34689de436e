"""Paged attention under a sliding window with sinks, over caches of 16 or 4 bits.

:class:`WindowAttention` has the ``plan_*`` / ``run_*`` surface of
:class:`~pagelora_amd.attention_backend.PagedDecodeAttention` for long contexts
held in little memory:

* a query at position p sees position t <= p where t > p - ``window`` or
  t < ``sinks``; ``window`` 0 sees every one;
* a layer's cache is bf16 or fp16 ``[P, 2, page, Hkv, D]`` (NHD) or a ``(k, v)``
  pair, or a 4-bit one (uint8, :mod:`pagelora_amd.kv4`); a run takes either.

``o = softmax(q . K^T / sqrt(D)) . V`` over what the query sees.  What it does not
see may hold anything, and a page of which nobody sees a token counts for
nothing: its entry of the page table may name any page of the pool, such as one
that was freed.  The reference attends every position of a 16-bit cache: it has
no counterpart.
"""

from __future__ import annotations

import ctypes
import math

import torch

from . import _lib
from .attention_backend import _cache_pointers, _upload_int32, _validate_host_table
from .kv4 import kv4_geometry

_CODES = {torch.bfloat16: _lib.PL_DTYPE_BF16, torch.float16: _lib.PL_DTYPE_F16}

class WindowAttention:
    """Decode and prefill attention with ``window`` and ``sinks`` (gfx950).

    Decode is planned on the device (``plan_decode`` reads nothing back and may
    be captured), prefill on the host.  A plan is shared by all layers of a step
    and holds copies of its tables.
    """

    def __init__(self, *, device: torch.device | str, num_qo_heads: int, num_kv_heads: int, head_dim: int,
                 page_size: int, window: int = 0, sinks: int = 0) -> None:
        self.device = torch.device(device)
        self.num_qo_heads = int(num_qo_heads)
        self.num_kv_heads = int(num_kv_heads)
        self.head_dim = int(head_dim)
        self.page_size = int(page_size)
        self.window = int(window)
        self.sinks = int(sinks)
        if self.num_kv_heads <= 0 or self.num_qo_heads <= 0 or self.num_qo_heads % self.num_kv_heads:
            raise ValueError("Q head count must be divisible by KV head count")
        if self.head_dim not in (64, 128):
            raise NotImplementedError(f"head_dim must be 64 or 128, got {self.head_dim}")
        if self.page_size < 1:
            raise ValueError(f"page_size must be >= 1, got {self.page_size}")
        if not 0 <= self.window < 2**31 or not 0 <= self.sinks < 2**31:
            raise ValueError(f"window and sinks must be >= 0, got {self.window} and {self.sinks}")
        self.sm_scale = 1.0 / math.sqrt(self.head_dim)
        self._lib = _lib.load() if self.device.type == "cuda" else None
        self._decode_plan: dict | None = None
        self._prefill_plan: dict | None = None
        self._captured: list = []  # plans that graphs read and do not hold themselves

    # -------------------------------------------------------------- shared
    def _need_device(self, what: str) -> int:
        if self._lib is None:
            raise RuntimeError(f"WindowAttention.{what} needs a ROCm device")
        return torch.cuda.current_device() if self.device.index is None else self.device.index

    def _cache(self, cache, dtype: torch.dtype, device: int, max_page: int | None):
        """(K and V addresses, page/token/head stride, pages, bits) of a layer that queries of ``dtype`` attend."""
        if isinstance(cache, torch.Tensor) and cache.dtype == torch.uint8:
            k, v, page_stride, head_stride, num_pages, at = kv4_geometry(cache, self.num_kv_heads, self.head_dim,
                                                                         self.page_size)
            token_stride, bits = 0, 4
        else:
            k, v, page_stride, token_stride, head_stride, num_pages, kv_dtype, at = _cache_pointers(
                cache, self.num_kv_heads, self.head_dim, self.page_size)
            if kv_dtype != dtype:
                raise ValueError(f"q dtype {dtype} != KV cache dtype {kv_dtype}")
            bits = 16
        if at != device:
            raise RuntimeError(f"the KV cache must be on the plan's device (cuda:{device})")
        if max_page is not None and max_page >= num_pages:
            raise ValueError(f"page id {max_page} is outside the {num_pages}-page KV pool")
        return k, v, page_stride, token_stride, head_stride, num_pages, bits

    def _queries(self, q: torch.Tensor, out: torch.Tensor, rows: int, device: int, what: str):
        """(dtype code, q's and out's strides) of packed queries and their output."""
        shape, dtype = q.shape, q.dtype
        if len(shape) != 3 or shape[1] != self.num_qo_heads or shape[2] != self.head_dim:
            raise ValueError(f"q must be [{what}, {self.num_qo_heads}, {self.head_dim}], got {tuple(shape)}")
        if shape[0] != rows:
            raise ValueError(f"q has {shape[0]} {what} but the plan has {rows}")
        code = _CODES.get(dtype)
        if code is None:
            raise NotImplementedError(f"q must be bfloat16 or float16, got {dtype}")
        qs, os_ = q.stride(), out.stride()
        if out.shape != shape or out.dtype != dtype or qs[2] != 1 or os_[2] != 1:
            raise ValueError("q and out must match in shape/dtype with a contiguous head_dim")
        if q.get_device() != device or out.get_device() != device:
            raise RuntimeError(f"q and out must be on the plan's device (cuda:{device})")
        return code, qs, os_

    def _on_stream(self, plan: dict) -> int:
        """The current stream's handle; the plan's memory and work are ordered with it."""
        stream = _lib.raw_stream(plan["device"])
        if not plan["kept"] or plan["captured"] or stream not in plan["streams"]:
            if torch.cuda.is_current_stream_capturing():
                if plan["captured"] == (_lib.capture_id(stream),):
                    # the plan's memory is its graph's, which holds what it captured
                    if stream not in plan["streams"]:
                        plan["memory"].record_stream(torch.cuda.current_stream(plan["device"]))
                        plan["streams"].add(stream)
                elif not plan["kept"]:
                    plan["kept"] = True
                    self._captured.append(plan)
            elif plan["captured"]:
                raise RuntimeError("the plan was captured: it is made when its graph is replayed; plan again for eager "
                                   "runs")
            elif stream not in plan["streams"]:
                here = torch.cuda.current_stream(plan["device"])
                here.wait_event(plan["ready"])
                plan["memory"].record_stream(here)
                plan["streams"].add(stream)
        return stream

    def release_captured(self) -> None:
        """Let go of the plans that captured runs read, for when their graphs are gone.

        A run that is captured without its plan replays on memory that this
        object keeps until then; a graph that holds both needs no keeping.
        """

        for plan in self._captured:
            plan["kept"] = False
        self._captured.clear()

    # -------------------------------------------------------------- decode
    def plan_decode(self, *, paged_kv_indptr: torch.Tensor, paged_kv_indices: torch.Tensor,
                    paged_kv_last_page_len: torch.Tensor) -> None:
        """Plan one query per request, at its last token, for all layers of a step.

        int32 tables, all on the host (validated, uploaded) or all on the device
        (trusted: the kernels clamp every index into its buffer).  With device
        tables it may be captured, together with the runs on it: the replays
        then follow the tables as they are, and the graph holds the plan.  A run
        captured on a plan made before its capture replays on that plan, which
        this object keeps until :meth:`release_captured`.  A request of no tokens
        is allowed.
        """

        tables = (paged_kv_indptr, paged_kv_indices, paged_kv_last_page_len)
        if any(t.dim() != 1 for t in tables):
            raise ValueError("page-table tensors must be 1-D")
        batch = paged_kv_last_page_len.numel()
        if paged_kv_indptr.numel() != batch + 1:
            raise ValueError("paged_kv_indptr must have batch + 1 entries")
        if any(t.dtype != torch.int32 for t in tables):
            raise ValueError("page-table tensors must be int32")
        if len({t.device.type for t in tables}) > 1:
            raise ValueError("page-table tensors must be all on the host or all on the device")
        host = paged_kv_indptr.device.type == "cpu"
        max_page = _validate_host_table(*tables, self.page_size) if host else None
        device = self._need_device("plan_decode")
        with _lib.on_device(device):
            capturing = torch.cuda.is_current_stream_capturing()
            if host:
                if capturing:
                    raise RuntimeError("plan_decode with host tables uploads them and cannot be captured")
                tables = _upload_int32(tables, self.device)
            else:
                if any(t.get_device() != device for t in tables):
                    raise ValueError(f"page-table tensors must be on cuda:{device}")
                tables = [t.contiguous() for t in tables]
            num_indices = tables[1].numel()
            heads, mask = (self.num_qo_heads, self.num_kv_heads), (self.page_size, self.window, self.sinks)
            nbytes = self._lib.pl_window_decode_plan_size(batch, num_indices, *heads, *mask)
            if nbytes == 0:
                raise ValueError(f"pl_window_decode_plan_size: {_lib.last_error()}")
            memory = torch.empty(nbytes, dtype=torch.uint8, device=self.device)
            stream = torch.cuda.current_stream(device)
            captured = capturing and (_lib.capture_id(stream.cuda_stream),)  # (true whatever the number)
            _lib.check(self._lib.pl_window_decode_plan(
                tables[0].data_ptr(), tables[1].data_ptr(), num_indices, tables[2].data_ptr(), batch, *heads,
                *mask, memory.data_ptr(), nbytes, stream.cuda_stream), "pl_window_decode_plan")
            self._decode_plan = {
                "device": device, "batch": batch, "mask": (self.window, self.sinks), "max_page": max_page,
                "memory": memory,
                "args": (memory.data_ptr(), nbytes, num_indices),
                "workspace_bytes": self._lib.pl_window_decode_workspace_size(batch, num_indices, *heads, self.head_dim,
                                                                             *mask),
                "captured": captured, "kept": False, "streams": {stream.cuda_stream},
                "ready": None if captured else stream.record_event(),
            }

    def run_decode(self, q: torch.Tensor, paged_kv_cache_layer) -> torch.Tensor:
        """One layer of decode attention: ``q`` is ``[B, Hq, D]`` or ``[B, Hq, 1, D]``; returns its shape."""
        if q.dim() == 4 and q.shape[2] == 1:
            return self.run_decode(q.squeeze(2), paged_kv_cache_layer).unsqueeze(2)
        return self.run_decode_into(q, paged_kv_cache_layer,
                                    torch.empty_like(q, memory_format=torch.contiguous_format))

    def run_decode_into(self, q: torch.Tensor, paged_kv_cache_layer, out: torch.Tensor,
                        lse: torch.Tensor | None = None) -> torch.Tensor:
        """Writes ``out`` ([B, Hq, D], head_dim contiguous) and optionally ``lse``
        ([B, Hq] fp32, natural log).  A request of no tokens gets 0 and -inf."""

        plan = self._decode_plan
        if plan is None:
            raise RuntimeError("plan_decode must be called before run_decode")
        device, batch = plan["device"], plan["batch"]
        code, qs, os_ = self._queries(q, out, batch, device, "rows")
        k, v, page_stride, token_stride, head_stride, num_pages, bits = self._cache(
            paged_kv_cache_layer, q.dtype, device, plan["max_page"])
        if lse is not None and (lse.dtype != torch.float32 or lse.shape != q.shape[:2] or not lse.is_contiguous()
                                or lse.get_device() != device):
            raise ValueError("lse must be a contiguous fp32 [B, Hq] tensor on the plan's device")
        if batch == 0:
            return out
        with _lib.on_device(device):
            stream = self._on_stream(plan)
            # per call, from torch's allocator: calls on other streams and graphs share nothing
            nbytes = plan["workspace_bytes"]
            ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device)
            status = self._lib.pl_window_decode_run(
                q.data_ptr(), qs[0], qs[1], k, v, page_stride, token_stride, head_stride, num_pages, bits,
                out.data_ptr(), os_[0], os_[1], lse.data_ptr() if lse is not None else None,
                batch, self.num_qo_heads, self.num_kv_heads, self.head_dim, self.page_size, *plan["mask"],
                self.sm_scale, code, *plan["args"], ws.data_ptr(), nbytes, stream)
            if status:
                _lib.check(status, "pl_window_decode_run")
        return out

    # ------------------------------------------------------------- prefill
    def plan_prefill(self, *, qo_indptr: torch.Tensor, paged_kv_indptr: torch.Tensor, paged_kv_indices: torch.Tensor,
                     paged_kv_last_page_len: torch.Tensor) -> None:
        """Plan packed multi-token attention, for all layers of a step.

        Request r owns query rows ``qo_indptr[r] .. qo_indptr[r+1]``, the last
        positions of its paged sequence.  int32 tables on the host or the device
        (read on the host; the work list is uploaded).  Cannot be captured; a run
        can, and replays on the plan it was captured with, which this object keeps
        until :meth:`release_captured`.
        """

        tables = (qo_indptr, paged_kv_indptr, paged_kv_indices, paged_kv_last_page_len)
        if any(t.dim() != 1 for t in tables):
            raise ValueError("prefill tables must be 1-D")
        batch = paged_kv_last_page_len.numel()
        if qo_indptr.numel() != batch + 1 or paged_kv_indptr.numel() != batch + 1:
            raise ValueError("qo_indptr and paged_kv_indptr must have batch + 1 entries")
        if any(t.dtype != torch.int32 for t in tables):
            raise ValueError("prefill tables must be int32")
        host = [t.detach().cpu().contiguous() for t in tables]
        qo_h, kv_h, ind_h, last_h = host
        max_page = _validate_host_table(kv_h, ind_h, last_h, self.page_size)
        device = self._need_device("plan_prefill")
        n, merges, ws_bytes = ctypes.c_int(0), ctypes.c_int(0), ctypes.c_size_t(0)
        counts = (ctypes.byref(n), ctypes.byref(merges), ctypes.byref(ws_bytes))
        args = (qo_h.data_ptr(), kv_h.data_ptr(), last_h.data_ptr(), batch, self.num_qo_heads, self.num_kv_heads,
                self.head_dim, self.page_size, self.window, self.sinks)
        room = 1024  # records, 16 words each; with more, the plan is made again
        items_h = torch.empty(16 * room, dtype=torch.int32)
        status = self._lib.pl_window_prefill_plan(*args, items_h.data_ptr(), room, *counts)
        if status == _lib.PL_ERR_WORKSPACE:
            room = n.value + merges.value
            items_h = torch.empty(16 * room, dtype=torch.int32)
            status = self._lib.pl_window_prefill_plan(*args, items_h.data_ptr(), room, *counts)
        _lib.check(status, "pl_window_prefill_plan")
        items_h = items_h[: max(16, 16 * (n.value + merges.value))]
        with _lib.on_device(device):
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("plan_prefill uploads host tables and cannot be captured")
            items_d, ids_d = _upload_int32((items_h, ind_h), self.device)
            stream = torch.cuda.current_stream(device)
            self._prefill_plan = {
                "device": device, "tokens": int(qo_h[-1]) if batch else 0,
                "mask": (self.window, self.sinks), "max_page": max_page,
                "memory": items_d,  # one allocation holds both
                "args": (ids_d.data_ptr(), items_d.data_ptr(), n.value, merges.value),
                "workspace_bytes": ws_bytes.value,
                "captured": False, "kept": False, "streams": {stream.cuda_stream}, "ready": stream.record_event(),
            }

    def run_prefill(self, q: torch.Tensor, paged_kv_cache_layer) -> torch.Tensor:
        """One layer of prefill attention: packed ``q`` ``[tokens, Hq, D]``, returns the same shape."""
        return self.run_prefill_into(q, paged_kv_cache_layer,
                                     torch.empty_like(q, memory_format=torch.contiguous_format))

    def run_prefill_into(self, q: torch.Tensor, paged_kv_cache_layer, out: torch.Tensor) -> torch.Tensor:
        """Writes ``out`` ([tokens, Hq, D], head_dim contiguous) for packed ``q``."""

        plan = self._prefill_plan
        if plan is None:
            raise RuntimeError("plan_prefill must be called before run_prefill")
        device = plan["device"]
        code, qs, os_ = self._queries(q, out, plan["tokens"], device, "tokens")
        k, v, page_stride, token_stride, head_stride, num_pages, bits = self._cache(
            paged_kv_cache_layer, q.dtype, device, plan["max_page"])
        if plan["tokens"] == 0:
            return out
        with _lib.on_device(device):
            stream = self._on_stream(plan)
            nbytes = plan["workspace_bytes"]
            ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device) if nbytes else None
            status = self._lib.pl_window_prefill_run(
                q.data_ptr(), qs[0], qs[1], k, v, page_stride, token_stride, head_stride, num_pages, bits,
                *plan["args"], out.data_ptr(), os_[0], os_[1], self.num_qo_heads, self.num_kv_heads, self.head_dim,
                self.page_size, *plan["mask"], self.sm_scale, code,
                ws.data_ptr() if nbytes else None, nbytes, nbytes, stream)
            if status:
                _lib.check(status, "pl_window_prefill_run")
        return out
