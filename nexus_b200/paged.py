"""Quantised paged KV cache over torch CUDA tensors (``nexus_cuda_kv_*``).

For programs that run their own layers next to the engine: the cache of one
layer, keys and values in 8 or 4 bits per (token, KV head), in pages that the
scheduler's page lists (``Scheduler``) name.  The reference packs one token
over all heads and serves one token of one sequence at a time
(src/engine/mod.rs:187-313, 452-499); here a ragged batch of sequences is
written, read back and attended in one call each.

    cache = PagedKvCache.empty(backend, num_pages=4096, kv_heads=8, head_dim=128, bits=(8, 4))
    batch = KvBatch(q_start, kv_len, page_table, max_q=1, max_kv=8192)
    cache.append(batch, k, v)                 # [rows, kv_heads, head_dim]
    out = cache.attention(batch, q)           # [rows, heads, head_dim]

Calls run on torch's current stream of the backend's device, return without
waiting and may be captured into a CUDA graph (the batch's device tensors are
read when the graph runs).  They are for serving: rows that require a gradient
are refused while torch records one.  ``cache.status()`` waits and raises
``NexusError`` for what only the device can see, such as a page id beyond the
pool.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional

import torch

from . import _lib as L
from .engine import CudaBackend

_FORMATS = {torch.float32: L.F32, torch.float16: L.F16, torch.bfloat16: L.BF16}
_KEPT = 64  # structs and sizes a batch keeps (a long-lived one may meet any number of streams)
# torch.cuda.current_stream(device).cuda_stream; the form without its object is
# not part of torch's interface, so that a torch without it is served by the other
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda device: torch.cuda.current_stream(device).cuda_stream)


def _invalid(msg: str) -> L.NexusError:
    return L.NexusError(L.NEXUS_E_INVALID, msg)


def _no_backward(what: str) -> L.NexusError:
    return _invalid(f"{what} has no backward pass: call it under torch.no_grad(), or detach what requires a gradient")


def _on(t: torch.Tensor, device: torch.device, what: str) -> None:
    if t.device != device:
        raise _invalid(f"{what} is on {t.device}, the backend on {device}")


class KvBatch:
    """A ragged batch: sequence b brings rows q_start[b]..q_start[b + 1] of the
    row tensors, the last of its kv_len[b] tokens; token t lives in page
    page_table[b, t // page_tokens].  int32 CUDA tensors (kept by reference:
    their contents may change between calls, not which tensors they are);
    max_q and max_kv bound the new tokens and the length of any sequence, as
    the columns of page_table (which may be a slice of a wider table) do."""

    def __init__(self, q_start: torch.Tensor, kv_len: torch.Tensor, page_table: torch.Tensor, max_q: int,
                 max_kv: int):
        n = kv_len.numel()
        for t, what in ((q_start, "q_start"), (kv_len, "kv_len"), (page_table, "page_table")):
            if t.dtype != torch.int32:
                raise _invalid(f"{what} must be int32")
            if not t.is_cuda:
                raise _invalid(f"{what} must be a CUDA tensor")
        if q_start.dim() != 1 or kv_len.dim() != 1 or q_start.numel() != n + 1:
            raise _invalid("q_start must have one entry more than kv_len")
        if page_table.dim() != 2 or page_table.shape[0] != n:
            raise _invalid("page_table must be [sequences, pages]")
        if not q_start.is_contiguous() or not kv_len.is_contiguous() or (page_table.numel() and
                                                                         page_table.stride(1) != 1):
            raise _invalid("batch arrays must be contiguous")
        if page_table.numel() and (n > 1 and page_table.stride(0) < page_table.shape[1]):
            raise _invalid("page_table rows overlap")
        if q_start.device != kv_len.device or page_table.device != kv_len.device:
            raise _invalid("batch arrays are on different devices")
        if not (0 <= max_q < 1 << 31 and 0 <= max_kv < 1 << 31):
            raise _invalid("max_q and max_kv must be in [0, 2^31)")
        self._tensors = q_start, kv_len, page_table
        self._bounds = int(max_q), int(max_kv)
        self._args = (page_table.stride(0) if n > 1 else page_table.shape[1], q_start.data_ptr(), kv_len.data_ptr(),
                      page_table.data_ptr())
        self._index = kv_len.get_device()
        self._structs = {}     # by stream and page size: filled once, never changed
        self._workspaces = {}  # bytes by what they depend on

    # What the calls are handed was taken from these once: contents may change, the
    # tensors and the bounds are another batch's.
    @property
    def q_start(self) -> torch.Tensor:
        return self._tensors[0]

    @property
    def kv_len(self) -> torch.Tensor:
        return self._tensors[1]

    @property
    def page_table(self) -> torch.Tensor:
        return self._tensors[2]

    @property
    def max_q(self) -> int:
        return self._bounds[0]

    @property
    def max_kv(self) -> int:
        return self._bounds[1]

    def _ref(self, stream: int, page_tokens: int):
        r = self._structs.get((stream, page_tokens))
        if r is None:
            if len(self._structs) >= _KEPT:
                self._structs.clear()
            # the rows of a table that is a slice of a wider one are further apart than they
            # have entries: a sequence ends with its entries, not with the row's pitch
            max_kv = min(self.max_kv, self.page_table.shape[1] * page_tokens)
            r = self._structs[stream, page_tokens] = C.byref(
                L.KvBatch(self.kv_len.numel(), self.max_q, max_kv, *self._args, stream, L.KV_CALLER_STREAM))
        return r


class PagedKvCache:
    """The cache of one layer over the caller's buffers: codes
    [pages, kv_heads, page_tokens, head_dim * bits / 8] uint8 and scales
    [pages, kv_heads, page_tokens, 1 (8 bits) or 2 (4 bits: scale, zero)] f32."""

    def __init__(self, backend: CudaBackend, k_codes: torch.Tensor, k_scales: torch.Tensor, v_codes: torch.Tensor,
                 v_scales: torch.Tensor):
        self.backend = backend
        self.device = torch.device("cuda", backend.device)
        bits = []
        for codes, scales, what in ((k_codes, k_scales, "key"), (v_codes, v_scales, "value")):
            if codes.dim() != 4 or codes.dtype != torch.uint8 or not codes.is_contiguous():
                raise _invalid(f"{what} codes must be a contiguous uint8 [pages, kv_heads, page_tokens, bytes]")
            if scales.dtype != torch.float32 or not scales.is_contiguous() or scales.shape[:-1] != codes.shape[:3] \
                    or scales.shape[-1] not in (1, 2):
                raise _invalid(f"{what} scales must be a contiguous float32 [pages, kv_heads, page_tokens, 1 or 2]")
            _on(codes, self.device, f"{what} codes")
            _on(scales, self.device, f"{what} scales")
            bits.append(8 if scales.shape[-1] == 1 else 4)
        if k_codes.shape[:3] != v_codes.shape[:3]:
            raise _invalid("keys and values differ in pages, heads or page size")
        self.num_pages, self.kv_heads, self.page_tokens = (int(x) for x in k_codes.shape[:3])
        self.bits = (bits[0], bits[1])
        self.head_dim = int(k_codes.shape[3]) * 8 // bits[0]
        if int(v_codes.shape[3]) * 8 // bits[1] != self.head_dim:
            raise _invalid("keys and values differ in head_dim")
        self.k_codes, self.k_scales, self.v_codes, self.v_scales = k_codes, k_scales, v_codes, v_scales
        self._struct = L.KvCache(self.kv_heads, self.head_dim, self.page_tokens, self.num_pages, bits[0], bits[1],
                                 k_codes.data_ptr(), v_codes.data_ptr(), k_scales.data_ptr(), v_scales.data_ptr())
        self._ref = C.byref(self._struct)
        self._shape = (self.kv_heads, self.head_dim, self.page_tokens, self.bits)
        self._lib = backend._lib

    @classmethod
    def empty(cls, backend: CudaBackend, num_pages: int, kv_heads: int, head_dim: int, page_tokens: int = 16,
              bits: tuple[int, int] = (8, 8)) -> "PagedKvCache":
        """A cache in buffers of its own, of num_pages pages."""
        if any(b not in (4, 8) for b in bits):
            raise _invalid("bits must be 8 or 4")
        dev = torch.device("cuda", backend.device)
        shape = (num_pages, kv_heads, page_tokens)
        buffers = []
        for b in bits:
            buffers.append(torch.zeros((*shape, head_dim * b // 8), dtype=torch.uint8, device=dev))
            buffers.append(torch.zeros((*shape, 1 if b == 8 else 2), dtype=torch.float32, device=dev))
        return cls(backend, *buffers)

    def _batch(self, batch: KvBatch):
        if batch._index != self.backend.device:
            raise _invalid(f"the batch is on cuda:{batch._index}, the backend on {self.device}")
        return batch._ref(_raw_stream(self.backend.device), self.page_tokens)

    def _rows(self, t: torch.Tensor, what: str) -> L.KvRows:
        fmt = _FORMATS.get(t.dtype)
        if fmt is None:
            raise _invalid(f"{what} must be float32, float16 or bfloat16")
        shape = t.shape
        if len(shape) != 3 or shape[2] != self.head_dim:
            raise _invalid(f"{what} must be [rows, heads, {self.head_dim}]")
        n, h, d = shape
        rs, hs, es = t.stride()
        if es != 1 and n and h:
            raise _invalid(f"{what}: the elements of a head must be adjacent")
        if not t.is_cuda or t.get_device() != self.backend.device:
            raise _invalid(f"{what} is on {t.device}, the backend on {self.device}")
        # a dimension of one has no stride that matters
        return L.KvRows(t.data_ptr(), fmt, h, n, rs if n > 1 else d * h, hs if h > 1 else d)

    def append(self, batch: KvBatch, k: torch.Tensor, v: torch.Tensor) -> None:
        """Quantise the batch's rows of k and v ([rows, kv_heads, head_dim]) into their slots."""
        if (k.requires_grad or v.requires_grad) and torch.is_grad_enabled():
            raise _no_backward("append")
        bt, rk, rv = self._batch(batch), self._rows(k, "k"), self._rows(v, "v")
        rc = self._lib.nexus_cuda_kv_append(self.backend.handle, self._ref, bt, C.byref(rk), C.byref(rv))
        if rc:
            L.check(rc, self.backend.handle)

    def read(self, batch: KvBatch, rows: int, dtype: torch.dtype = torch.float32,
             out: Optional[tuple[torch.Tensor, torch.Tensor]] = None) -> tuple[torch.Tensor, torch.Tensor]:
        """The values the cache holds for the batch's rows: (k, v), each
        [rows, kv_heads, head_dim].  Rows outside every sequence are left as
        they were (undefined without `out`)."""
        if out is None:
            shape = (rows, self.kv_heads, self.head_dim)
            out = (torch.empty(shape, dtype=dtype, device=self.device),
                   torch.empty(shape, dtype=dtype, device=self.device))
        bt = self._batch(batch)
        rk, rv = self._rows(out[0], "k"), self._rows(out[1], "v")
        if rk.rows != rows or rv.rows != rows:
            raise _invalid(f"out must have {rows} rows")
        rc = self._lib.nexus_cuda_kv_read(self.backend.handle, self._ref, bt, C.byref(rk), C.byref(rv))
        if rc:
            L.check(rc, self.backend.handle)
        return out

    def attention(self, batch: KvBatch, q: torch.Tensor, scale: Optional[float] = None, window: int = 0,
                  sinks: int = 0, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Causal GQA attention of q ([rows, heads, head_dim]) over the cached
        tokens, the rows' own among them; with a window, key j is visible to
        position i when j > i - window or j < sinks.  `scale` (default
        1/sqrt(head_dim)) is positive; `out` may be q itself.  Rows outside
        every sequence are left as they were (undefined without `out`)."""
        if not (0 <= window < 1 << 31 and 0 <= sinks < 1 << 31):  # (the call would see their low 32 bits)
            raise _invalid("window and sinks must be in [0, 2^31)")
        if scale is not None and not scale > 1e-45:  # 0 in f32 would ask for the default
            raise _invalid("scale must be positive")
        if q.requires_grad and torch.is_grad_enabled():
            raise _no_backward("attention")
        if out is None:
            out = torch.empty(q.shape, dtype=q.dtype, device=self.device)
        bt, rq, ro = self._batch(batch), self._rows(q, "q"), self._rows(out, "out")
        qr = C.byref(rq)
        key = (rq.heads, rq.format, rq.rows, window, sinks, self._shape)
        need = batch._workspaces.get(key)
        if need is None:
            size = C.c_size_t()
            L.check(self._lib.nexus_cuda_kv_attention_workspace(self._ref, bt, qr, window, sinks, C.byref(size)))
            if len(batch._workspaces) >= _KEPT:
                batch._workspaces.clear()
            need = batch._workspaces[key] = size.value
        # (held until the launch; reused by the allocator in stream order after it)
        ws = torch.empty(need, dtype=torch.uint8, device=self.device) if need else None
        rc = self._lib.nexus_cuda_kv_attention(self.backend.handle, self._ref, bt, qr, C.byref(ro),
                                               0.0 if scale is None else scale, window, sinks,
                                               None if ws is None else ws.data_ptr(), need)
        if rc:
            L.check(rc, self.backend.handle)
        return out

    def status(self) -> None:
        """Wait for torch's current stream; raise NexusError for what the calls
        of this backend found wrong on the device (then cleared)."""
        L.check(self._lib.nexus_cuda_kv_status(self.backend.handle, _raw_stream(self.backend.device), L.KV_CALLER_STREAM),
                self.backend.handle)
