"""A key-value cache in pages (include/webgllm_paged.h) for sequences of
different length, next to the contiguous caches of webgllm_b200.model.

``rope_kv_paged`` appends (qk-norm, RoPE, keys and values into their pages) and
``attention_paged`` attends over the pages, causally or with a sliding window
and a few first positions that stay visible. ``PagedCache`` holds the pages of
a model's layers and hands them out to sequences.

Tensors are CUDA tensors of one device; the work is enqueued on torch's current
stream of that device. ``k`` and ``v`` are [pages][KV heads][page size][head dim],
float16 or bfloat16: any view of that shape whose last dimension is dense and
whose other strides are multiples of 8 (pages of all layers in one tensor, rows
before heads, keys next to values); both the same strides.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from ._lib import WG_BF16, WG_F16, GpuError, ShapeError, wg_paged_kv
from .q4 import context_of, host_calls

__all__ = ["PagedCache", "attention_paged", "rope_kv_paged"]

_CODES = {torch.float16: WG_F16, torch.bfloat16: WG_BF16}
_workspace_bytes: dict = {}  # (device, head dim) -> bytes


def _bad(msg: str):
    return ShapeError(_lib.WG_INVALID_SHAPE, msg)


def _arg(msg: str):
    return GpuError(_lib.WG_INVALID_ARGUMENT, msg)


def _int32(t: torch.Tensor, what: str, shape: tuple, device: int) -> int:
    if t.dtype is not torch.int32 or t.get_device() != device or t.shape != shape or not t.is_contiguous():
        raise _arg(f"{what} must be a contiguous int32 {list(shape)} tensor on CUDA device {device}")
    return t.data_ptr()


def _check_out(t: torch.Tensor, dtype, shape: tuple, device: int) -> None:
    if t.dtype is not dtype or t.get_device() != device or t.shape != shape or not t.is_contiguous():
        raise _arg(f"out must be a contiguous {dtype} {list(shape)} tensor on CUDA device {device}")


def _cache(k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, batch: int, device: int) -> wg_paged_kv:
    shape, strides = k.shape, k.stride()
    if len(shape) != 4 or v.shape != shape or v.stride() != strides:
        raise _bad(f"k {tuple(shape)} and v {tuple(v.shape)} must be [pages][KV heads][page size][head dim] alike")
    code = _CODES.get(k.dtype)
    if code is None or v.dtype is not k.dtype:
        raise _arg(f"pages must be float16 or bfloat16, not {k.dtype} and {v.dtype}")
    if device < 0 or v.get_device() != device:
        raise _arg("pages must be CUDA tensors of one device")
    if table.dim() != 2 or table.shape[0] != batch:
        raise _bad(f"table {tuple(table.shape)} must be [{batch}][pages of a sequence]")
    t = _int32(table, "table", table.shape, device)
    sp, sh, sr, sd = strides
    if sd != 1 or (sp | sh | sr) & 7 or sp <= 0 or sh <= 0 or sr <= 0:
        # the stride of a dimension of one entry is never walked and may be anything
        sp, sh, sr, sd = (0 if n == 1 else s for n, s in zip(shape, strides))
        if sd > 1 or (sp | sh | sr) & 7 or any(n > 1 and s <= 0 for n, s in zip(shape, (sp, sh, sr, sd))):
            raise _bad(f"pages of strides {strides}: the last must be 1, the others positive multiples of 8")
    return wg_paged_kv(k.data_ptr(), v.data_ptr(), t, code, shape[0], shape[2], table.shape[1], sp, sh, sr)


def _ptr(t: torch.Tensor | None):
    return None if t is None else t.data_ptr()


def rope_kv_paged(qkv: torch.Tensor, pos: torch.Tensor, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, *,
                  heads: int, theta: float = 1e4, q_norm: torch.Tensor | None = None,
                  k_norm: torch.Tensor | None = None, eps: float = 1e-5, row_start: torch.Tensor | None = None,
                  out: torch.Tensor | None = None) -> torch.Tensor:
    """wg_paged_rope_kv: qkv float32 [rows][(heads + 2 KV heads) head dim] of
    pos.numel() sequences (rows / batch each, or by row_start) -> the rotated,
    scaled queries [rows][heads][head dim] in the pages' dtype; keys and values
    go into the pages. Rows that belong to no sequence stay as they were in
    `out` (uninitialised in a new one)."""
    host = host_calls()
    if host is not None:
        done = host.rope_kv_paged(qkv, pos, k, v, table, heads, theta, q_norm, k_norm, eps, row_start, out)
        if done is not None:
            return done
    batch, device = pos.numel(), k.get_device()
    kv = _cache(k, v, table, batch, device)
    _, hkv, _, dim = k.shape
    if qkv.dim() != 2 or qkv.shape[1] != (heads + 2 * hkv) * dim:
        raise _bad(f"qkv {tuple(qkv.shape)} does not hold {heads} + 2 x {hkv} heads of {dim}")
    if qkv.dtype is not torch.float32 or qkv.get_device() != device:
        raise _arg(f"qkv must be float32 on CUDA device {device}")
    if not qkv.is_contiguous():
        qkv = qkv.contiguous()
    rows = qkv.shape[0]
    for n in (q_norm, k_norm):
        if n is not None and (n.dtype is not torch.float32 or n.get_device() != device or n.shape != (dim,)
                              or not n.is_contiguous()):
            raise _arg(f"norm weights must be contiguous float32 [{dim}] on CUDA device {device}")
    if out is None:
        out = torch.empty((rows, heads, dim), dtype=k.dtype, device=k.device)
    else:
        _check_out(out, k.dtype, (rows, heads, dim), device)
    p = _int32(pos, "pos", (batch,), device)
    rs = None if row_start is None else _int32(row_start, "row_start", (batch + 1,), device)
    context_of(device).enqueue(_lib.lib().wg_paged_rope_kv, qkv.data_ptr(), rows, batch, rs, heads, hkv, dim, p, theta,
                               _ptr(q_norm), _ptr(k_norm), eps, out.data_ptr(), ctypes.byref(kv))
    return out


def workspace_bytes(device: int, head_dim: int) -> int:
    """wg_paged_attention_workspace on a CUDA device (its index)."""
    n = _workspace_bytes.get((device, head_dim))
    if n is None:
        b = ctypes.c_size_t()
        ctx = context_of(device)
        with ctx.lock:
            ctx._check(_lib.lib().wg_paged_attention_workspace(ctx.handle, head_dim, ctypes.byref(b)))
        n = _workspace_bytes[device, head_dim] = b.value
    return n


def attention_paged(q: torch.Tensor, pos: torch.Tensor, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, *,
                    window: int = 0, sinks: int = 0, row_start: torch.Tensor | None = None,
                    out: torch.Tensor | None = None, workspace: torch.Tensor | None = None) -> torch.Tensor:
    """wg_paged_attention: q [rows][heads][head dim] (scaled, as rope_kv_paged
    leaves it) of pos.numel() sequences -> out of the same shape. window 0: every
    row sees the keys up to its own position; else the last `window` of them
    and the first `sinks` positions. `workspace`: a uint8 tensor of
    workspace_bytes(...) that no overlapping call uses (default: a new one from
    torch's allocator, safe on any stream and inside a graph). Prompt chunks and
    single rows over long contexts are faster in two calls than in one."""
    host = host_calls()
    if host is not None:
        done = host.attention_paged(q, pos, k, v, table, window, sinks, row_start, out, workspace)
        if done is not None:
            return done
    batch, device = pos.numel(), k.get_device()
    kv = _cache(k, v, table, batch, device)
    _, hkv, _, dim = k.shape
    if q.dim() != 3 or q.shape[2] != dim or q.shape[1] % hkv:
        raise _bad(f"q {tuple(q.shape)} does not match {hkv} KV heads of {dim}")
    if q.dtype is not k.dtype or q.get_device() != device:
        raise _arg(f"q must be {k.dtype} on CUDA device {device}")
    if not q.is_contiguous():
        q = q.contiguous()
    rows, heads, _ = q.shape
    if out is None:
        out = torch.empty_like(q)
    else:
        _check_out(out, q.dtype, q.shape, device)
    p = _int32(pos, "pos", (batch,), device)
    rs = None if row_start is None else _int32(row_start, "row_start", (batch + 1,), device)
    if workspace is None:
        workspace = torch.empty(workspace_bytes(device, dim), dtype=torch.uint8, device=k.device)
    elif workspace.get_device() != device or not workspace.is_contiguous():
        raise _arg(f"workspace must be contiguous on CUDA device {device}")
    context_of(device).enqueue(_lib.lib().wg_paged_attention, q.data_ptr(), rows, batch, rs, heads, hkv, dim, p,
                               ctypes.byref(kv), window, sinks, out.data_ptr(), workspace.data_ptr(), workspace.nbytes)
    return out


class PagedCache:
    """The pages of `layers` attention layers and the table that says which
    sequence holds which (one table for all layers: a page is the same slots in
    each). Bookkeeping is on the host; the table's device copy is updated on
    torch's current stream, so work enqueued before still sees the old one."""

    def __init__(self, layers: int, batch: int, kv_heads: int, head_dim: int, num_pages: int, max_len: int,
                 page_size: int = 64, dtype: torch.dtype = torch.float16, device="cuda"):
        if page_size <= 0 or page_size % 16:
            raise _bad(f"page size {page_size} must be a multiple of 16")
        if dtype not in _CODES:
            raise _arg(f"pages must be float16 or bfloat16, not {dtype}")
        if min(layers, batch, kv_heads, num_pages, max_len) <= 0:
            raise _bad(f"{layers} layers, {batch} sequences, {kv_heads} heads, {num_pages} pages, length {max_len}")
        self.page_size, self.batch, self.num_pages = page_size, batch, num_pages
        self.max_pages = -(-max_len // page_size)
        self.max_len = self.max_pages * page_size
        self.k = torch.empty((layers, num_pages, kv_heads, page_size, head_dim), dtype=dtype, device=device)
        self.v = torch.empty_like(self.k)
        self.table = torch.full((batch, self.max_pages), -1, dtype=torch.int32, device=device)
        self.host = [[-1] * self.max_pages for _ in range(batch)]
        self.free = list(range(num_pages - 1, -1, -1))

    def _upload(self, rows) -> None:
        for b in rows:
            self.table[b].copy_(torch.tensor(self.host[b], dtype=torch.int32))

    def reserve(self, b: int, length: int, start: int = 0) -> None:
        """Pages for positions start .. length - 1 of sequence b (those it has
        it keeps). Without enough free pages nothing changes and
        GpuError(WG_OUT_OF_MEMORY) is raised."""
        if not 0 <= start <= length <= self.max_len:
            raise _lib.RangeError(_lib.WG_OUT_OF_RANGE, f"positions {start}..{length} of {self.max_len}")
        need = [i for i in range(start // self.page_size, -(-length // self.page_size)) if self.host[b][i] < 0]
        if len(need) > len(self.free):
            raise GpuError(_lib.WG_OUT_OF_MEMORY, f"{len(need)} pages needed, {len(self.free)} of {self.num_pages} free")
        for i in need:
            self.host[b][i] = self.free.pop()
        if need:
            self._upload([b])

    def trim(self, b: int, position: int, window: int, sinks: int = 0) -> int:
        """Takes back the pages of sequence b that no row at `position` or later
        sees through the window and the sinks; returns how many."""
        if sinks < 0:
            raise _arg(f"sinks {sinks}")
        if window <= 0:
            return 0
        gone = 0
        past = min(max(0, position - window + 1) // self.page_size, self.max_pages)
        for i in range(-(-sinks // self.page_size), past):
            if self.host[b][i] >= 0:
                self.free.append(self.host[b][i])
                self.host[b][i] = -1
                gone += 1
        if gone:
            self._upload([b])
        return gone

    def release(self, b: int) -> None:
        """Takes back all pages of sequence b."""
        held = [i for i in self.host[b] if i >= 0]
        if held:
            self.free += held
            self.host[b] = [-1] * self.max_pages
            self._upload([b])

    def layer(self, i: int) -> wg_paged_kv:
        """Layer i for the C entry points."""
        return _cache(self.k[i], self.v[i], self.table, self.batch, self.k.get_device())
