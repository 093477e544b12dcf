"""A paged q8 key/value cache on the device: append, attention and read (qwc_op_paged_*).

`PagedCache` names one layer's pool of pages, `PagedBatch` the tokens of one step; both hold
torch tensors (device memory, nothing is computed by torch) and the descriptors that the C ABI
takes, so a call is one ABI call on torch's current stream of the device that holds them. A refused argument
raises `QwcError` with the status, as everywhere in this package.

    cache = PagedCache.zeros(pages=512, page_size=64, kv_heads=8, head_dim=128)     # one for each layer
    batch = PagedBatch(query_starts, context_lens, page_table, tokens=n, max_query=q, max_context=c)
    q = append(cache, batch, q, k, v, cos, sin, q_norm=qn, k_norm=kn, eps=1e-6)
    out = attention(cache, batch, q)
"""

from __future__ import annotations

import ctypes

import torch

from .quant import GROUP
from .runtime import (FORMAT_BF16, FORMAT_F16, FORMAT_F32, PAGED_WORKSPACE_HEAD, STATUS_CODE, PagedBatchDesc, PagedCacheDesc,
                      QwcError, check, lib)

FORMATS = {torch.float32: FORMAT_F32, torch.float16: FORMAT_F16, torch.bfloat16: FORMAT_BF16}


def refuse(name: str, call: str):
    raise QwcError(STATUS_CODE[name], call)


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def current_stream(device: torch.device) -> int:
    """torch's current stream of a device, as the C ABI takes it."""
    if _raw_stream is not None and device.index is not None:
        return _raw_stream(device.index)
    return torch.cuda.current_stream(device).cuda_stream


_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


def elsewhere(index: int | None, call: str):
    """A kernel is launched on the current device: the context that makes device `index` the current one, or None where it
    is already. Memory that no GPU holds (no index) is refused."""
    if index is None:
        refuse("invalid_argument", call)
    return None if index == _current_device() else torch.cuda.device(index)


def cuda_index(device: torch.device) -> int | None:
    return device.index if device.type == "cuda" else None


def format_of(t: torch.Tensor, call: str) -> int:
    fmt = FORMATS.get(t.dtype)
    if fmt is None:
        refuse("unsupported", call)
    return fmt


class PagedCache:
    """One layer's pool: f16 scales [pages * page_size, kv_heads * head_dim / 64] and u8 codes
    [pages * page_size, kv_heads * head_dim], keys and values."""

    def __init__(self, k_scales: torch.Tensor, k_codes: torch.Tensor, v_scales: torch.Tensor, v_codes: torch.Tensor, *,
                 page_size: int, kv_heads: int, head_dim: int):
        width = kv_heads * head_dim
        rows = k_codes.shape[0] if k_codes.dim() == 2 else -1
        if page_size < 1 or rows < 0 or rows % page_size or width % GROUP:
            refuse("shape_mismatch", "PagedCache")
        for t, cols, dtype in ((k_scales, width // GROUP, torch.float16), (k_codes, width, torch.uint8),
                               (v_scales, width // GROUP, torch.float16), (v_codes, width, torch.uint8)):
            if t.dtype != dtype or t.device != k_codes.device or not t.is_contiguous():
                refuse("invalid_argument", "PagedCache")
            if t.shape != (rows, cols):
                refuse("shape_mismatch", "PagedCache")
        self.k_scales, self.k_codes, self.v_scales, self.v_codes = k_scales, k_codes, v_scales, v_codes
        self.device = k_codes.device
        self.pages, self.page_size, self.kv_heads, self.head_dim = rows // page_size, page_size, kv_heads, head_dim
        self.desc = PagedCacheDesc(k_scales.data_ptr(), k_codes.data_ptr(), v_scales.data_ptr(), v_codes.data_ptr(),
                                   self.pages, page_size, kv_heads, head_dim)
        self._ref = ctypes.addressof(self.desc)
        self._index = cuda_index(self.device)
        self._key = (self.pages, page_size, kv_heads, head_dim)

    @classmethod
    def zeros(cls, pages: int, page_size: int, kv_heads: int, head_dim: int, device="cuda") -> "PagedCache":
        rows, width = pages * page_size, kv_heads * head_dim
        s = [torch.zeros(rows, width // GROUP, dtype=torch.float16, device=device) for _ in range(2)]
        c = [torch.zeros(rows, width, dtype=torch.uint8, device=device) for _ in range(2)]
        return cls(s[0], c[0], s[1], c[1], page_size=page_size, kv_heads=kv_heads, head_dim=head_dim)


class PagedBatch:
    """The tokens of one step: query_starts [sequences + 1], context_lens [sequences] and page_table
    [sequences, entries], int32 on the device (see qwc_paged_batch). `max_query` and `max_context`
    bound what they hold; the arrays may change on the device between calls."""

    def __init__(self, query_starts: torch.Tensor, context_lens: torch.Tensor, page_table: torch.Tensor, *, tokens: int,
                 max_query: int, max_context: int):
        for t in (query_starts, context_lens, page_table):
            if t.dtype != torch.int32 or t.device != query_starts.device:
                refuse("invalid_argument", "PagedBatch")
        n = context_lens.numel()
        if (query_starts.shape != (n + 1,) or context_lens.shape != (n,) or page_table.dim() != 2
                or page_table.shape[0] != n or min(tokens, max_query, max_context) < 0):
            refuse("shape_mismatch", "PagedBatch")
        if not (query_starts.is_contiguous() and context_lens.is_contiguous()
                and (page_table.stride(1) == 1 or page_table.shape[1] <= 1)):
            refuse("invalid_argument", "PagedBatch")
        self.query_starts, self.context_lens, self.page_table = query_starts, context_lens, page_table
        self.device, self.tokens = query_starts.device, tokens
        # A view's rows may lie further apart than they are long (or be one row): the length bounds what is read.
        entries = page_table.shape[1]
        self.desc = PagedBatchDesc(query_starts.data_ptr(), context_lens.data_ptr(), page_table.data_ptr(), n, tokens,
                                   page_table.stride(0) if n > 1 and entries else entries, max_query, max_context, entries)
        self._ref = ctypes.addressof(self.desc)
        self._workspace_bytes: dict = {}


def _rows(t: torch.Tensor, batch: PagedBatch, heads: int, dim: int, call: str) -> int:
    """The row stride of a [tokens, heads, dim] tensor whose rows are whole (a view of wider rows is fine)."""
    if t.shape != (batch.tokens, heads, dim):
        refuse("shape_mismatch", call)
    if t.device != batch.device:
        refuse("invalid_argument", call)
    row, head, one = t.stride()
    if (one != 1 and dim > 1) or (head != dim and heads > 1):
        refuse("invalid_argument", call)
    return row if batch.tokens > 1 else heads * dim  # (nothing is a stride away from the only row)


def _table(t: torch.Tensor, shape: tuple, device: torch.device, call: str) -> None:
    """f32 values of `shape` (rotation tables, norm weights)."""
    if t.shape != shape:
        refuse("shape_mismatch", call)
    if t.dtype != torch.float32 or t.device != device or not t.is_contiguous():
        refuse("invalid_argument", call)


# Partial results of attention, one buffer for each (device, stream), kept at the largest size asked for.
_workspaces: dict = {}


def _new_workspace(need: int, device: torch.device) -> torch.Tensor:
    buffer = torch.empty(need, dtype=torch.uint8, device=device)
    buffer[:PAGED_WORKSPACE_HEAD].zero_()
    return buffer


def workspace_bytes(cache: PagedCache, batch: PagedBatch, heads: int, fmt: int) -> int:
    key = (cache._key, fmt, heads)
    need = batch._workspace_bytes.get(key)
    if need is None:
        n = ctypes.c_uint64(0)
        check(lib().qwc_op_paged_attention_workspace(cache._ref, batch._ref, fmt, heads, ctypes.byref(n)),
              "qwc_op_paged_attention_workspace")
        need = batch._workspace_bytes[key] = n.value
    return need


def workspace(cache: PagedCache, batch: PagedBatch, heads: int, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """A workspace for `attention` with this pool, batch and head count, to be used by one stream at a time."""
    fmt = FORMATS.get(dtype)
    if fmt is None:
        refuse("unsupported", "qwc_op_paged_attention_workspace")
    return _new_workspace(workspace_bytes(cache, batch, heads, fmt), cache.device)


def _workspace(cache: PagedCache, need: int, stream: int) -> tuple[int, int, torch.Tensor]:
    """(address, bytes, tensor) of the stream's buffer, at least what this call needs. The caller holds the tensor until
    its launch is enqueued: another thread on the stream may put a larger one in its place at any time. (After the launch
    the order of the stream keeps it.)"""
    if torch.cuda.is_current_stream_capturing():
        # A graph may be replayed on any stream and outlive the stream's buffer: it gets one of its own, from the
        # graph's pool, and zeroes its head in each replay.
        buffer = _new_workspace(need, cache.device)
        return buffer.data_ptr(), need, buffer
    at = (cache._index, stream)
    held = _workspaces.get(at)
    if held is None or held[1] < need:
        buffer = _new_workspace(need, cache.device)
        if held is not None:
            buffer[:4].copy_(held[2][:4])  # a wait that ran out is still to be told of
        held = _workspaces[at] = (buffer.data_ptr(), need, buffer)
    return held


def check_waits(workspace: torch.Tensor | None = None, device: torch.device | None = None) -> None:
    """Raises `QwcError` if a bounded wait inside an attention kernel ran out (its rows are undefined then), and makes
    the workspace ready again. Without a workspace, of the current stream's own. Waits for the stream. (The workspace that a
    captured graph makes for itself is not kept and cannot be asked: capture with one of the caller's.)"""
    if workspace is None:
        if device is None or device.index is None:
            device = torch.device("cuda", torch.cuda.current_device())
        held = _workspaces.get((device.index, current_stream(device)))
        if held is None:
            return
        workspace = held[2]
    if int(workspace[:4].view(torch.int32)[0]):
        workspace[:PAGED_WORKSPACE_HEAD].zero_()
        refuse("invalid_state", "qwc_op_paged_attention")


def append(cache: PagedCache, batch: PagedBatch, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cos: torch.Tensor,
           sin: torch.Tensor, *, q_norm: torch.Tensor | None = None, k_norm: torch.Tensor | None = None,
           eps: float = 1e-6, q_out: torch.Tensor | None = None) -> torch.Tensor:
    """QK-RMSNorm, rotation and the q8 append of [tokens, heads, head_dim] rows; returns the queries
    for attention (`q_out`, a new tensor unless given; may be `q`)."""
    call = "qwc_op_paged_append"
    away = elsewhere(cache._index, call)
    if away is not None:
        with away:
            return append(cache, batch, q, k, v, cos, sin, q_norm=q_norm, k_norm=k_norm, eps=eps, q_out=q_out)
    fmt = format_of(q, call)
    dtype, device = q.dtype, batch.device
    if k.dtype != dtype or v.dtype != dtype or cache.device != device or q.dim() != 3:
        refuse("invalid_argument", call)
    heads, dim, kv_heads = q.shape[1], cache.head_dim, cache.kv_heads
    q_stride, k_stride = _rows(q, batch, heads, dim, call), _rows(k, batch, kv_heads, dim, call)
    v_stride = _rows(v, batch, kv_heads, dim, call)
    if q_out is None:
        q_out, out_stride = torch.empty((batch.tokens, heads, dim), dtype=dtype, device=device), heads * dim
    elif q_out.dtype != dtype:
        refuse("invalid_argument", call)
    else:
        out_stride = _rows(q_out, batch, heads, dim, call)
    rope_rows = cos.shape[0]
    _table(cos, (rope_rows, dim // 2), device, call)
    _table(sin, (rope_rows, dim // 2), device, call)
    if q_norm is not None:
        _table(q_norm, (dim,), device, call)
    if k_norm is not None:
        _table(k_norm, (dim,), device, call)
    st = lib().qwc_op_paged_append(
        cache._ref, batch._ref, fmt, q.data_ptr(), q_stride, k.data_ptr(), k_stride, v.data_ptr(), v_stride, heads,
        None if q_norm is None else q_norm.data_ptr(), None if k_norm is None else k_norm.data_ptr(), eps, cos.data_ptr(),
        sin.data_ptr(), rope_rows, q_out.data_ptr(), out_stride, current_stream(device))
    if st:
        check(st, call)
    return q_out


def attention(cache: PagedCache, batch: PagedBatch, q: torch.Tensor, out: torch.Tensor | None = None,
              workspace: torch.Tensor | None = None) -> torch.Tensor:
    """Causal attention of the batch's [tokens, heads, head_dim] queries over their sequences' pages. `workspace`: one
    made by `workspace(...)`; without it, the current stream's own (in a graph under capture, the graph's own)."""
    call = "qwc_op_paged_attention"
    away = elsewhere(cache._index, call)
    if away is not None:
        with away:
            return attention(cache, batch, q, out, workspace)
    fmt = format_of(q, call)
    if cache.device != batch.device or q.dim() != 3:
        refuse("invalid_argument", call)
    heads, dim = q.shape[1], cache.head_dim
    q_stride = _rows(q, batch, heads, dim, call)
    if out is None:
        out, out_stride = torch.empty((batch.tokens, heads, dim), dtype=q.dtype, device=q.device), heads * dim
    elif out.dtype != q.dtype:
        refuse("invalid_argument", call)
    else:
        out_stride = _rows(out, batch, heads, dim, call)
    stream = current_stream(cache.device)
    if workspace is None:
        work, size, held = _workspace(cache, workspace_bytes(cache, batch, heads, fmt), stream)  # noqa: F841 (held until the launch)
    elif workspace.dtype != torch.uint8 or workspace.device != cache.device or not workspace.is_contiguous():
        refuse("invalid_argument", call)
    else:
        work, size = workspace.data_ptr(), workspace.numel()
    st = lib().qwc_op_paged_attention(cache._ref, batch._ref, fmt, q.data_ptr(), q_stride, heads, out.data_ptr(), out_stride,
                                      work, size, stream)
    if st:
        check(st, call)
    return out


def read(cache: PagedCache, batch: PagedBatch, dtype: torch.dtype = torch.float32, k_out: torch.Tensor | None = None,
         v_out: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """The cached key and value rows of the batch's tokens as values, [tokens, kv_heads, head_dim]."""
    call = "qwc_op_paged_read"
    away = elsewhere(cache._index, call)
    if away is not None:
        with away:
            return read(cache, batch, dtype, k_out, v_out)
    tokens, kv_heads, dim, device = batch.tokens, cache.kv_heads, cache.head_dim, batch.device
    if cache.device != device:
        refuse("invalid_argument", call)
    if k_out is None:
        k_out, k_stride = torch.empty((tokens, kv_heads, dim), dtype=dtype, device=device), kv_heads * dim
    else:
        k_stride = _rows(k_out, batch, kv_heads, dim, call)
    if v_out is None:
        v_out, v_stride = torch.empty((tokens, kv_heads, dim), dtype=dtype, device=device), kv_heads * dim
    else:
        v_stride = _rows(v_out, batch, kv_heads, dim, call)
    fmt = format_of(k_out, call)
    if k_out.dtype != v_out.dtype:
        refuse("invalid_argument", call)
    st = lib().qwc_op_paged_read(cache._ref, batch._ref, fmt, k_out.data_ptr(), k_stride, v_out.data_ptr(), v_stride,
                                 current_stream(device))
    if st:
        check(st, call)
    return k_out, v_out
