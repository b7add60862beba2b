"""Attention of each request's new tokens over its pages of the pool.

The step after a link: a chunk of a prompt behind the linked context, or one
new token of every request of a decode batch, over the pool that the link and
``append_rotated_kv_inplace`` write.  The reference leaves it to its runtime's
attention backend (native decode and extend, patched_sglang_files/python/sglang/
srt/model_executor/model_runner.py:3264); here it is hand-written gfx950 kernels
behind ``ll_paged_attention``.

Lengths, query starts and pages stay on the device: nothing is planned on the
host, no call synchronises, and a captured call serves every length that its
page table holds.
"""

from __future__ import annotations

import math
from typing import Optional

import torch

from . import _native

_DTYPES = {torch.float16: _native.DTYPE_FLOAT16, torch.bfloat16: _native.DTYPE_BFLOAT16}
_INDEX_DTYPES = {torch.int32: _native.DTYPE_INT32, torch.int64: _native.DTYPE_INT64}


# The call in one native call where it takes it (an output of its own among
# others is left to the Python checks, which also name the reason where a call
# must not run).
_calls = _native.step_calls()


class PagedAttentionError(RuntimeError):
    """A paged attention call that must not run."""


def _check_counts(name: str, counts: torch.Tensor, size: int, device: torch.device) -> None:
    if counts.ndim != 1 or int(counts.numel()) != size or counts.device != device or not counts.is_contiguous():
        raise PagedAttentionError(f"{name} must be a contiguous vector of {size} entries on the query's device")
    if counts.dtype not in _INDEX_DTYPES:
        raise PagedAttentionError(f"{name} must be int32 or int64")


def paged_attention(query: torch.Tensor, key_buffer: torch.Tensor, value_buffer: torch.Tensor,
                    page_table: torch.Tensor, kv_lengths: torch.Tensor, *, page_size: int = 1,
                    query_starts: Optional[torch.Tensor] = None, scale: Optional[float] = None,
                    output: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One layer's attention of ``query`` [queries, q heads, dim] (fp16 or bf16,
    dim 64, 128 or 256; any token and head strides, as a view of a fused
    projection has) over ``key_buffer`` / ``value_buffer`` [slots, kv heads, dim].

    ``page_table`` int32 [requests, pages]: key j of request r is row
    ``page_table[r, j // page_size] * page_size + j % page_size`` (page size 1:
    rows of the runtime's ``req_to_token``).  ``kv_lengths`` [requests] counts
    each request's keys, its new ones among them.  ``query_starts`` [requests +
    1] says where each request's queries begin; without it each request has one.
    Query i of a request's n sees its keys up to position length - n + i, itself
    included.  ``scale`` is 1 / sqrt(dim) by default, and in [1e-37, 1e30).

    Returns (or fills, with ``output``) [queries, q heads, dim].  A query that
    sees no key gets zeros; rows of no request keep what they held (undefined in
    a new tensor).  Pages outside the pool are invisible.  A call suits its average
    request: a chunk among many single tokens, or beside many rows without queries,
    is faster in a call of its own.  Work goes to the
    current stream; the call's workspace comes from torch's allocator and belongs
    to that stream (or to the graph that captures the call).
    """

    if _calls is not None and output is None and query.is_cuda:
        current = torch._C._cuda_getDevice()
        done = _calls.paged_attention(
            _native.entry_address("ll_paged_attention"), torch._C._cuda_getCurrentRawStream(current), current,
            _native.entry_address("ll_paged_attention_workspace_bytes"), query, key_buffer, value_buffer, page_table,
            kv_lengths, page_size, query_starts, scale)
        if type(done) is int:
            _native.check_status(done)
        elif done is not None:
            return done
    if _native.differentiated(query, key_buffer, value_buffer, output):
        raise PagedAttentionError("paged attention has no gradient: call it under torch.no_grad()")
    device, dtype = query.device, query.dtype
    if dtype not in _DTYPES:
        raise PagedAttentionError(f"unsupported query dtype: {dtype} (fp16 or bf16)")
    if key_buffer.dtype != dtype or value_buffer.dtype != dtype:
        raise PagedAttentionError("query, key_buffer and value_buffer must have one dtype")
    if query.ndim != 3 or key_buffer.ndim != 3 or value_buffer.shape != key_buffer.shape:
        raise PagedAttentionError("query must be [queries, q heads, dim] and the buffers [slots, kv heads, dim]")
    (queries, q_heads, dim), (slots, kv_heads, key_dim) = query.shape, key_buffer.shape
    if dim != key_dim or dim not in (64, 128, 256):
        raise PagedAttentionError(f"one head dim of 64, 128 or 256 is needed, got {dim} and {key_dim}")
    if kv_heads < 1 or q_heads < 1 or q_heads % kv_heads:
        raise PagedAttentionError("the query heads must be a multiple of the KV heads")
    for name, buffer in (("key_buffer", key_buffer), ("value_buffer", value_buffer)):
        if buffer.device != device or not buffer.is_contiguous() or buffer.data_ptr() % 16:
            raise PagedAttentionError(f"{name} must be contiguous, 16-byte aligned and on the query's device")
    if page_table.ndim != 2 or page_table.dtype != torch.int32 or page_table.device != device or (
            page_table.shape[1] > 1 and page_table.stride(1) != 1):
        raise PagedAttentionError("page_table must be int32 [requests, pages] with dense rows on the query's device")
    requests, pages = page_table.shape
    page_size = _native.whole_number(page_size)
    if page_size is None or page_size < 1:
        raise PagedAttentionError("page_size must be positive and whole")
    _check_counts("kv_lengths", kv_lengths, requests, device)
    if query_starts is not None:
        _check_counts("query_starts", query_starts, requests + 1, device)
    elif queries != requests:
        raise PagedAttentionError("without query_starts every request has one query")
    scale = 1.0 / math.sqrt(dim) if scale is None else float(scale)
    if not 1e-37 <= scale < 1e30:  # a normal number in the kernels' fp32
        raise PagedAttentionError("scale must be in [1e-37, 1e30)")
    if output is None:
        output = torch.empty((queries, q_heads, dim), dtype=dtype, device=device)
    elif output.shape != query.shape or output.dtype != dtype or output.device != device or (
            not output.is_contiguous() or output.data_ptr() % 16):
        raise PagedAttentionError("output must be contiguous, 16-byte aligned and of the query's shape, dtype and device")
    elif any(_meets(output, other) for other in (query, key_buffer, value_buffer, page_table, kv_lengths, query_starts)
             if other is not None):
        raise PagedAttentionError("output must not overlap the call's other tensors")
    if device.type != "cuda":
        raise PagedAttentionError("device tensors are required")
    if query.stride(2) != 1 or query.stride(0) % 8 or query.stride(1) % 8 or query.data_ptr() % 16:
        query = query.clone(memory_format=torch.contiguous_format)  # the kernels read 16-byte chunks
    args = _native.PagedAttentionArgs()
    args.query = query.data_ptr()
    args.query_token_stride, args.query_head_stride = query.stride(0), query.stride(1)
    args.output = output.data_ptr()
    args.num_queries = queries
    args.key_buffer, args.value_buffer = key_buffer.data_ptr(), value_buffer.data_ptr()
    args.num_slots = slots
    args.num_q_heads, args.num_kv_heads, args.head_dim = q_heads, kv_heads, dim
    args.kv_dtype = _DTYPES[dtype]
    args.softmax_scale = scale
    args.page_table = page_table.data_ptr()
    args.page_table_stride, args.page_table_columns = page_table.stride(0), pages
    args.page_size = page_size
    args.kv_lengths, args.kv_lengths_dtype = kv_lengths.data_ptr(), _INDEX_DTYPES[kv_lengths.dtype]
    if query_starts is not None:
        args.query_starts, args.query_starts_dtype = query_starts.data_ptr(), _INDEX_DTYPES[query_starts.dtype]
    args.num_requests = requests
    with _native.on_device(device):
        needed = _native.paged_attention_workspace_bytes(args)
        if needed:
            workspace = torch.empty(needed, dtype=torch.uint8, device=device)
            args.workspace, args.workspace_bytes = workspace.data_ptr(), needed
        _native.paged_attention(args, _native.stream_handle(None, device))
    return output


def _meets(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Do the spans of two tensors share bytes?"""

    def span(t: torch.Tensor) -> tuple[int, int]:
        reach = sum((size - 1) * stride for size, stride in zip(t.shape, t.stride()))
        return t.data_ptr(), t.data_ptr() + (reach + 1) * t.element_size()

    if a.numel() == 0 or b.numel() == 0:
        return False
    (a_begin, a_end), (b_begin, b_end) = span(a), span(b)
    return a_begin < b_end and b_begin < a_end
