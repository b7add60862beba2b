"""A paged pool held in 8 bits: written, linked, read back and attended.

One layer's keys and values are codes of ``torch.float8_e4m3fn`` [slots, kv
heads, dim], with a scale of ``torch.float8_e8m0fnu`` (a power of two) for each
head of every ``scale_block`` slots, [slots // scale_block, kv heads]: a row's
value is its code times its block's scale.  The reference's pool holds its model's
own type only (patched_sglang_files/python/sglang/srt/pic_runtime.py:6283-6289);
this one takes half the memory of it, and a decode step reads half as much.

* ``append_quantized_kv_inplace``: a step's new tokens into the pool, as
  ``append_rotated_kv_inplace`` does for a 16-bit pool;
* ``link_quantized_kv_inplace``: cached rows to a new request's slots, their keys
  turned to their new positions, as ``fused_kv_link_inplace`` does;
* ``load_quantized_kv``: rows back in 16 or 32 bits, for the repair pass and for
  pools of the model's type;
* ``quantized_paged_attention``: ``paged_attention`` over this pool's pages.

A pool that holds nothing is zeros in codes and scales.  Rows that a call adds to a
block raise its scale where they need it (the rows that it held are rounded again
under it) and never lower it, unless the call writes the whole block.  So who gives
a block to another request clears its scales first::

    key_scales.view(torch.uint8)[blocks] = 0      # and value_scales

or the new rows may be rounded under the scale of the old ones (and are NaN under a
byte of 255).  Only a block that one call writes whole needs no clearing: a link with a
repair mask leaves rows out, and a prompt's last block is mostly partial.

Everything is enqueued on the current stream; no call synchronises, and all may be
captured into a HIP graph.  Inference only: tensors that need a gradient or carry a
forward-mode tangent are refused.
"""

from __future__ import annotations

import math
from typing import Optional, Sequence

import torch

from . import _native
from .head_rotary import _overlap

CODE_DTYPE = torch.float8_e4m3fn
SCALE_DTYPE = torch.float8_e8m0fnu

_HALF_DTYPES = {torch.float16: _native.DTYPE_FLOAT16, torch.bfloat16: _native.DTYPE_BFLOAT16}
_FLOAT_DTYPES = {**_HALF_DTYPES, torch.float32: _native.DTYPE_FLOAT32}
_INDEX_DTYPES = {torch.int32: _native.DTYPE_INT32, torch.int64: _native.DTYPE_INT64}
_MOST_BLOCK = 128


# Each call in one native call where it takes it; the Python checks take the others,
# and name the reason where a call must not run.
_calls = _native.step_calls()


class QuantizedPoolError(RuntimeError):
    """A call over an 8-bit pool that must not run."""


def _native_call(call, name: str, *arguments):
    """What the native call made of it: its result, or None where it did not take it."""

    device = torch._C._cuda_getDevice()
    done = call(_native.entry_address(name), torch._C._cuda_getCurrentRawStream(device), device, *arguments)
    if type(done) is int:
        _native.check_status(done)
    return done


def _refuse_gradients(*tensors: Optional[torch.Tensor]) -> None:
    if _native.differentiated(*tensors):
        raise QuantizedPoolError("these operators have no gradient: call them under torch.no_grad()")


def _meets(tensor: torch.Tensor, others: Sequence[Optional[torch.Tensor]]) -> bool:
    return any(other is not None and _overlap(tensor, other) for other in others)


def _check_pool(key_buffer: torch.Tensor, value_buffer: torch.Tensor, key_scales: torch.Tensor,
                value_scales: torch.Tensor, scale_block: int) -> int:
    """Checks the pool's four tensors; returns ``scale_block`` as an int."""

    block = _native.whole_number(scale_block)
    if block is None or not 1 <= block <= _MOST_BLOCK or block & (block - 1):
        raise QuantizedPoolError(f"scale_block must be a power of two, at most {_MOST_BLOCK}")
    if key_buffer.ndim != 3 or value_buffer.shape != key_buffer.shape:
        raise QuantizedPoolError("the buffers must be [slots, kv heads, dim] of one shape")
    slots, heads, dim = key_buffer.shape
    if slots % block:
        raise QuantizedPoolError(f"the pool must be whole blocks of {block} slots, got {slots} slots")
    if heads < 1 or dim < 16 or dim > 256 or dim % 16:
        raise QuantizedPoolError("head dims are multiples of 16, at most 256")
    for name, buffer in (("key_buffer", key_buffer), ("value_buffer", value_buffer)):
        if buffer.dtype != CODE_DTYPE:
            raise QuantizedPoolError(f"{name} must be {CODE_DTYPE}, got {buffer.dtype}")
        if buffer.device != key_buffer.device or not buffer.is_contiguous() or buffer.data_ptr() % 16:
            raise QuantizedPoolError(f"{name} must be contiguous, 16-byte aligned and on the pool's device")
    for name, scales in (("key_scales", key_scales), ("value_scales", value_scales)):
        if scales.dtype != SCALE_DTYPE or tuple(scales.shape) != (slots // block, heads):
            raise QuantizedPoolError(f"{name} must be {SCALE_DTYPE} [{slots // block}, {heads}], got {scales.dtype} "
                                     f"{list(scales.shape)}")
        if scales.device != key_buffer.device or not scales.is_contiguous():
            raise QuantizedPoolError(f"{name} must be contiguous and on the pool's device")
    return block


def _fill_pool(pool: _native.QuantizedPool, key_buffer: torch.Tensor, value_buffer: torch.Tensor,
               key_scales: torch.Tensor, value_scales: torch.Tensor, block: int) -> None:
    pool.key_buffer, pool.value_buffer = key_buffer.data_ptr(), value_buffer.data_ptr()
    pool.key_scales, pool.value_scales = key_scales.data_ptr(), value_scales.data_ptr()
    pool.num_slots, pool.num_kv_heads, pool.head_dim = key_buffer.shape
    pool.scale_block = block


def _check_written_pool(tensors: Sequence[torch.Tensor], others: Sequence[Optional[torch.Tensor]]) -> None:
    """The pool's four tensors, which the call writes, share no bytes with each
    other or with the call's other tensors."""

    for i, tensor in enumerate(tensors):
        if _meets(tensor, tensors[:i]) or _meets(tensor, others):
            raise QuantizedPoolError("the pool's tensors must not overlap each other or the call's other tensors")


def _check_rows(name: str, rows: torch.Tensor, shape: tuple, dtype: torch.dtype, device: torch.device) -> None:
    if rows.ndim != 3 or rows.shape[1] < 1 or any(want not in (None, got) for want, got in zip(shape, rows.shape)):
        raise QuantizedPoolError(f"{name} must be [tokens, heads, dim] of {shape}, got {list(rows.shape)}")
    if rows.dtype != dtype:
        raise QuantizedPoolError(f"{name} must be {dtype} as the query, got {rows.dtype}")
    if rows.device != device:
        raise QuantizedPoolError(f"{name} must be on the pool's device")


def _in_chunks(rows: torch.Tensor) -> bool:
    """Can the kernels read (or write) these rows in 16-byte chunks?"""

    return rows.stride(2) == 1 and rows.stride(0) % 8 == 0 and rows.stride(1) % 8 == 0 and rows.data_ptr() % 16 == 0


def _check_vector(name: str, values: torch.Tensor, count: int, device: torch.device, dtypes=_INDEX_DTYPES) -> None:
    if values.ndim != 1 or int(values.numel()) != count or values.device != device or not values.is_contiguous():
        raise QuantizedPoolError(f"{name} must be a contiguous vector of {count} entries on the pool's device")
    if values.dtype not in dtypes:
        raise QuantizedPoolError(f"{name} must be one of {', '.join(str(dtype) for dtype in dtypes)}")


def _check_table(cos_sin_cache: torch.Tensor, rotary_dim: int, dim: int, device: torch.device) -> int:
    rotary = _native.whole_number(rotary_dim)
    if rotary is None or rotary < 16 or rotary % 16 or rotary > dim:
        raise QuantizedPoolError("rotary_dim must be a multiple of 16 and in [16, head dim]")
    if cos_sin_cache.ndim != 2 or int(cos_sin_cache.shape[1]) < rotary or cos_sin_cache.device != device:
        raise QuantizedPoolError("cos_sin_cache must be [positions, >= rotary_dim] on the pool's device")
    if cos_sin_cache.dtype not in _FLOAT_DTYPES or cos_sin_cache.stride(1) != 1:
        raise QuantizedPoolError("cos_sin_cache must be fp32, fp16 or bf16 with dense rows")
    return rotary


def _fill_table(args, cos_sin_cache: torch.Tensor, rotary: int, is_neox_style: bool) -> None:
    args.cos_sin_cache = cos_sin_cache.data_ptr()
    args.cos_sin_dtype = _FLOAT_DTYPES[cos_sin_cache.dtype]
    args.cos_sin_rows, args.cos_sin_cols = cos_sin_cache.shape
    args.cos_sin_stride_row = cos_sin_cache.stride(0)
    args.rotary_dim = rotary
    args.is_neox_style = 1 if is_neox_style else 0


def _check_counter(skipped_rows: Optional[torch.Tensor], device: torch.device,
                   others: Sequence[Optional[torch.Tensor]]) -> None:
    if skipped_rows is None:
        return
    if skipped_rows.dtype != torch.int64 or skipped_rows.numel() != 1 or skipped_rows.device != device:
        raise QuantizedPoolError("skipped_rows must be a one-element int64 tensor on the pool's device")
    if _meets(skipped_rows, others):
        raise QuantizedPoolError("skipped_rows must not overlap the call's other tensors")


def _launch(call, args, device: torch.device) -> None:
    if device.type != "cuda":
        raise QuantizedPoolError("device tensors are required")
    with _native.on_device(device):
        call(args, _native.stream_handle(None, device))


def append_quantized_kv_inplace(*, key_buffer: torch.Tensor, value_buffer: torch.Tensor, key_scales: torch.Tensor,
                                value_scales: torch.Tensor, scale_block: int, destination_slots: torch.Tensor,
                                query: torch.Tensor, key: torch.Tensor, value: torch.Tensor,
                                positions: torch.Tensor, cos_sin_cache: torch.Tensor, rotary_dim: int,
                                is_neox_style: bool = True, query_norm_weight: Optional[torch.Tensor] = None,
                                key_norm_weight: Optional[torch.Tensor] = None, norm_eps: float = 1e-6,
                                query_output: Optional[torch.Tensor] = None,
                                skipped_rows: Optional[torch.Tensor] = None) -> torch.Tensor:
    """A step's new tokens into one layer of the pool: ``query`` [tokens, q heads,
    dim] and ``key`` [tokens, kv heads, dim] (fp16 or bf16; any strides, as views
    of a fused projection have) are normed for each head by the given weights and
    turned to ``positions``; the keys and ``value`` [tokens, kv heads, dim] go to
    the rows ``destination_slots`` in 8 bits.  Returns the queries (or fills
    ``query_output``, which may be the query itself).

    The slots that are written must be pairwise distinct, and those of one block
    stand next to each other in the call, as a request's new tokens do: in any
    order, with padding between them or not, but no row of another block (not
    checked: what a block holds whose rows do not is undefined).  A
    negative slot is padding (its queries are turned, nothing is written), a slot
    past the pool likewise and counted in ``skipped_rows``; a token whose position
    is outside the table is left out whole and counted.  ``rotary_dim`` is a
    multiple of 16.
    """

    if _calls is not None and query.is_cuda:
        done = _native_call(_calls.quantized_append, "ll_quantized_append", query, key, positions, cos_sin_cache,
                            rotary_dim, is_neox_style, query_norm_weight, key_norm_weight, norm_eps, skipped_rows,
                            query_output, value, destination_slots, key_buffer, value_buffer, key_scales, value_scales,
                            scale_block)
        if done is not None:
            return done
    _refuse_gradients(query, key, value, query_norm_weight, key_norm_weight, cos_sin_cache, query_output, key_buffer,
                      value_buffer, key_scales, value_scales)
    block = _check_pool(key_buffer, value_buffer, key_scales, value_scales, scale_block)
    device, dtype = key_buffer.device, query.dtype
    if dtype not in _HALF_DTYPES:
        raise QuantizedPoolError(f"unsupported query dtype: {dtype} (fp16 or bf16)")
    heads, dim = key_buffer.shape[1:]
    tokens = int(query.shape[0]) if query.ndim else 0
    _check_rows("query", query, (tokens, None, dim), dtype, device)
    _check_rows("key", key, (tokens, heads, dim), dtype, device)
    _check_rows("value", value, (tokens, heads, dim), dtype, device)
    _check_vector("positions", positions, tokens, device)
    _check_vector("destination_slots", destination_slots, tokens, device)
    rotary = _check_table(cos_sin_cache, rotary_dim, dim, device)
    weights = [weight for weight in (query_norm_weight, key_norm_weight) if weight is not None]
    for weight in weights:
        _check_vector("a norm weight", weight, dim, device, _FLOAT_DTYPES)
        if weight.dtype != weights[0].dtype:
            raise QuantizedPoolError("norm weights must be of one type")
    if not float(norm_eps) >= 0.0:
        raise QuantizedPoolError("norm_eps must not be negative")
    pool = (key_buffer, value_buffer, key_scales, value_scales)
    beside = (positions, destination_slots, cos_sin_cache, query_norm_weight, key_norm_weight)
    _check_counter(skipped_rows, device, (query, key, value, *pool, *beside))
    _check_written_pool(pool, (query, key, value, skipped_rows, *beside))
    output = query_output
    if output is None:
        output = torch.empty(query.shape, dtype=dtype, device=device)
    else:
        _check_rows("query_output", output, tuple(query.shape), dtype, device)
        if not _in_chunks(output):
            raise QuantizedPoolError("query_output's rows must be dense and begin at multiples of 16 bytes")
        _, q_heads, _ = output.shape
        token, head = output.stride(0), output.stride(1)
        if not (((q_heads == 1 or head >= dim) and (tokens <= 1 or token >= (q_heads - 1) * head + dim))
                or ((tokens <= 1 or token >= dim) and (q_heads == 1 or head >= (tokens - 1) * token + dim))):
            raise QuantizedPoolError("query_output's rows must not overlap each other")
        same = output.data_ptr() == query.data_ptr() and output.stride() == query.stride()
        if (not same and _overlap(output, query)) or _meets(output, (key, value, skipped_rows, *pool, *beside)):
            raise QuantizedPoolError("query_output must be the query itself or not overlap the call's tensors")
    # The kernel reads 16-byte chunks.
    query, key, value = (rows if _in_chunks(rows) else rows.clone(memory_format=torch.contiguous_format)
                         for rows in (query, key, value))
    query_norm_weight, key_norm_weight = (weight if weight is None or weight.data_ptr() % 16 == 0 else weight.clone()
                                          for weight in (query_norm_weight, key_norm_weight))
    args = _native.QuantizedAppendArgs()
    _fill_pool(args.pool, *pool, block)
    args.num_tokens, args.num_q_heads, args.dtype = tokens, query.shape[1], _HALF_DTYPES[dtype]
    for name, rows in (("query", query), ("query_output", output), ("key", key), ("value", value)):
        setattr(args, name, rows.data_ptr())
        setattr(args, f"{name}_token_stride", rows.stride(0))
        setattr(args, f"{name}_head_stride", rows.stride(1))
    args.destination_slots = destination_slots.data_ptr()
    args.destination_slots_dtype = _INDEX_DTYPES[destination_slots.dtype]
    args.positions, args.positions_dtype = positions.data_ptr(), _INDEX_DTYPES[positions.dtype]
    _fill_table(args, cos_sin_cache, rotary, is_neox_style)
    args.query_norm_weight = None if query_norm_weight is None else query_norm_weight.data_ptr()
    args.key_norm_weight = None if key_norm_weight is None else key_norm_weight.data_ptr()
    args.norm_weight_dtype = _FLOAT_DTYPES[weights[0].dtype] if weights else 0
    args.norm_eps = float(norm_eps)
    args.skipped_rows = None if skipped_rows is None else skipped_rows.data_ptr()
    _launch(_native.quantized_append, args, device)
    return output


def link_quantized_kv_inplace(*, key_buffer: torch.Tensor, value_buffer: torch.Tensor, key_scales: torch.Tensor,
                              value_scales: torch.Tensor, scale_block: int, source_slots: torch.Tensor,
                              destination_slots: torch.Tensor, local_positions: torch.Tensor,
                              global_positions: torch.Tensor, cos_sin_cache: torch.Tensor, rotary_dim: int,
                              is_neox_style: bool = True, prefix_token_count: int = 0,
                              repair_mask: Optional[torch.Tensor] = None,
                              skipped_rows: Optional[torch.Tensor] = None) -> None:
    """Link one layer in place: for every token t (left out where ``repair_mask``
    is set) row ``source_slots[t]`` goes to row ``destination_slots[t]``, its key
    turned from ``local_positions[t]`` to ``global_positions[t]`` unless t is below
    ``prefix_token_count``.

    Destinations are as in ``append_quantized_kv_inplace``; no source lies in a
    block that the call writes.  Slots are of one integer type, positions too.
    Tokens with an index out of range are left out and counted in
    ``skipped_rows``; a negative destination is padding.
    """

    if _calls is not None and key_buffer.is_cuda:
        if _native_call(_calls.quantized_link, "ll_quantized_link", key_buffer, value_buffer, key_scales, value_scales,
                        scale_block, source_slots, destination_slots, local_positions, global_positions, cos_sin_cache,
                        rotary_dim, is_neox_style, prefix_token_count, repair_mask, skipped_rows) is not None:
            return
    _refuse_gradients(key_buffer, value_buffer, key_scales, value_scales, cos_sin_cache)
    block = _check_pool(key_buffer, value_buffer, key_scales, value_scales, scale_block)
    device, tokens = key_buffer.device, int(source_slots.numel())
    for name, values in (("source_slots", source_slots), ("destination_slots", destination_slots),
                         ("local_positions", local_positions), ("global_positions", global_positions)):
        _check_vector(name, values, tokens, device)
    if source_slots.dtype != destination_slots.dtype or local_positions.dtype != global_positions.dtype:
        raise QuantizedPoolError("both slots must be of one type, and both positions")
    if repair_mask is not None:
        _check_vector("repair_mask", repair_mask, tokens, device, (torch.bool, torch.uint8))
    prefix = _native.whole_number(prefix_token_count)
    if prefix is None or not 0 <= prefix <= tokens:
        raise QuantizedPoolError("prefix_token_count must be in [0, tokens]")
    rotary = _check_table(cos_sin_cache, rotary_dim, key_buffer.shape[2], device)
    pool = (key_buffer, value_buffer, key_scales, value_scales)
    beside = (source_slots, destination_slots, local_positions, global_positions, repair_mask, cos_sin_cache)
    _check_counter(skipped_rows, device, (*pool, *beside))
    _check_written_pool(pool, (skipped_rows, *beside))
    args = _native.QuantizedLinkArgs()
    _fill_pool(args.pool, *pool, block)
    args.num_tokens = tokens
    args.source_slots, args.destination_slots = source_slots.data_ptr(), destination_slots.data_ptr()
    args.slots_dtype = _INDEX_DTYPES[source_slots.dtype]
    args.local_positions, args.global_positions = local_positions.data_ptr(), global_positions.data_ptr()
    args.positions_dtype = _INDEX_DTYPES[local_positions.dtype]
    args.repair_mask = None if repair_mask is None else repair_mask.data_ptr()
    args.prefix_token_count = prefix
    _fill_table(args, cos_sin_cache, rotary, is_neox_style)
    args.skipped_rows = None if skipped_rows is None else skipped_rows.data_ptr()
    _launch(_native.quantized_link, args, device)


def load_quantized_kv(key_buffer: torch.Tensor, value_buffer: torch.Tensor, key_scales: torch.Tensor,
                      value_scales: torch.Tensor, *, scale_block: int, slots: Optional[torch.Tensor] = None,
                      dtype: torch.dtype = torch.bfloat16, key_output: Optional[torch.Tensor] = None,
                      value_output: Optional[torch.Tensor] = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Rows ``slots`` of the pool (all of them by default) as the values they stand
    for, in ``dtype`` (fp16, bf16 or fp32): (keys, values), each [rows, kv heads,
    dim], new or ``key_output`` and ``value_output`` filled.  A slot outside the
    pool gives zeros."""

    if _calls is not None and key_output is None and value_output is None and key_buffer.is_cuda:
        done = _native_call(_calls.quantized_load, "ll_quantized_load", key_buffer, value_buffer, key_scales,
                            value_scales, scale_block, slots, _FLOAT_DTYPES.get(dtype))
        if done is not None:
            return done
    _refuse_gradients(key_buffer, value_buffer, key_scales, value_scales, key_output, value_output)
    block = _check_pool(key_buffer, value_buffer, key_scales, value_scales, scale_block)
    device = key_buffer.device
    if dtype not in _FLOAT_DTYPES:
        raise QuantizedPoolError(f"unsupported dtype: {dtype} (fp16, bf16 or fp32)")
    rows = int(key_buffer.shape[0]) if slots is None else int(slots.numel())
    if slots is not None:
        _check_vector("slots", slots, rows, device)
    shape = (rows, *key_buffer.shape[1:])
    outputs = []
    for name, output in (("key_output", key_output), ("value_output", value_output)):
        if output is None:
            output = torch.empty(shape, dtype=dtype, device=device)
        elif tuple(output.shape) != shape or output.dtype != dtype or output.device != device or (
                not output.is_contiguous() or output.data_ptr() % 16):
            raise QuantizedPoolError(f"{name} must be a contiguous, 16-byte aligned {dtype} tensor {list(shape)} on the "
                                     "pool's device")
        elif _meets(output, (key_buffer, value_buffer, key_scales, value_scales, slots, *outputs)):
            raise QuantizedPoolError(f"{name} must not overlap the call's other tensors")
        outputs.append(output)
    if key_output is None and value_output is not None and _overlap(*outputs):
        raise QuantizedPoolError("the outputs must not overlap")
    args = _native.QuantizedLoadArgs()
    _fill_pool(args.pool, key_buffer, value_buffer, key_scales, value_scales, block)
    args.num_rows = rows
    if slots is not None:
        args.slots, args.slots_dtype = slots.data_ptr(), _INDEX_DTYPES[slots.dtype]
    args.key_output, args.value_output = (output.data_ptr() for output in outputs)
    args.dtype = _FLOAT_DTYPES[dtype]
    _launch(_native.quantized_load, args, device)
    return outputs[0], outputs[1]


def quantized_paged_attention(query: torch.Tensor, key_buffer: torch.Tensor, value_buffer: torch.Tensor,
                              key_scales: torch.Tensor, value_scales: torch.Tensor, page_table: torch.Tensor,
                              kv_lengths: torch.Tensor, *, scale_block: int, page_size: int,
                              query_starts: Optional[torch.Tensor] = None, scale: Optional[float] = None,
                              output: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``paged_attention`` over the pages of an 8-bit pool: ``query`` [queries, q
    heads, dim] (fp16 or bf16, dim 64, 128 or 256) over keys and values taken as
    ``load_quantized_kv`` gives them in the query's type.  ``page_table``,
    ``kv_lengths``, ``query_starts``, ``scale``, ``output`` and what is returned are
    as there; pages are whole blocks (``page_size`` a multiple of
    ``scale_block``), and blocks of 16 slots at least.  The call's workspace comes
    from torch's allocator and belongs to the current stream (or to the graph that
    captures the call).
    """

    if _calls is not None and output is None and query.is_cuda:
        done = _native_call(_calls.quantized_attention, "ll_quantized_attention",
                            _native.entry_address("ll_quantized_attention_workspace_bytes"), query, key_buffer,
                            value_buffer, key_scales, value_scales, scale_block, page_table, kv_lengths, page_size,
                            query_starts, scale)
        if done is not None:
            return done
    _refuse_gradients(query, key_buffer, value_buffer, key_scales, value_scales, output)
    block = _check_pool(key_buffer, value_buffer, key_scales, value_scales, scale_block)
    device, dtype = key_buffer.device, query.dtype
    if dtype not in _HALF_DTYPES:
        raise QuantizedPoolError(f"unsupported query dtype: {dtype} (fp16 or bf16)")
    slots, kv_heads, dim = key_buffer.shape
    _check_rows("query", query, (None, None, dim), dtype, device)
    queries, q_heads, _ = query.shape
    if dim not in (64, 128, 256):
        raise QuantizedPoolError(f"a head dim of 64, 128 or 256 is needed, got {dim}")
    if q_heads % kv_heads:
        raise QuantizedPoolError("the query heads must be a multiple of the KV heads")
    page = _native.whole_number(page_size)
    if block < 16 or page is None or page < 1 or page % block:
        raise QuantizedPoolError("page_size must be a multiple of scale_block, and scale_block at least 16")
    if page_table.ndim != 2 or page_table.dtype != torch.int32 or page_table.device != device or (
            page_table.shape[1] > 1 and page_table.stride(1) != 1):
        raise QuantizedPoolError("page_table must be int32 [requests, pages] with dense rows on the pool's device")
    requests, pages = page_table.shape
    _check_vector("kv_lengths", kv_lengths, requests, device)
    if query_starts is not None:
        _check_vector("query_starts", query_starts, requests + 1, device)
    elif queries != requests:
        raise QuantizedPoolError("without query_starts every request has one query")
    scale = 1.0 / math.sqrt(dim) if scale is None else float(scale)
    if not 1e-37 <= scale < 1e30:  # a normal number in the kernels' fp32
        raise QuantizedPoolError("scale must be in [1e-37, 1e30)")
    if output is None:
        output = torch.empty((queries, q_heads, dim), dtype=dtype, device=device)
    elif output.shape != query.shape or output.dtype != dtype or output.device != device or (
            not output.is_contiguous() or output.data_ptr() % 16):
        raise QuantizedPoolError("output must be contiguous, 16-byte aligned and of the query's shape, dtype and device")
    elif _meets(output, (query, key_buffer, value_buffer, key_scales, value_scales, page_table, kv_lengths,
                         query_starts)):
        raise QuantizedPoolError("output must not overlap the call's other tensors")
    if device.type != "cuda":
        raise QuantizedPoolError("device tensors are required")
    if not _in_chunks(query):
        query = query.clone(memory_format=torch.contiguous_format)  # the kernels read 16-byte chunks
    args = _native.QuantizedAttentionArgs()
    paged = args.paged
    paged.query = query.data_ptr()
    paged.query_token_stride, paged.query_head_stride = query.stride(0), query.stride(1)
    paged.output = output.data_ptr()
    paged.num_queries = queries
    paged.key_buffer, paged.value_buffer = key_buffer.data_ptr(), value_buffer.data_ptr()
    paged.num_slots = slots
    paged.num_q_heads, paged.num_kv_heads, paged.head_dim = q_heads, kv_heads, dim
    paged.kv_dtype = _HALF_DTYPES[dtype]
    paged.softmax_scale = scale
    paged.page_table = page_table.data_ptr()
    paged.page_table_stride, paged.page_table_columns = page_table.stride(0), pages
    paged.page_size = page
    paged.kv_lengths, paged.kv_lengths_dtype = kv_lengths.data_ptr(), _INDEX_DTYPES[kv_lengths.dtype]
    if query_starts is not None:
        paged.query_starts, paged.query_starts_dtype = query_starts.data_ptr(), _INDEX_DTYPES[query_starts.dtype]
    paged.num_requests = requests
    args.key_scales, args.value_scales = key_scales.data_ptr(), value_scales.data_ptr()
    args.scale_block = block
    with _native.on_device(device):
        needed = _native.quantized_attention_workspace_bytes(args)
        if needed:
            workspace = torch.empty(needed, dtype=torch.uint8, device=device)
            paged.workspace, paged.workspace_bytes = workspace.data_ptr(), needed
        _native.quantized_attention(args, _native.stream_handle(None, device))
    return output
