"""Norms and rotation of a step's queries and keys, and their append to the pool.

A model's step over the pool that the link fills: the new tokens' queries and
keys are normed for each head (where the model has such norms) and turned to
their positions, and the keys and values go to the tokens' slots.  The
reference's models do this with a norm, the rotary module and the pool's write
one after another (patched_sglang_files/python/sglang/srt/models/qwen2.py:
110-177, ``set_kv_buffer``); here each call is one gfx950 kernel launch behind
``ll_head_rotary``:

* ``rotate_heads``: queries and keys to new tensors, or in place -- what a
  batch needs whose keys another path writes (the repair pass's seam);
* ``append_rotated_kv_inplace``: the same with the keys and values written to
  the pool on the way.

Everything is computed in fp32 and rounded once; the calls are enqueued on the
current stream, allocate nothing but the outputs they return, and may be
captured into a HIP graph.  Inference only: tensors that need a gradient or carry
a forward-mode tangent are refused.
"""

from __future__ import annotations

from typing import Optional, Sequence

import torch

from . import _native

_DTYPES = {torch.float16: _native.DTYPE_FLOAT16, torch.bfloat16: _native.DTYPE_BFLOAT16}
_TABLE_DTYPES = {**_DTYPES, torch.float32: _native.DTYPE_FLOAT32}
_INDEX_DTYPES = {torch.int32: _native.DTYPE_INT32, torch.int64: _native.DTYPE_INT64}


# Both calls in one native call where it takes them; the Python checks take the
# others, and name the reason where a call must not run.
_calls = _native.step_calls()


class HeadRotaryError(RuntimeError):
    """A norm-and-rotate or append call that must not run."""


def _span(tensor: torch.Tensor) -> tuple[int, int]:
    """First byte of a tensor's elements and the byte behind its last."""

    begin = tensor.data_ptr()
    reach = sum((size - 1) * stride for size, stride in zip(tensor.shape, tensor.stride()))
    return begin, begin + (reach + 1) * tensor.element_size()


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Do two sets of rows [tokens, heads, dim] share bytes?  Exact for dense
    heads of one token stride (views of one fused projection); other tensors whose
    spans meet count as overlapping."""

    if a.numel() == 0 or b.numel() == 0:
        return False
    (a_begin, a_end), (b_begin, b_end) = _span(a), _span(b)
    if a_end <= b_begin or b_end <= a_begin:
        return False

    def dense(rows: torch.Tensor) -> bool:
        return rows.ndim == 3 and rows.stride(2) == 1 and (rows.shape[1] == 1 or rows.stride(1) == rows.shape[2])

    if not (dense(a) and dense(b)) or a.stride(0) != b.stride(0):
        return True
    stride = a.stride(0) * a.element_size()
    a_width, b_width = (rows.shape[1] * rows.shape[2] * rows.element_size() for rows in (a, b))
    if stride < max(a_width, b_width):
        return True
    offset = (b_begin - a_begin) % stride
    return offset < a_width or stride - offset < b_width


def _same_view(a: torch.Tensor, b: torch.Tensor) -> bool:
    return a.data_ptr() == b.data_ptr() and a.stride() == b.stride() and a.shape == b.shape


def _check_rows(name: str, rows: torch.Tensor, tokens: int, dtype: torch.dtype, device: torch.device) -> None:
    if rows.ndim != 3 or int(rows.shape[0]) != tokens or rows.shape[1] < 1 or rows.shape[2] < 1:
        raise HeadRotaryError(f"{name} must be [tokens, heads, dim] with {tokens} tokens, got {tuple(rows.shape)}")
    if rows.dtype != dtype:
        raise HeadRotaryError(f"{name} must be {dtype} as the query, got {rows.dtype}")
    if rows.device != device:
        raise HeadRotaryError(f"{name} must be on the query's device")
    if rows.shape[2] > 1 and rows.stride(2) != 1:
        raise HeadRotaryError(f"{name}'s rows must be dense")


def _check_output(name: str, output: torch.Tensor, source: torch.Tensor, others: Sequence[torch.Tensor]) -> None:
    """An output is its own source or meets nothing of it, and meets none of the
    call's other tensors, be they the source's own object in another role."""

    if output.shape != source.shape:
        raise HeadRotaryError(f"{name} must have the shape {tuple(source.shape)}, got {tuple(output.shape)}")
    _check_rows(name, output, int(source.shape[0]), source.dtype, source.device)
    tokens, heads, dim = output.shape
    token, head = output.stride(0), output.stride(1)
    by_token = (heads == 1 or head >= dim) and (tokens == 1 or token >= (heads - 1) * head + dim)
    by_head = (tokens == 1 or token >= dim) and (heads == 1 or head >= (tokens - 1) * token + dim)
    if not (by_token or by_head):
        raise HeadRotaryError(f"{name}'s rows must not overlap each other")
    if (not _same_view(output, source) and _overlap(output, source)) or any(_overlap(output, t) for t in others):
        raise HeadRotaryError(f"{name} must be its input itself or not overlap the call's tensors")


def _check_vector(name: str, values: torch.Tensor, count: int, device: torch.device) -> None:
    if values.ndim != 1 or int(values.numel()) != count or values.device != device or not values.is_contiguous():
        raise HeadRotaryError(f"{name} must be a contiguous vector of {count} entries on the query's device")


def _rotary_args(query: torch.Tensor, key: torch.Tensor, positions: torch.Tensor, cos_sin_cache: torch.Tensor,
                 rotary_dim: int, is_neox_style: bool, query_norm_weight: Optional[torch.Tensor],
                 key_norm_weight: Optional[torch.Tensor], norm_eps: float,
                 skipped_rows: Optional[torch.Tensor]) -> _native.HeadRotaryArgs:
    """Checks what both calls have in common and fills their block with it."""

    device, dtype = query.device, query.dtype
    if dtype not in _DTYPES:
        raise HeadRotaryError(f"unsupported query dtype: {dtype} (fp16 or bf16)")
    tokens = int(query.shape[0]) if query.ndim else 0
    _check_rows("query", query, tokens, dtype, device)
    _check_rows("key", key, tokens, dtype, device)
    dim = int(query.shape[2])
    if int(key.shape[2]) != dim:
        raise HeadRotaryError("query and key must have one head dim")
    if dim > 256:
        raise HeadRotaryError("head dims are at most 256")
    rotary_dim = _native.whole_number(rotary_dim)
    if rotary_dim is None or rotary_dim < 2 or rotary_dim % 2 or rotary_dim > dim:
        raise HeadRotaryError("rotary_dim must be even and in [2, head dim]")
    _check_vector("positions", positions, tokens, device)
    if positions.dtype not in _INDEX_DTYPES:
        raise HeadRotaryError("positions must be int32 or int64")
    if cos_sin_cache.ndim != 2 or int(cos_sin_cache.shape[1]) < rotary_dim or cos_sin_cache.device != device:
        raise HeadRotaryError("cos_sin_cache must be [positions, >= rotary_dim] on the query's device")
    if cos_sin_cache.dtype not in _TABLE_DTYPES or cos_sin_cache.stride(1) != 1:
        raise HeadRotaryError("cos_sin_cache must be fp32, fp16 or bf16 with dense rows")
    weights = [weight for weight in (query_norm_weight, key_norm_weight) if weight is not None]
    for weight in weights:
        _check_vector("a norm weight", weight, dim, device)
        if weight.dtype not in _TABLE_DTYPES or weight.dtype != weights[0].dtype:
            raise HeadRotaryError("norm weights must be fp32, fp16 or bf16, both of one type")
    if not float(norm_eps) >= 0.0:
        raise HeadRotaryError("norm_eps must not be negative")
    if skipped_rows is not None and (skipped_rows.dtype != torch.int64 or skipped_rows.numel() != 1
                                     or skipped_rows.device != device):
        raise HeadRotaryError("skipped_rows must be a one-element int64 tensor on the query's device")
    args = _native.HeadRotaryArgs()
    args.num_tokens = tokens
    args.num_q_heads = int(query.shape[1])
    args.num_kv_heads = int(key.shape[1])
    args.head_dim = dim
    args.dtype = _DTYPES[dtype]
    args.query = query.data_ptr()
    args.query_token_stride, args.query_head_stride = query.stride(0), query.stride(1)
    args.key = key.data_ptr()
    args.key_token_stride, args.key_head_stride = key.stride(0), key.stride(1)
    args.positions = positions.data_ptr()
    args.positions_dtype = _INDEX_DTYPES[positions.dtype]
    args.cos_sin_cache = cos_sin_cache.data_ptr()
    args.cos_sin_dtype = _TABLE_DTYPES[cos_sin_cache.dtype]
    args.cos_sin_rows, args.cos_sin_cols = cos_sin_cache.shape
    args.cos_sin_stride_row = cos_sin_cache.stride(0)
    args.rotary_dim = rotary_dim
    args.is_neox_style = 1 if is_neox_style else 0
    args.query_norm_weight = None if query_norm_weight is None else query_norm_weight.data_ptr()
    args.key_norm_weight = None if key_norm_weight is None else key_norm_weight.data_ptr()
    args.norm_weight_dtype = _TABLE_DTYPES[weights[0].dtype] if weights else 0
    args.norm_eps = float(norm_eps)
    args.skipped_rows = None if skipped_rows is None else skipped_rows.data_ptr()
    return args


def _check_counter(skipped_rows: Optional[torch.Tensor], others: Sequence[torch.Tensor]) -> None:
    if skipped_rows is not None and any(_overlap(skipped_rows, tensor) for tensor in others):
        raise HeadRotaryError("skipped_rows must not overlap the call's other tensors")


def _launch(args: _native.HeadRotaryArgs, device: torch.device) -> None:
    if device.type != "cuda":
        raise HeadRotaryError("device tensors are required")
    with _native.on_device(device):
        _native.head_rotary(args, _native.stream_handle(None, device))


def _refuse_gradients(*tensors: Optional[torch.Tensor]) -> None:
    if _native.differentiated(*tensors):
        raise HeadRotaryError("these operators have no gradient: call them under torch.no_grad()")


def rotate_heads(query: torch.Tensor, key: torch.Tensor, *, positions: torch.Tensor, cos_sin_cache: torch.Tensor,
                 rotary_dim: int, is_neox_style: bool = True, query_norm_weight: Optional[torch.Tensor] = None,
                 key_norm_weight: Optional[torch.Tensor] = None, norm_eps: float = 1e-6,
                 query_output: Optional[torch.Tensor] = None, key_output: Optional[torch.Tensor] = None,
                 skipped_rows: Optional[torch.Tensor] = None) -> tuple[torch.Tensor, torch.Tensor]:
    """``query`` [tokens, q heads, dim] and ``key`` [tokens, kv heads, dim] (fp16
    or bf16; any token and head strides, as views of a fused projection have)
    normed for each head by the given weights and turned to ``positions``.

    The table is the link's (``rope.build_cos_sin_cache``).  ``query_output`` and
    ``key_output`` may be the inputs themselves (in place, each its own; what is
    written overlaps none of the call's other tensors); they are new dense
    tensors by default.  A token whose position is outside the table is left
    out: its output rows keep what they held (undefined in a new tensor), and
    ``skipped_rows`` counts it.
    """

    if _calls is not None and query.is_cuda:
        device = torch._C._cuda_getDevice()
        done = _calls.rotate_heads(
            _native.entry_address("ll_head_rotary"), torch._C._cuda_getCurrentRawStream(device), device, query, key,
            positions, cos_sin_cache, rotary_dim, is_neox_style, query_norm_weight, key_norm_weight, norm_eps,
            skipped_rows, query_output, key_output)
        if type(done) is tuple:
            return done
        if done is not None:
            _native.check_status(done)
    _refuse_gradients(query, key, query_norm_weight, key_norm_weight, cos_sin_cache, query_output, key_output)
    args = _rotary_args(query, key, positions, cos_sin_cache, rotary_dim, is_neox_style, query_norm_weight,
                        key_norm_weight, norm_eps, skipped_rows)
    beside = [t for t in (positions, cos_sin_cache, query_norm_weight, key_norm_weight) if t is not None]
    _check_counter(skipped_rows, (query, key, *beside))
    if skipped_rows is not None:
        beside.append(skipped_rows)
    if query_output is None:
        query_output = torch.empty(query.shape, dtype=query.dtype, device=query.device)
    else:
        _check_output("query_output", query_output, query, (key, *beside))
    if key_output is None:
        key_output = torch.empty(key.shape, dtype=key.dtype, device=key.device)
    else:
        _check_output("key_output", key_output, key, (query, *beside))
        if _overlap(key_output, query_output):
            raise HeadRotaryError("query_output and key_output must not overlap")
    args.query_output = query_output.data_ptr()
    args.query_output_token_stride, args.query_output_head_stride = query_output.stride(0), query_output.stride(1)
    args.key_output = key_output.data_ptr()
    args.key_output_token_stride, args.key_output_head_stride = key_output.stride(0), key_output.stride(1)
    _launch(args, query.device)
    return query_output, key_output


def append_rotated_kv_inplace(*, key_buffer: torch.Tensor, value_buffer: torch.Tensor,
                              destination_slots: torch.Tensor, query: torch.Tensor, key: torch.Tensor,
                              value: torch.Tensor, positions: torch.Tensor, cos_sin_cache: torch.Tensor,
                              rotary_dim: int, is_neox_style: bool = True,
                              query_norm_weight: Optional[torch.Tensor] = None,
                              key_norm_weight: Optional[torch.Tensor] = None, norm_eps: float = 1e-6,
                              query_output: Optional[torch.Tensor] = None,
                              skipped_rows: Optional[torch.Tensor] = None) -> torch.Tensor:
    """A step's new tokens into one layer of the pool: ``rotate_heads`` with the
    keys written to row ``destination_slots[t]`` of ``key_buffer`` [slots, kv
    heads, dim] and ``value`` [tokens, kv heads, value dim] to that row of
    ``value_buffer``; returns the queries.

    A pool of pages is the same pool: slot = page * page_size + offset.  A
    negative slot is padding (its queries are turned, nothing is written), a
    slot past the pool likewise and counted in ``skipped_rows``; a token whose
    position is outside the table is left out whole and counted.  The slots that
    are written must be pairwise distinct.
    """

    if _calls is not None and query.is_cuda:
        device = torch._C._cuda_getDevice()
        done = _calls.append(
            _native.entry_address("ll_head_rotary"), torch._C._cuda_getCurrentRawStream(device), device, query, key,
            positions, cos_sin_cache, rotary_dim, is_neox_style, query_norm_weight, key_norm_weight, norm_eps,
            skipped_rows, query_output, value, key_buffer, value_buffer, destination_slots)
        if type(done) is int:
            _native.check_status(done)
        elif done is not None:
            return done
    _refuse_gradients(query, key, value, query_norm_weight, key_norm_weight, cos_sin_cache, query_output,
                      key_buffer, value_buffer)
    args = _rotary_args(query, key, positions, cos_sin_cache, rotary_dim, is_neox_style, query_norm_weight,
                        key_norm_weight, norm_eps, skipped_rows)
    _check_rows("value", value, args.num_tokens, query.dtype, query.device)
    _check_vector("destination_slots", destination_slots, args.num_tokens, query.device)
    if destination_slots.dtype not in _INDEX_DTYPES:
        raise HeadRotaryError("destination_slots must be int32 or int64")
    if value.shape[1] != key.shape[1]:
        raise HeadRotaryError("key and value must have the same heads")
    if int(value.shape[2]) > 256:
        raise HeadRotaryError("head dims are at most 256")
    beside = [t for t in (positions, cos_sin_cache, query_norm_weight, key_norm_weight, destination_slots)
              if t is not None]
    _check_counter(skipped_rows, (query, key, value, *beside))
    if skipped_rows is not None:
        beside.append(skipped_rows)
    for name, buffer, rows in (("key_buffer", key_buffer, key), ("value_buffer", value_buffer, value)):
        if buffer.ndim != 3 or buffer.shape[1:] != rows.shape[1:] or buffer.shape[0] != key_buffer.shape[0]:
            raise HeadRotaryError(f"{name} must be [slots, kv heads, dim] as the rows, got {tuple(buffer.shape)}")
        if buffer.dtype != query.dtype or buffer.device != query.device or not buffer.is_contiguous():
            raise HeadRotaryError(f"{name} must be a contiguous {query.dtype} tensor on the query's device")
        if any(_overlap(buffer, other) for other in (query, key, value, *beside)):
            raise HeadRotaryError(f"{name} must not overlap the call's other tensors")
    if _overlap(key_buffer, value_buffer):
        raise HeadRotaryError("key_buffer and value_buffer must not overlap")
    if query_output is None:
        query_output = torch.empty(query.shape, dtype=query.dtype, device=query.device)
    else:
        _check_output("query_output", query_output, query, (key, value, key_buffer, value_buffer, *beside))
    args.query_output = query_output.data_ptr()
    args.query_output_token_stride, args.query_output_head_stride = query_output.stride(0), query_output.stride(1)
    args.value = value.data_ptr()
    args.value_token_stride, args.value_head_stride = value.stride(0), value.stride(1)
    args.value_head_dim = int(value.shape[2])
    args.key_buffer = key_buffer.data_ptr()
    args.value_buffer = value_buffer.data_ptr()
    args.num_slots = int(key_buffer.shape[0])
    args.destination_slots = destination_slots.data_ptr()
    args.destination_slots_dtype = _INDEX_DTYPES[destination_slots.dtype]
    _launch(args, query.device)
    return query_output
