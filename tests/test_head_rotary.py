"""Refusals of the norm-and-rotate and append operators: argument checks of the
Python entries and of the C entry, none of which reaches a device."""

from __future__ import annotations

import ctypes

import pytest
import torch

from legolink_amd import _native
from legolink_amd.head_rotary import HeadRotaryError, append_rotated_kv_inplace, rotate_heads
from legolink_amd.rope import build_cos_sin_cache


def _heads(tokens=3, q_heads=4, kv_heads=2, dim=32, dtype=torch.bfloat16, rotary=32):
    projected = torch.zeros(tokens, (q_heads + 2 * kv_heads) * dim, dtype=dtype)
    query, key, value = (part.unflatten(-1, (-1, dim)) for part in
                         projected.split([q_heads * dim, kv_heads * dim, kv_heads * dim], dim=-1))
    return dict(query=query, key=key, positions=torch.arange(tokens), rotary_dim=rotary,
                cos_sin_cache=build_cos_sin_cache(16, rotary)), value


def _append(**options):
    arguments, value = _heads(**options)
    kv_heads, dim = value.shape[1:]
    pool = torch.zeros(2, 8, kv_heads, dim, dtype=value.dtype)
    return dict(**arguments, value=value, key_buffer=pool[0], value_buffer=pool[1],
                destination_slots=torch.arange(value.shape[0]))


def test_valid_calls_stop_at_the_device_check():
    arguments, _ = _heads()
    with pytest.raises(HeadRotaryError, match="device tensors are required"):
        rotate_heads(**arguments)
    with pytest.raises(HeadRotaryError, match="device tensors are required"):
        rotate_heads(**arguments, query_output=arguments["query"], key_output=arguments["key"])
    with pytest.raises(HeadRotaryError, match="device tensors are required"):
        append_rotated_kv_inplace(**_append(), query_norm_weight=torch.ones(32), key_norm_weight=torch.ones(32))


@pytest.mark.parametrize("change,message", [
    (dict(query=torch.zeros(3, 4, 32)), "unsupported query dtype"),
    (dict(query=torch.zeros(3, 128, dtype=torch.bfloat16)), "query must be"),
    (dict(query=torch.zeros((), dtype=torch.bfloat16)), "query must be"),
    (dict(query=torch.zeros(3, 32, 8, dtype=torch.bfloat16).transpose(1, 2)), "rows must be dense"),
    (dict(key=torch.zeros(2, 2, 32, dtype=torch.bfloat16)), "key must be"),
    (dict(key=torch.zeros(3, 2, 32, dtype=torch.float16)), "key must be"),
    (dict(key=torch.zeros(3, 2, 16, dtype=torch.bfloat16)), "one head dim"),
    (dict(key=torch.zeros(3, 0, 32, dtype=torch.bfloat16)), "key must be"),
    (dict(rotary_dim=31), "rotary_dim"),
    (dict(rotary_dim=0), "rotary_dim"),
    (dict(rotary_dim=34), "rotary_dim"),
    (dict(positions=torch.arange(4)), "positions"),
    (dict(positions=torch.arange(6)[::2]), "positions"),
    (dict(positions=torch.zeros(3)), "int32 or int64"),
    (dict(cos_sin_cache=torch.zeros(16, 30)), "cos_sin_cache"),
    (dict(cos_sin_cache=torch.zeros(16, 32, dtype=torch.float64)), "cos_sin_cache"),
    (dict(cos_sin_cache=torch.zeros(32, 16).t()), "dense rows"),
    (dict(query_norm_weight=torch.ones(31)), "norm weight"),
    (dict(query_norm_weight=torch.ones(32), key_norm_weight=torch.ones(32, dtype=torch.bfloat16)), "both of one type"),
    (dict(norm_eps=-1.0), "norm_eps"),
    (dict(norm_eps=float("nan")), "norm_eps"),
    (dict(skipped_rows=torch.zeros(1, dtype=torch.int32)), "skipped_rows"),
    (dict(query_output=torch.zeros(3, 4, 16, dtype=torch.bfloat16)), "query_output"),
    (dict(query_output=torch.zeros(1, 4, 32, dtype=torch.bfloat16).expand(3, 4, 32)), "overlap each other"),
    (dict(key_output=torch.zeros(3, 2, 32, dtype=torch.float16)), "key_output"),
])
def test_rotate_heads_refuses(change, message):
    arguments, _ = _heads()
    with pytest.raises(HeadRotaryError, match=message):
        rotate_heads(**{**arguments, **change})


def test_outputs_that_overlap_are_refused():
    arguments, value = _heads()
    query, key = arguments["query"], arguments["key"]
    shifted = torch.zeros(4, 4, 32, dtype=torch.bfloat16)
    with pytest.raises(HeadRotaryError, match="query_output"):  # shifted by one token
        rotate_heads(**{**arguments, "query": shifted[:3]}, query_output=shifted[1:])
    with pytest.raises(HeadRotaryError, match="key_output"):  # the query's place
        rotate_heads(**arguments, key_output=query[:, :2])
    with pytest.raises(HeadRotaryError, match="must not overlap"):
        output = torch.zeros(3, 4, 32, dtype=torch.bfloat16)
        rotate_heads(**arguments, query_output=output, key_output=output[:, :2])
    with pytest.raises(HeadRotaryError, match="query_output"):  # the values' place, which are read
        append = _append()
        append_rotated_kv_inplace(**{**append, "value": append["query"][:, :2]}, query_output=append["query"])
    # Rows between those of the inputs are no overlap.
    with pytest.raises(HeadRotaryError, match="device tensors are required"):
        rotate_heads(**arguments, query_output=query, key_output=value)


@pytest.mark.parametrize("change,message", [
    (dict(value=torch.zeros(3, 3, 32, dtype=torch.bfloat16)), "same heads"),
    (dict(value=torch.zeros(2, 2, 32, dtype=torch.bfloat16)), "value must be"),
    (dict(destination_slots=torch.zeros(3)), "int32 or int64"),
    (dict(destination_slots=torch.arange(2)), "destination_slots"),
    (dict(key_buffer=torch.zeros(8, 2, 16, dtype=torch.bfloat16)), "key_buffer"),
    (dict(key_buffer=torch.zeros(8, 2, 32, dtype=torch.float16)), "key_buffer"),
    (dict(value_buffer=torch.zeros(7, 2, 32, dtype=torch.bfloat16)), "value_buffer"),
    (dict(value_buffer=torch.zeros(2, 8, 32, dtype=torch.bfloat16).transpose(0, 1)), "value_buffer"),
])
def test_append_refuses(change, message):
    with pytest.raises(HeadRotaryError, match=message):
        append_rotated_kv_inplace(**{**_append(), **change})


def test_append_refuses_rows_and_outputs_inside_the_pool():
    append = _append()
    pool = append["key_buffer"]
    with pytest.raises(HeadRotaryError, match="must not overlap"):
        append_rotated_kv_inplace(**{**append, "key": pool[2:5]})
    with pytest.raises(HeadRotaryError, match="must not overlap"):
        append_rotated_kv_inplace(**{**append, "value_buffer": pool})
    with pytest.raises(HeadRotaryError, match="query_output"):
        wide = torch.zeros(8, 4, 32, dtype=torch.bfloat16)
        arguments = {**append, "query": wide[:3].clone(), "key_buffer": wide.view(16, 2, 32)[:8]}
        append_rotated_kv_inplace(**arguments, query_output=wide[:3])


def test_gradients_are_refused():
    arguments, _ = _heads()
    query = arguments["query"].clone().requires_grad_()
    with pytest.raises(HeadRotaryError, match="no gradient"):
        rotate_heads(**{**arguments, "query": query})
    with torch.no_grad(), pytest.raises(HeadRotaryError, match="device tensors are required"):
        rotate_heads(**{**arguments, "query": query})


def _block(**overrides):
    """A block whose pointers are never followed: every case is refused before a launch."""

    args = _native.HeadRotaryArgs()
    args.num_tokens, args.num_q_heads, args.num_kv_heads, args.head_dim = 3, 4, 2, 32
    args.dtype, args.rotary_dim, args.is_neox_style = _native.DTYPE_BFLOAT16, 32, 1
    args.query = args.query_output = args.key = args.key_output = 64
    args.positions = args.cos_sin_cache = 64
    args.positions_dtype, args.cos_sin_dtype = _native.DTYPE_INT64, _native.DTYPE_FLOAT32
    args.cos_sin_rows, args.cos_sin_cols, args.cos_sin_stride_row = 16, 32, 32
    for name, value in overrides.items():
        setattr(args, name, value)
    return args


@pytest.mark.parametrize("overrides,reason", [
    (dict(num_tokens=-1), "invalid_argument"),
    (dict(num_tokens=2 ** 31), "invalid_argument"),
    (dict(num_q_heads=0), "kv_head_layout_mismatch"),
    (dict(num_kv_heads=65536), "kv_head_layout_mismatch"),
    (dict(dtype=_native.DTYPE_FLOAT32), "fp16_or_bf16_required"),
    (dict(head_dim=257), "head_dimension_out_of_range"),
    (dict(rotary_dim=3), "even_rotary_dim_required"),
    (dict(rotary_dim=34), "rotary_dim_exceeds_head_dim"),
    (dict(cos_sin_dtype=_native.DTYPE_INT32), "unsupported_cos_sin_dtype"),
    (dict(cos_sin_cols=30), "unsupported_cos_sin_cache"),
    (dict(positions_dtype=_native.DTYPE_FLOAT32), "integer_token_maps_required"),
    (dict(query=None), "invalid_argument"),
    (dict(positions=None), "invalid_argument"),
    (dict(key_output=None), "invalid_argument"),
    (dict(key_buffer=64), "invalid_argument"),
    (dict(destination_slots=64, key_output=None), "head_dimension_out_of_range"),
    (dict(destination_slots=64, key_output=None, value_head_dim=32), "integer_token_maps_required"),
    (dict(destination_slots=64, value_head_dim=32, destination_slots_dtype=_native.DTYPE_INT32, value=64),
     "invalid_argument"),
    (dict(destination_slots=64, key_output=None, value_head_dim=32, destination_slots_dtype=_native.DTYPE_INT32),
     "invalid_argument"),
    (dict(destination_slots=64, key_output=None, value_head_dim=32, destination_slots_dtype=_native.DTYPE_INT32,
          value=64, num_slots=1), "invalid_argument"),
    (dict(destination_slots=64, key_output=None, value_head_dim=32, destination_slots_dtype=_native.DTYPE_INT32,
          value=64, num_slots=-1), "invalid_argument"),
    (dict(query_norm_weight=64), "invalid_argument"),
    (dict(query_norm_weight=64, norm_weight_dtype=_native.DTYPE_FLOAT32, norm_eps=-1.0), "invalid_argument"),
    (dict(num_tokens=2 ** 31 - 1), "invalid_argument"),  # more rows than a launch holds
])
def test_the_c_entry_refuses_before_any_launch(overrides, reason):
    with pytest.raises(_native.NativeCallError) as error:
        _native.head_rotary(_block(**overrides), 0)
    assert error.value.reason == reason


def test_the_c_entry_checks_its_struct():
    lib = _native.load_library()
    assert lib.ll_head_rotary(None, None) == _native.LL_ERR_INVALID_ARGUMENT
    args = _block()
    args.struct_size = 8
    assert lib.ll_head_rotary(ctypes.byref(args), None) == _native.LL_ERR_INVALID_ARGUMENT
    assert "struct_size" in lib.ll_last_error().decode()


def test_no_tokens_launch_nothing():
    _native.head_rotary(_block(num_tokens=0, query=None, positions=None), 0)
