"""The 8-bit pool on the CPU: the format's model against torch's types, refusals of
the Python entries and of the C entries, none of which reaches a device."""

from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest
import torch

from legolink_amd import _native, quantized_pool as qp
from tests import quantized_pool_math as qm


def test_the_model_of_the_format_is_torchs():
    codes = torch.arange(256, dtype=torch.uint8)
    values = codes.view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(values, qm.VALUES, equal_nan=True)
    assert np.array_equal(np.signbit(values[128:255]), np.ones(127, bool))
    rng = np.random.default_rng(1)
    some = np.concatenate((rng.normal(size=4000) * 60, qm._MIDDLES, -qm._MIDDLES, qm._SIZES,
                           rng.normal(size=2000) * 2.0 ** -8, [0.0, -0.0, np.inf, -np.inf, np.nan])).clip(-448, 448)
    some = np.float32(some).astype(np.float64)
    want = torch.from_numpy(some).float().to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert qm.same_codes(qm.encoded(some), want)
    scales = torch.arange(256, dtype=torch.uint8).view(torch.float8_e8m0fnu).double().numpy()
    assert np.array_equal(qm.values_of(np.full((256, 1, 1), 0x38, np.uint8), np.arange(256)[:, None], 1)[:, 0, 0],
                          scales, equal_nan=True)
    assert [qm.least_byte(x) for x in (0.0, 448.0, 448.5, 896.0, 2.0 ** -130)] == [0, 127, 128, 128, 0]


def test_the_package_names_the_module():
    import legolink_amd

    assert "quantized_pool" in legolink_amd.__all__ and "legolink_amd.quantized_pool" in legolink_amd.__doc__


def _pool(slots=64, heads=2, dim=64, block=16):
    return dict(key_buffer=torch.zeros(slots, heads, dim, dtype=torch.float8_e4m3fn),
                value_buffer=torch.zeros(slots, heads, dim, dtype=torch.float8_e4m3fn),
                key_scales=torch.zeros(slots // block, heads, dtype=torch.uint8).view(torch.float8_e8m0fnu),
                value_scales=torch.zeros(slots // block, heads, dtype=torch.uint8).view(torch.float8_e8m0fnu),
                scale_block=block)


def _append(tokens=3, dtype=torch.bfloat16):
    return dict(**_pool(), query=torch.zeros(tokens, 4, 64, dtype=dtype), key=torch.zeros(tokens, 2, 64, dtype=dtype),
                value=torch.zeros(tokens, 2, 64, dtype=dtype), destination_slots=torch.arange(tokens),
                positions=torch.arange(tokens), cos_sin_cache=torch.zeros(8, 64), rotary_dim=64)


def _link(tokens=3):
    return dict(**_pool(), source_slots=torch.arange(tokens), destination_slots=torch.arange(tokens) + 32,
                local_positions=torch.arange(tokens), global_positions=torch.arange(tokens),
                cos_sin_cache=torch.zeros(8, 64), rotary_dim=64)


def _load():
    return dict(**_pool(), slots=torch.arange(5))


def _attention(requests=2):
    return dict(**_pool(), query=torch.zeros(requests, 4, 64, dtype=torch.bfloat16),
                page_table=torch.zeros(requests, 4, dtype=torch.int32),
                kv_lengths=torch.ones(requests, dtype=torch.int64), page_size=16)


CALLS = {"append": (qp.append_quantized_kv_inplace, _append), "link": (qp.link_quantized_kv_inplace, _link),
         "load": (qp.load_quantized_kv, _load), "attention": (qp.quantized_paged_attention, _attention)}


@pytest.mark.parametrize("name", CALLS)
def test_valid_calls_stop_at_the_device_check(name):
    call, arguments = CALLS[name]
    with pytest.raises(qp.QuantizedPoolError, match="device tensors are required"):
        call(**arguments())


POOL_REFUSALS = [
    (dict(scale_block=0), "scale_block"), (dict(scale_block=24), "scale_block"), (dict(scale_block=256), "scale_block"),
    (dict(scale_block=16.5), "scale_block"), (dict(scale_block=8), "key_scales must be"),
    (dict(key_buffer=torch.zeros(64, 2, 64, dtype=torch.bfloat16)), "shape|key_buffer must be"),
    (dict(value_buffer=torch.zeros(64, 2, 64, dtype=torch.float8_e5m2)), "value_buffer must be"),
    (dict(value_buffer=torch.zeros(48, 2, 64, dtype=torch.float8_e4m3fn)), "one shape"),
    (dict(key_buffer=torch.zeros(56, 2, 64, dtype=torch.float8_e4m3fn),
          value_buffer=torch.zeros(56, 2, 64, dtype=torch.float8_e4m3fn)), "whole blocks"),
    (dict(key_buffer=torch.zeros(64, 2, 72, dtype=torch.float8_e4m3fn),
          value_buffer=torch.zeros(64, 2, 72, dtype=torch.float8_e4m3fn)), "head dims"),
    (dict(key_buffer=torch.zeros(2, 64, 64, dtype=torch.float8_e4m3fn).transpose(0, 1)), "contiguous"),
    (dict(key_buffer=torch.zeros(64 * 2 * 64 + 1, dtype=torch.float8_e4m3fn)[1:].view(64, 2, 64)), "aligned"),
    (dict(key_scales=torch.zeros(4, 2)), "key_scales must be"),
    (dict(value_scales=torch.zeros(5, 2, dtype=torch.uint8).view(torch.float8_e8m0fnu)), "value_scales must be"),
    (dict(value_scales=torch.zeros(2, 4, dtype=torch.uint8).view(torch.float8_e8m0fnu).t()), "contiguous"),
]


@pytest.mark.parametrize("name", CALLS)
@pytest.mark.parametrize("change,message", POOL_REFUSALS)
def test_every_call_refuses_a_bad_pool(name, change, message):
    call, arguments = CALLS[name]
    with pytest.raises(qp.QuantizedPoolError, match=message):
        call(**{**arguments(), **change})


APPEND_REFUSALS = [
    (dict(query=torch.zeros(3, 4, 64)), "unsupported query dtype"),
    (dict(query=torch.zeros(3, 4, 128, dtype=torch.bfloat16)), "query must be"),
    (dict(query=torch.zeros(3, 0, 64, dtype=torch.bfloat16)), "query must be"),
    (dict(query=torch.zeros(3, 256, dtype=torch.bfloat16)), "query must be"),
    (dict(key=torch.zeros(3, 4, 64, dtype=torch.bfloat16)), "key must be"),
    (dict(key=torch.zeros(3, 2, 64, dtype=torch.float16)), "key must be"),
    (dict(value=torch.zeros(2, 2, 64, dtype=torch.bfloat16)), "value must be"),
    (dict(positions=torch.arange(2)), "positions"), (dict(positions=torch.zeros(3)), "positions"),
    (dict(destination_slots=torch.arange(6)[::2]), "destination_slots"),
    (dict(rotary_dim=24), "rotary_dim"), (dict(rotary_dim=0), "rotary_dim"), (dict(rotary_dim=128), "rotary_dim"),
    (dict(rotary_dim=32.5), "rotary_dim"),
    (dict(cos_sin_cache=torch.zeros(8, 32)), "cos_sin_cache"),
    (dict(cos_sin_cache=torch.zeros(8, 64, dtype=torch.float64)), "cos_sin_cache"),
    (dict(cos_sin_cache=torch.zeros(64, 8).t()), "cos_sin_cache"),
    (dict(query_norm_weight=torch.zeros(32)), "norm weight"),
    (dict(query_norm_weight=torch.zeros(64), key_norm_weight=torch.zeros(64, dtype=torch.bfloat16)), "one type"),
    (dict(norm_eps=-1.0), "norm_eps"), (dict(norm_eps=float("nan")), "norm_eps"),
    (dict(skipped_rows=torch.zeros(1)), "skipped_rows"), (dict(skipped_rows=torch.zeros(2, dtype=torch.int64)), "skipped"),
    (dict(query_output=torch.zeros(3, 4, 64)), "query_output"),
    (dict(query_output=torch.zeros(1, 4, 64, dtype=torch.bfloat16).expand(3, 4, 64)), "must not overlap"),
    (dict(query_output=torch.zeros(3, 64, 4, dtype=torch.bfloat16).transpose(1, 2)), "query_output's rows must be dense"),
]


@pytest.mark.parametrize("change,message", APPEND_REFUSALS)
def test_append_refuses(change, message):
    with pytest.raises(qp.QuantizedPoolError, match=message):
        qp.append_quantized_kv_inplace(**{**_append(), **change})


LINK_REFUSALS = [
    (dict(source_slots=torch.arange(2)), "destination_slots"),
    (dict(source_slots=torch.arange(3, dtype=torch.int32)), "one type"),
    (dict(global_positions=torch.arange(3, dtype=torch.int32)), "one type"),
    (dict(local_positions=torch.zeros(3)), "local_positions"),
    (dict(repair_mask=torch.zeros(2, dtype=torch.bool)), "repair_mask"),
    (dict(repair_mask=torch.zeros(3, dtype=torch.int64)), "repair_mask"),
    (dict(prefix_token_count=4), "prefix"), (dict(prefix_token_count=-1), "prefix"),
    (dict(rotary_dim=40), "rotary_dim"), (dict(skipped_rows=torch.zeros(1)), "skipped_rows"),
]


@pytest.mark.parametrize("change,message", LINK_REFUSALS)
def test_link_refuses(change, message):
    with pytest.raises(qp.QuantizedPoolError, match=message):
        qp.link_quantized_kv_inplace(**{**_link(), **change})


LOAD_REFUSALS = [
    (dict(dtype=torch.float64), "unsupported dtype"), (dict(slots=torch.zeros(5)), "slots"),
    (dict(slots=torch.zeros(5, 1, dtype=torch.int64)), "slots"),
    (dict(key_output=torch.zeros(5, 2, 64)), "key_output"),
    (dict(value_output=torch.zeros(4, 2, 64, dtype=torch.bfloat16)), "value_output"),
    (dict(key_output=torch.zeros(5, 64, 2, dtype=torch.bfloat16).transpose(1, 2)), "key_output"),
]


@pytest.mark.parametrize("change,message", LOAD_REFUSALS)
def test_load_refuses(change, message):
    with pytest.raises(qp.QuantizedPoolError, match=message):
        qp.load_quantized_kv(**{**_load(), **change})


ATTENTION_REFUSALS = [
    (dict(query=torch.zeros(2, 4, 64)), "unsupported query dtype"),
    (dict(query=torch.zeros(2, 4, 128, dtype=torch.bfloat16)), "query must be"),
    (dict(query=torch.zeros(2, 5, 64, dtype=torch.bfloat16)), "multiple of the KV heads"),
    (dict(page_size=8), "page_size"), (dict(page_size=24), "page_size"), (dict(page_size=0), "page_size"),
    (dict(page_table=torch.zeros(2, 4, dtype=torch.int64)), "page_table"),
    (dict(page_table=torch.zeros(4, 2, dtype=torch.int32).t()), "page_table"),
    (dict(kv_lengths=torch.ones(3, dtype=torch.int32)), "kv_lengths"), (dict(kv_lengths=torch.ones(2)), "kv_lengths"),
    (dict(query_starts=torch.zeros(2, dtype=torch.int32)), "query_starts"),
    (dict(query=torch.zeros(3, 4, 64, dtype=torch.bfloat16)), "one query"),
    (dict(scale=0.0), "scale"), (dict(scale=float("nan")), "scale"), (dict(scale=1e30), "scale"),
    (dict(output=torch.zeros(2, 4, 64)), "output"),
    (dict(output=torch.zeros(2, 64, 4, dtype=torch.bfloat16).transpose(1, 2)), "output"),
]


@pytest.mark.parametrize("change,message", ATTENTION_REFUSALS)
def test_attention_refuses(change, message):
    with pytest.raises(qp.QuantizedPoolError, match=message):
        qp.quantized_paged_attention(**{**_attention(), **change})


def test_blocks_below_16_and_other_dims_are_not_attended():
    pool = _pool(block=8)
    with pytest.raises(qp.QuantizedPoolError, match="at least 16"):
        qp.quantized_paged_attention(**{**_attention(), **pool})
    pool = _pool(dim=80)
    with pytest.raises(qp.QuantizedPoolError, match="64, 128 or 256"):
        qp.quantized_paged_attention(**{**_attention(), **pool, "query": torch.zeros(2, 4, 80, dtype=torch.bfloat16)})


def test_what_is_written_overlaps_nothing_else():
    call = _append()
    with pytest.raises(qp.QuantizedPoolError, match="overlap"):
        qp.append_quantized_kv_inplace(**{**call, "value_buffer": call["key_buffer"]})
    with pytest.raises(qp.QuantizedPoolError, match="overlap"):
        qp.append_quantized_kv_inplace(**{**call, "value_scales": call["key_scales"]})
    with pytest.raises(qp.QuantizedPoolError, match="overlap"):
        qp.append_quantized_kv_inplace(**{**call, "value": call["key_buffer"].view(torch.bfloat16).view(-1)[:384]
                                          .view(3, 2, 64)})
    with pytest.raises(qp.QuantizedPoolError, match="overlap"):
        qp.append_quantized_kv_inplace(**call, skipped_rows=call["positions"][:1])
    shared = torch.zeros(3, 8, 64, dtype=torch.bfloat16)
    with pytest.raises(qp.QuantizedPoolError, match="query_output"):
        qp.append_quantized_kv_inplace(**{**call, "query": shared[:, :4], "query_output": shared[:, 2:6]})
    with pytest.raises(qp.QuantizedPoolError, match="device tensors"):  # in place
        qp.append_quantized_kv_inplace(**{**call, "query": shared[:, :4], "key": shared[:, 4:6], "value": shared[:, 6:],
                                          "query_output": shared[:, :4]})
    link = _link()
    with pytest.raises(qp.QuantizedPoolError, match="overlap"):
        qp.link_quantized_kv_inplace(**{**link, "cos_sin_cache": link["key_buffer"].view(torch.float32).view(-1, 64)})
    load = _load()
    with pytest.raises(qp.QuantizedPoolError, match="overlap"):
        qp.load_quantized_kv(**load, key_output=load["key_buffer"].view(torch.bfloat16).view(-1)[:640].view(5, 2, 64))
    same = torch.zeros(5, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(qp.QuantizedPoolError, match="overlap"):
        qp.load_quantized_kv(**load, key_output=same, value_output=same)
    attention = _attention()
    with pytest.raises(qp.QuantizedPoolError, match="overlap"):
        qp.quantized_paged_attention(**attention, output=attention["query"])


@pytest.mark.parametrize("name,changed", [("append", "query"), ("append", "key"), ("append", "cos_sin_cache"),
                                          ("link", "cos_sin_cache"), ("attention", "query")])
def test_gradients_and_tangents_are_refused(name, changed):
    call, arguments = CALLS[name]
    arguments = arguments()
    with pytest.raises(qp.QuantizedPoolError, match="no gradient"):
        call(**{**arguments, changed: arguments[changed].clone().requires_grad_()})
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(arguments[changed], torch.ones_like(arguments[changed]))
        with pytest.raises(qp.QuantizedPoolError, match="no gradient"), torch.no_grad():
            call(**{**arguments, changed: dual})


# -- the C entries: pointers that are never followed ------------------------


def _fill_pool(pool):
    pool.key_buffer = pool.value_buffer = pool.key_scales = pool.value_scales = 64
    pool.num_slots, pool.scale_block, pool.num_kv_heads, pool.head_dim = 64, 16, 2, 64


def _append_block():
    args = _native.QuantizedAppendArgs()
    _fill_pool(args.pool)
    args.num_tokens, args.num_q_heads, args.dtype = 3, 4, _native.DTYPE_BFLOAT16
    for name in ("query", "query_output", "key", "value"):
        setattr(args, name, 64)
        setattr(args, f"{name}_token_stride", 256)
        setattr(args, f"{name}_head_stride", 64)
    args.destination_slots = args.positions = args.cos_sin_cache = 64
    args.destination_slots_dtype = args.positions_dtype = _native.DTYPE_INT64
    args.cos_sin_dtype, args.cos_sin_rows, args.cos_sin_cols, args.cos_sin_stride_row = _native.DTYPE_FLOAT32, 8, 64, 64
    args.rotary_dim = 64
    return args


def _link_block():
    args = _native.QuantizedLinkArgs()
    _fill_pool(args.pool)
    args.num_tokens = 3
    args.source_slots = args.destination_slots = args.local_positions = args.global_positions = args.cos_sin_cache = 64
    args.slots_dtype = args.positions_dtype = _native.DTYPE_INT32
    args.cos_sin_dtype, args.cos_sin_rows, args.cos_sin_cols, args.cos_sin_stride_row = _native.DTYPE_FLOAT32, 8, 64, 64
    args.rotary_dim = 64
    return args


def _load_block():
    args = _native.QuantizedLoadArgs()
    _fill_pool(args.pool)
    args.num_rows, args.dtype, args.key_output, args.value_output = 3, _native.DTYPE_FLOAT32, 64, 64
    args.slots, args.slots_dtype = 64, _native.DTYPE_INT64
    return args


def _attention_block():
    args = _native.QuantizedAttentionArgs()
    paged = args.paged
    paged.query = paged.output = paged.key_buffer = paged.value_buffer = paged.page_table = paged.kv_lengths = 64
    paged.query_token_stride, paged.query_head_stride = 256, 64
    paged.num_queries = paged.num_requests = 2
    paged.num_slots, paged.num_q_heads, paged.num_kv_heads, paged.head_dim = 64, 4, 2, 64
    paged.kv_dtype, paged.softmax_scale = _native.DTYPE_BFLOAT16, 0.125
    paged.page_table_stride = paged.page_table_columns = 40
    paged.page_size, paged.kv_lengths_dtype = 16, _native.DTYPE_INT32
    args.key_scales = args.value_scales = 64
    args.scale_block = 16
    return args


BLOCKS = {"append": (_native.quantized_append, _append_block), "link": (_native.quantized_link, _link_block),
          "load": (_native.quantized_load, _load_block),
          "attention": (_native.quantized_attention, _attention_block)}
BAD_POOL = [
    ("pool.scale_block", 0, "invalid_argument"), ("pool.scale_block", 48, "invalid_argument"),
    ("pool.scale_block", 256, "invalid_argument"), ("pool.num_slots", 40, "invalid_argument"),
    ("pool.num_slots", -16, "invalid_argument"), ("pool.num_slots", 2 ** 31, "invalid_argument"),
    ("pool.num_kv_heads", 0, "kv_head_layout_mismatch"), ("pool.num_kv_heads", 65536, "kv_head_layout_mismatch"),
    ("pool.head_dim", 8, "head_dimension_out_of_range"), ("pool.head_dim", 72, "head_dimension_out_of_range"),
    ("pool.head_dim", 272, "head_dimension_out_of_range"), ("pool.key_buffer", None, "invalid_argument"),
    ("pool.value_scales", None, "invalid_argument"), ("pool.value_buffer", 72, "invalid_argument"),
]
BAD_TABLE = [
    ("rotary_dim", 24, "invalid_argument"), ("rotary_dim", 15, "even_rotary_dim_required"),
    ("rotary_dim", 80, "rotary_dim_exceeds_head_dim"), ("cos_sin_dtype", _native.DTYPE_INT32, "unsupported_cos_sin_dtype"),
    ("cos_sin_cols", 32, "unsupported_cos_sin_cache"), ("cos_sin_rows", -1, "unsupported_cos_sin_cache"),
    ("cos_sin_cache", None, "invalid_argument"),
]
BAD = {
    "append": [*BAD_POOL, *BAD_TABLE, ("num_tokens", -1, "invalid_argument"), ("num_tokens", 2 ** 31, "invalid_argument"),
               ("num_q_heads", 0, "kv_head_layout_mismatch"), ("dtype", _native.DTYPE_FLOAT32, "fp16_or_bf16_required"),
               ("positions_dtype", _native.DTYPE_FLOAT32, "integer_token_maps_required"),
               ("destination_slots_dtype", 0, "integer_token_maps_required"), ("query", None, "invalid_argument"),
               ("value", 72, "invalid_argument"), ("key_token_stride", 12, "invalid_argument"),
               ("query_norm_weight", 64, "invalid_argument"), ("num_tokens", 2 ** 31 - 1, "invalid_argument")],
    "link": [*BAD_POOL, *BAD_TABLE, ("num_tokens", -1, "invalid_argument"), ("prefix_token_count", 4, "invalid_argument"),
             ("slots_dtype", 0, "integer_token_maps_required"), ("positions_dtype", 0, "integer_token_maps_required"),
             ("source_slots", None, "invalid_argument"), ("num_tokens", 2 ** 31 - 1, "invalid_argument")],
    "load": [*BAD_POOL, ("num_rows", -1, "invalid_argument"), ("dtype", _native.DTYPE_INT32, "invalid_argument"),
             ("slots_dtype", 0, "integer_token_maps_required"), ("key_output", None, "invalid_argument"),
             ("value_output", 72, "invalid_argument"), ("num_rows", 2 ** 31 - 1, "invalid_argument")],
    "attention": [("scale_block", 8, "invalid_argument"), ("scale_block", 256, "invalid_argument"),
                  ("scale_block", 48, "invalid_argument"), ("scale_block", 32, "invalid_argument"),
                  ("paged.num_slots", 72, "invalid_argument"), ("key_scales", None, "invalid_argument"),
                  ("paged.head_dim", 96, "head_dimension_out_of_range"), ("paged.num_q_heads", 5, "kv_head_layout_mismatch"),
                  ("paged.softmax_scale", 0.0, "invalid_argument"), ("paged.workspace", None, "invalid_argument"),
                  ("paged.query", 72, "invalid_argument")],
}


@pytest.mark.parametrize("name,field,value,reason", [(name, *bad) for name, bads in BAD.items() for bad in bads])
def test_the_c_entries_refuse_before_any_launch(name, field, value, reason):
    call, block = BLOCKS[name]
    args = block()
    owner, _, leaf = field.rpartition(".")
    setattr(getattr(args, owner) if owner else args, leaf, value)
    if field == "scale_block" and value == 32:
        args.paged.num_slots = 64
    with pytest.raises(_native.NativeCallError) as error:
        call(args, 0)
    assert error.value.reason == reason


@pytest.mark.parametrize("name", BLOCKS)
def test_the_c_entries_check_their_struct(name):
    lib = _native.load_library()
    entry = getattr(lib, f"ll_quantized_{name}")
    assert entry(None, None) == _native.LL_ERR_INVALID_ARGUMENT
    args = BLOCKS[name][1]()
    args.struct_size = 8
    assert entry(ctypes.byref(args), None) == _native.LL_ERR_INVALID_ARGUMENT
    assert "struct_size" in lib.ll_last_error().decode()


def test_nothing_to_do_launches_nothing():
    for name, field in (("append", "num_tokens"), ("link", "num_tokens"), ("load", "num_rows")):
        args = BLOCKS[name][1]()
        setattr(args, field, 0)
        BLOCKS[name][0](args, 0)
    args = _attention_block()
    args.paged.num_queries = args.paged.num_requests = 0
    assert _native.quantized_attention_workspace_bytes(args) == 0
    _native.quantized_attention(args, 0)


def test_the_workspace_is_that_of_paged_attention():
    args = _attention_block()
    assert _native.quantized_attention_workspace_bytes(args) == _native.paged_attention_workspace_bytes(args.paged) > 0


@pytest.mark.parametrize("dtype,exact", [(torch.bfloat16, range(3, 247)), (torch.float32, range(247)),
                                         (torch.float16, range(127 - 15, 127 + 8))])
def test_the_scales_whose_values_a_type_holds(dtype, exact):
    """Every code under every scale byte: which bytes make values that the type holds."""

    codes = torch.arange(256, dtype=torch.uint8)[:, None].expand(256, 255).contiguous().numpy()
    scales = np.arange(255)
    values = torch.from_numpy(qm.VALUES[codes] * np.ldexp(1.0, scales - 127))
    held = values.to(dtype)
    same = ((held.double() == values) | values.isnan()).all(0).tolist()
    assert [byte for byte in range(255) if same[byte]] == list(exact)
    # What is past the type is infinite; elsewhere a value is off by no more than half its least step.
    past = held.isinf()
    assert bool((values[past].abs() >= torch.finfo(dtype).max).all())
    step = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    assert bool(((held.double() - values).abs()[~past & ~values.isnan()] <= step / 2).all())
    if dtype == torch.float16:  # exact from 2^-21 on, up to the largest
        size = values.abs()
        assert bool((held.double() == values)[(size >= 2.0 ** -21) & (size <= 65504)].all())


def test_the_largest_rows_are_held_as_two_to_the_128():
    """1.9375 * 2^127 lies between the codes 240 and 256 of byte 247, and goes to the even one."""

    byte = qm.least_byte(1.9375 * 2.0 ** 127)
    assert byte == 247
    below, at = np.float64([1.9375 * 2.0 ** 127 * (1 - 2.0 ** -50), 1.9375 * 2.0 ** 127]) * 2.0 ** -120
    assert qm.VALUES[qm.encoded(np.array([below]))][0] == 240 and qm.VALUES[qm.encoded(np.array([at]))][0] == 256


def _attention_workspace(requests, kv_heads, dim, keys):
    args = _attention_block()
    paged = args.paged
    paged.num_queries = paged.num_requests = requests
    paged.num_q_heads = paged.num_kv_heads = kv_heads
    paged.head_dim = dim
    paged.page_table_stride = paged.page_table_columns = -(-keys // 16)
    return _native.quantized_attention_workspace_bytes(args)


@pytest.mark.parametrize("kv_heads,dim,places", [(8, 128, 64), (10, 128, 51), (12, 128, 42), (8, 256, 32), (16, 64, 64),
                                                 (7, 128, 36)])
def test_the_rounds_of_single_tokens_have_no_point_of_their_own(kv_heads, dim, places):
    """Partial results: 2 (places - requests) + 4 for one round of units, 4 places + 2 for
    two; tables of 1,000 (places / requests)^2 keys of 128 leave room for two."""

    partial = kv_heads * 16 * (dim + 2) * 4
    for requests in range(-(-32 // kv_heads), places // 2 + 1):  # (heads that share a workgroup)
        one, two = (2 * (places - requests) + 4) * partial, (4 * places + 2) * partial
        pages = 1000 * (places / requests) ** 2 * 128 / dim / 16
        for keys in (1024 * 128 // dim, 16 * math.floor(pages - 1e-9)):
            assert _attention_workspace(requests, kv_heads, dim, keys) == one, (requests, keys)
        for keys in (16 * math.ceil(pages + 1e-9), 131072):
            want = two if 4 * requests > places else one
            assert _attention_workspace(requests, kv_heads, dim, keys) == want, (requests, keys)
    assert _attention_workspace(places // 2 + 1, kv_heads, dim, 1024) == (4 * places + 2) * partial
