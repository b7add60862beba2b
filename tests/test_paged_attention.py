"""Refusals of paged attention: checks of the Python entry and of the C entry,
none of which reaches a device, and the workspace that shapes ask for."""

from __future__ import annotations

import ctypes

import pytest
import torch

from legolink_amd import _native
from legolink_amd.paged_attention import PagedAttentionError, paged_attention


def _arguments(requests=2, q_heads=4, kv_heads=2, dim=64, dtype=torch.bfloat16):
    return dict(query=torch.zeros(requests, q_heads, dim, dtype=dtype),
                key_buffer=torch.zeros(32, kv_heads, dim, dtype=dtype),
                value_buffer=torch.zeros(32, kv_heads, dim, dtype=dtype),
                page_table=torch.zeros(requests, 4, dtype=torch.int32),
                kv_lengths=torch.ones(requests, dtype=torch.int64), page_size=8)


def test_valid_calls_stop_at_the_device_check():
    with pytest.raises(PagedAttentionError, match="device tensors are required"):
        paged_attention(**_arguments())
    with pytest.raises(PagedAttentionError, match="device tensors are required"):
        paged_attention(**{**_arguments(), "query": torch.zeros(5, 4, 64, dtype=torch.bfloat16)},
                        query_starts=torch.tensor([0, 2, 5]), output=torch.zeros(5, 4, 64, dtype=torch.bfloat16))


@pytest.mark.parametrize("change,message", [
    (dict(query=torch.zeros(2, 4, 64)), "unsupported query dtype"),
    (dict(query=torch.zeros(2, 4, 64, dtype=torch.float16)), "one dtype"),
    (dict(query=torch.zeros(2, 256, dtype=torch.bfloat16)), "query must be"),
    (dict(value_buffer=torch.zeros(31, 2, 64, dtype=torch.bfloat16)), "query must be"),
    (dict(query=torch.zeros(2, 4, 128, dtype=torch.bfloat16)), "head dim"),
    (dict(query=torch.zeros(2, 5, 64, dtype=torch.bfloat16)), "multiple of the KV heads"),
    (dict(query=torch.zeros(2, 0, 64, dtype=torch.bfloat16)), "multiple of the KV heads"),
    (dict(key_buffer=torch.zeros(32, 64, 2, dtype=torch.bfloat16).transpose(1, 2)), "key_buffer"),
    (dict(key_buffer=torch.zeros(32 * 2 * 64 + 1, dtype=torch.bfloat16)[1:].view(32, 2, 64)), "key_buffer"),
    (dict(page_table=torch.zeros(2, 4, dtype=torch.int64)), "page_table"),
    (dict(page_table=torch.zeros(4, 2, dtype=torch.int32).t()), "page_table"),
    (dict(page_table=torch.zeros(8, dtype=torch.int32)), "page_table"),
    (dict(page_size=0), "page_size"),
    (dict(kv_lengths=torch.ones(3, dtype=torch.int32)), "kv_lengths"),
    (dict(kv_lengths=torch.ones(2)), "int32 or int64"),
    (dict(kv_lengths=torch.ones(4, dtype=torch.int32)[::2]), "kv_lengths"),
    (dict(query_starts=torch.zeros(2, dtype=torch.int32)), "query_starts"),
    (dict(query=torch.zeros(3, 4, 64, dtype=torch.bfloat16)), "one query"),
    (dict(scale=0.0), "scale"),
    (dict(scale=-1.0), "scale"),
    (dict(scale=float("nan")), "scale"),
    (dict(scale=float("inf")), "scale"),
    (dict(output=torch.zeros(2, 4, 64)), "output"),
    (dict(output=torch.zeros(2, 64, 4, dtype=torch.bfloat16).transpose(1, 2)), "output"),
    (dict(output=torch.zeros(2 * 4 * 64 + 1, dtype=torch.bfloat16)[1:].view(2, 4, 64)), "output"),
])
def test_paged_attention_refuses(change, message):
    with pytest.raises(PagedAttentionError, match=message):
        paged_attention(**{**_arguments(), **change})


def test_an_output_over_the_inputs_is_refused():
    arguments = _arguments()
    with pytest.raises(PagedAttentionError, match="must not overlap"):
        paged_attention(**arguments, output=arguments["query"])
    with pytest.raises(PagedAttentionError, match="must not overlap"):
        paged_attention(**arguments, output=arguments["value_buffer"].view(-1, 4, 64)[:2])


def test_gradients_are_refused():
    arguments = _arguments()
    query = arguments["query"].clone().requires_grad_()
    with pytest.raises(PagedAttentionError, match="no gradient"):
        paged_attention(**{**arguments, "query": query})


def _block(**overrides):
    """A block whose pointers are never followed: every case is refused before a launch."""

    args = _native.PagedAttentionArgs()
    args.struct_size = ctypes.sizeof(_native.PagedAttentionArgs)
    args.query = args.output = args.key_buffer = args.value_buffer = args.page_table = args.kv_lengths = 64
    args.query_token_stride, args.query_head_stride = 256, 64
    args.num_queries = args.num_requests = 2
    args.num_slots, args.num_q_heads, args.num_kv_heads, args.head_dim = 32, 4, 2, 64
    args.kv_dtype, args.softmax_scale = _native.DTYPE_BFLOAT16, 0.125
    args.page_table_stride = args.page_table_columns = 40
    args.page_size, args.kv_lengths_dtype = 8, _native.DTYPE_INT32
    for name, value in overrides.items():
        setattr(args, name, value)
    return args


@pytest.mark.parametrize("overrides,reason", [
    (dict(num_q_heads=5), "kv_head_layout_mismatch"),
    (dict(num_kv_heads=0), "kv_head_layout_mismatch"),
    (dict(num_q_heads=131072), "kv_head_layout_mismatch"),
    (dict(head_dim=96), "head_dimension_out_of_range"),
    (dict(kv_dtype=_native.DTYPE_FLOAT32), "fp16_or_bf16_required"),
    (dict(softmax_scale=0.0), "invalid_argument"),
    (dict(softmax_scale=float("nan")), "invalid_argument"),
    (dict(num_queries=3), "invalid_argument"),
    (dict(num_queries=-1), "invalid_argument"),
    (dict(num_queries=2 ** 29, num_requests=2 ** 29), "invalid_argument"),
    (dict(num_requests=2 ** 30), "invalid_argument"),
    (dict(query_starts=64), "integer_token_maps_required"),
    (dict(kv_lengths_dtype=_native.DTYPE_FLOAT32), "integer_token_maps_required"),
    (dict(page_size=0), "invalid_argument"),
    (dict(page_size=2 ** 30, page_table_columns=1), "invalid_argument"),
    (dict(page_table_columns=2 ** 27), "invalid_argument"),
    (dict(page_table_columns=-1), "invalid_argument"),
    (dict(page_table_stride=-1), "invalid_argument"),
    (dict(num_slots=2 ** 31), "invalid_argument"),
    (dict(query_token_stride=255), "invalid_argument"),
    (dict(query_head_stride=4), "invalid_argument"),
    (dict(query=None), "invalid_argument"),
    (dict(query=72), "invalid_argument"),
    (dict(output=72), "invalid_argument"),
    (dict(key_buffer=None), "invalid_argument"),
    (dict(page_table=None), "invalid_argument"),
    (dict(num_queries=2 ** 27, num_requests=2 ** 27), "invalid_argument"),  # more than a launch holds
    (dict(workspace=None), "invalid_argument"),
    (dict(workspace=64, workspace_bytes=64), "invalid_argument"),
    (dict(workspace=72, workspace_bytes=2 ** 40), "invalid_argument"),
])
def test_the_c_entry_refuses_before_any_launch(overrides, reason):
    with pytest.raises(_native.NativeCallError) as error:
        _native.paged_attention(_block(**overrides), 0)
    assert error.value.reason == reason


def test_the_c_entry_checks_its_struct():
    lib = _native.load_library()
    assert lib.ll_paged_attention(None, None) == _native.LL_ERR_INVALID_ARGUMENT
    assert lib.ll_paged_attention_workspace_bytes(None) == _native.LL_ERR_INVALID_ARGUMENT
    args = _block(struct_size=8)
    assert lib.ll_paged_attention(ctypes.byref(args), None) == _native.LL_ERR_INVALID_ARGUMENT
    assert "struct_size" in lib.ll_last_error().decode()


def test_nothing_to_do_launches_nothing():
    for empty in (dict(num_queries=0, num_requests=0), dict(num_queries=0, query_starts=64,
                                                            query_starts_dtype=_native.DTYPE_INT64)):
        args = _block(query=None, output=None, **empty)
        assert _native.paged_attention_workspace_bytes(args) == 0
        _native.paged_attention(args, 0)


def test_the_workspace_follows_from_the_shapes():
    assert _native.paged_attention_workspace_bytes(_block(page_table_columns=4)) == 0  # 32 keys: never split
    small = _native.paged_attention_workspace_bytes(_block())
    assert small > 0 and _native.paged_attention_workspace_bytes(_block(page_table_columns=2 ** 20)) == small
    assert _native.paged_attention_workspace_bytes(_block(num_queries=500, num_requests=500)) > small
    # Long prompts need no more than what is split: about 70 MB, whatever the lengths and heads.
    for heads, dim in ((1, 128), (4, 128), (8, 64), (2, 256), (300, 64)):
        prompt = dict(num_queries=100000, num_requests=1, query_starts=64, query_starts_dtype=_native.DTYPE_INT64,
                      num_q_heads=heads, num_kv_heads=heads, head_dim=dim, page_table_columns=2 ** 20)
        assert 0 < _native.paged_attention_workspace_bytes(_block(**prompt)) < 85 * 10 ** 6 * max(1, heads / 256)
    with pytest.raises(_native.NativeCallError):
        _native.paged_attention_workspace_bytes(_block(head_dim=96))
