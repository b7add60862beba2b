"""A tensor in two roles of a step's call: what is written may be its own input,
and meets nothing else that the call reads or writes, also where the other is the
same tensor object.  Refusals of the Python checks, and the native checks decline
every such call (on the CPU: no call reaches a device)."""

from __future__ import annotations

import pytest
import torch

from legolink_amd.head_rotary import HeadRotaryError, append_rotated_kv_inplace, rotate_heads
from legolink_amd.paged_attention import PagedAttentionError, paged_attention
from legolink_amd.rope import build_cos_sin_cache
from tests.test_head_rotary import _append, _heads
from tests.test_paged_attention import _arguments
from tests.test_step_calls import _append as native_append
from tests.test_step_calls import _rotate as native_rotate


def _same(heads=2):
    """One tensor that may stand for queries, keys and values."""

    rows = torch.zeros(3, heads, 32, dtype=torch.bfloat16)
    return rows, dict(query=rows, key=rows, positions=torch.arange(3), rotary_dim=32,
                      cos_sin_cache=build_cos_sin_cache(16, 32))


@pytest.mark.parametrize("outputs", [("query_output",), ("key_output",), ("query_output", "key_output")])
def test_queries_and_keys_of_one_tensor_are_not_rotated_in_place(outputs):
    rows, arguments = _same()
    for view in (rows, rows.view_as(rows)):  # the same object, and another of the same rows
        call = {**arguments, "key": view}
        call.update({name: call[name.removesuffix("_output")] for name in outputs})
        assert native_rotate(call) is None
        with pytest.raises(HeadRotaryError, match="overlap"):
            rotate_heads(**call)


def test_queries_and_keys_of_one_tensor_are_taken_with_new_outputs():
    _, arguments = _same()
    assert native_rotate(arguments) is True
    with pytest.raises(HeadRotaryError, match="device tensors are required"):
        rotate_heads(**arguments)


@pytest.mark.parametrize("names", [("key",), ("value",), ("key", "value")])
def test_appended_rows_are_not_the_queries_in_place(names):
    append = _append(q_heads=2)
    call = {**append, **{name: append["query"] for name in names}, "query_output": append["query"]}
    assert native_append(call) is None
    with pytest.raises(HeadRotaryError, match="query_output"):
        append_rotated_kv_inplace(**call)
    call.pop("query_output")  # to a new tensor they may be
    assert native_append(call) is True
    with pytest.raises(HeadRotaryError, match="device tensors are required"):
        append_rotated_kv_inplace(**call)


def _inside(rows, like, dtype):
    """A tensor of ``like``'s shape over the bytes of ``rows``."""

    return rows.flatten().view(dtype)[:like.numel()].view(like.shape)


# What a call reads beside its rows: a tensor of this type.
READ = {"positions": torch.int64, "cos_sin_cache": torch.float32, "query_norm_weight": torch.float32,
        "skipped_rows": torch.int64}


@pytest.mark.parametrize("name", list(READ))
@pytest.mark.parametrize("output", ["query_output", "key_output"])
def test_outputs_over_what_a_rotation_reads_are_refused(name, output):
    arguments, _ = _heads(tokens=40, rotary=2)
    arguments = {k: v.clone() if isinstance(v, torch.Tensor) else v for k, v in arguments.items()}
    arguments.update(query_norm_weight=torch.ones(32), skipped_rows=torch.zeros(1, dtype=torch.int64),
                     cos_sin_cache=build_cos_sin_cache(16, 2))
    source = output.removesuffix("_output")
    assert native_rotate({**arguments, output: arguments[source]}) is True
    arguments[name] = _inside(arguments[source], arguments[name], READ[name])
    assert native_rotate({**arguments, output: arguments[source]}) is None
    with pytest.raises(HeadRotaryError, match=f"{output}|skipped_rows"):
        rotate_heads(**arguments, **{output: arguments[source]})
    new = torch.zeros_like(arguments[source])
    arguments[name] = _inside(new, arguments[name], READ[name])
    with pytest.raises(HeadRotaryError, match=f"{output}|skipped_rows"):
        rotate_heads(**arguments, **{output: new})


@pytest.mark.parametrize("name", [*READ, "destination_slots"])
@pytest.mark.parametrize("written", ["query_output", "key_buffer", "value_buffer"])
def test_what_an_append_reads_is_not_written(name, written):
    append = _append(tokens=40, rotary=2)
    append = {k: v.clone() if isinstance(v, torch.Tensor) else v for k, v in append.items()}
    append.update(query_norm_weight=torch.ones(32), skipped_rows=torch.zeros(1, dtype=torch.int64),
                  cos_sin_cache=build_cos_sin_cache(16, 2), query_output=append["query"],
                  key_buffer=torch.zeros(64, 2, 32, dtype=torch.bfloat16),
                  value_buffer=torch.zeros(64, 2, 32, dtype=torch.bfloat16))
    assert native_append(append) is True
    append[name] = _inside(append[written], append[name], READ.get(name, torch.int64))
    assert native_append(append) is None
    with pytest.raises(HeadRotaryError, match=f"{written}|skipped_rows"):
        append_rotated_kv_inplace(**append)


@pytest.mark.parametrize("name", ["positions", "cos_sin_cache", "key_norm_weight", "destination_slots", "value"])
def test_the_counter_of_skipped_rows_is_apart_from_what_is_read(name):
    append = {**_append(), "key_norm_weight": torch.ones(32)}
    append = {k: v.clone() if isinstance(v, torch.Tensor) else v for k, v in append.items()}
    append["skipped_rows"] = append[name].flatten().view(torch.int64)[:1]
    assert native_append(append) is None
    with pytest.raises(HeadRotaryError, match="skipped_rows"):
        append_rotated_kv_inplace(**append)


@pytest.mark.parametrize("name", ["query_starts", "kv_lengths", "page_table"])
def test_an_attention_output_over_what_it_reads_is_refused(name):
    arguments = {**_arguments(), "query_starts": torch.tensor([0, 1, 2])}
    output = torch.zeros_like(arguments["query"])
    arguments[name] = _inside(output, arguments[name], arguments[name].dtype)
    with pytest.raises(PagedAttentionError, match="overlap"):
        paged_attention(**arguments, output=output)
