"""The native calls over an 8-bit pool take a call only where the Python checks
support it: their checks alone (entry 0), on the CPU."""

from __future__ import annotations

import pytest
import torch

from legolink_amd import _native, quantized_pool
from tests import test_quantized_pool as cases

_calls = _native.step_calls()
_POOL = ("key_buffer", "value_buffer", "key_scales", "value_scales", "scale_block")


def _take(name, arguments):
    get = {"is_neox_style": True, "norm_eps": 1e-6, "prefix_token_count": 0, "dtype": torch.bfloat16, **arguments}.get
    if name == "append":
        return _calls.quantized_append(0, 0, 0, *(get(n) for n in (
            "query", "key", "positions", "cos_sin_cache", "rotary_dim", "is_neox_style", "query_norm_weight",
            "key_norm_weight", "norm_eps", "skipped_rows", "query_output", "value", "destination_slots", *_POOL)))
    if name == "link":
        return _calls.quantized_link(0, 0, 0, *(get(n) for n in (
            *_POOL, "source_slots", "destination_slots", "local_positions", "global_positions", "cos_sin_cache",
            "rotary_dim", "is_neox_style", "prefix_token_count", "repair_mask", "skipped_rows")))
    if name == "load":
        return _calls.quantized_load(0, 0, 0, *(get(n) for n in (*_POOL, "slots")),
                                     quantized_pool._FLOAT_DTYPES.get(get("dtype")))
    return _calls.quantized_attention(0, 0, 0, 0, *(get(n) for n in (
        "query", *_POOL, "page_table", "kv_lengths", "page_size", "query_starts", "scale")))


def test_plain_calls_are_taken():
    assert quantized_pool._calls is _calls is not None
    for name, (_, arguments) in cases.CALLS.items():
        assert _take(name, arguments()) is True, name
    append = cases._append()
    assert _take("append", {**append, "query_output": append["query"], "positions": append["positions"].int(),
                            "query_norm_weight": torch.ones(64), "skipped_rows": torch.zeros(1, dtype=torch.int64),
                            "is_neox_style": False}) is True
    assert _take("link", {**cases._link(), "repair_mask": torch.zeros(3, dtype=torch.bool), "prefix_token_count": 3,
                          "skipped_rows": torch.zeros(1, dtype=torch.int64)}) is True
    assert _take("load", {**cases._load(), "slots": None, "dtype": torch.float32}) is True
    assert _take("attention", {**cases._attention(), "query": torch.zeros(5, 4, 64, dtype=torch.bfloat16), "scale": 0.5,
                               "query_starts": torch.tensor([0, 2, 5])}) is True


@pytest.mark.parametrize("name", cases.CALLS)
@pytest.mark.parametrize("change", [change for change, _ in cases.POOL_REFUSALS])
def test_a_bad_pool_is_declined(name, change):
    assert _take(name, {**cases.CALLS[name][1](), **change}) is None


REFUSALS = [*(("append", change) for change, _ in cases.APPEND_REFUSALS),
            *(("link", change) for change, _ in cases.LINK_REFUSALS),
            *(("load", change) for change, _ in cases.LOAD_REFUSALS if not any("output" in key for key in change)),
            *(("attention", change) for change, _ in cases.ATTENTION_REFUSALS if "output" not in change)]


@pytest.mark.parametrize("name,change", REFUSALS)
def test_what_python_refuses_is_declined(name, change):
    assert _take(name, {**cases.CALLS[name][1](), **change}) is None


def test_overlaps_gradients_and_tangents_are_declined():
    append, link = cases._append(), cases._link()
    for change in (dict(value_buffer=append["key_buffer"]), dict(value_scales=append["key_scales"]),
                   dict(value=append["key_buffer"].view(torch.bfloat16).view(-1)[:384].view(3, 2, 64)),
                   dict(skipped_rows=append["positions"][:1]),
                   dict(cos_sin_cache=append["key_buffer"].view(torch.float32).view(-1, 64)),
                   dict(key=append["query"][:, :2], query_output=append["query"])):
        assert _take("append", {**append, **change}) is None
    for change in (dict(cos_sin_cache=link["key_buffer"].view(torch.float32).view(-1, 64)),
                   dict(skipped_rows=link["source_slots"][:1]),
                   dict(repair_mask=link["key_scales"].view(torch.uint8).view(-1)[:3])):
        assert _take("link", {**link, **change}) is None
    for name, changed in (("append", "query"), ("append", "cos_sin_cache"), ("link", "cos_sin_cache"),
                          ("attention", "query")):
        arguments = cases.CALLS[name][1]()
        assert _take(name, {**arguments, changed: arguments[changed].clone().requires_grad_()}) is None
        with torch.autograd.forward_ad.dual_level():
            dual = torch.autograd.forward_ad.make_dual(arguments[changed], torch.ones_like(arguments[changed]))
            with torch.no_grad():
                assert _take(name, {**arguments, changed: dual}) is None


def test_rows_off_alignment_and_blocks_below_16_are_left_to_python():
    append = cases._append()
    odd = torch.zeros(3 * 2 * 64 + 1, dtype=torch.bfloat16)[1:].view(3, 2, 64)
    assert _take("append", {**append, "key": odd}) is None
    assert _take("append", {**append, "key_norm_weight": torch.zeros(65, dtype=torch.bfloat16)[1:]}) is None
    assert _take("attention", {**cases._attention(), **cases._pool(block=8)}) is None
    for name, arguments in cases.CALLS.items():
        assert _take(name, {**arguments[1](), "scale_block": True}) is None
