"""The native step calls take a call only where the Python checks support it:
their checks alone (entry 0), on the CPU."""

from __future__ import annotations

import os
import subprocess
import sys
from pathlib import Path

import pytest
import torch

from legolink_amd import _native, head_rotary, paged_attention
from tests import test_head_rotary as rotary_cases
from tests import test_paged_attention as attention_cases

_step_calls = _native.step_calls()


def _parameters(test, name):
    """The argument values of a parametrised test of the refusals."""

    for mark in test.pytestmark:
        if mark.name == "parametrize":
            return [values[mark.args[0].split(",").index(name)] for values in mark.args[1]]
    raise AssertionError(name)


def _rotate(arguments):
    get = {"is_neox_style": True, "norm_eps": 1e-6, **arguments}.get
    return _step_calls.rotate_heads(0, 0, 0, *(get(name) for name in (
        "query", "key", "positions", "cos_sin_cache", "rotary_dim", "is_neox_style", "query_norm_weight",
        "key_norm_weight", "norm_eps", "skipped_rows", "query_output", "key_output")))


def _append(arguments):
    get = {"is_neox_style": True, "norm_eps": 1e-6, **arguments}.get
    return _step_calls.append(0, 0, 0, *(get(name) for name in (
        "query", "key", "positions", "cos_sin_cache", "rotary_dim", "is_neox_style", "query_norm_weight",
        "key_norm_weight", "norm_eps", "skipped_rows", "query_output", "value", "key_buffer", "value_buffer",
        "destination_slots")))


def _attend(arguments):
    get = arguments.get
    return _step_calls.paged_attention(0, 0, 0, 0, *(get(name) for name in (
        "query", "key_buffer", "value_buffer", "page_table", "kv_lengths", "page_size", "query_starts", "scale")))


def test_the_module_is_built_for_this_torch():
    assert _step_calls is not None
    assert head_rotary._calls is _step_calls and paged_attention._calls is _step_calls


def test_plain_calls_are_taken():
    arguments, value = rotary_cases._heads()
    assert _rotate(arguments) is True
    assert _rotate({**arguments, "query_output": arguments["query"], "key_output": arguments["key"]}) is True
    assert _rotate({**arguments, "query_norm_weight": torch.ones(32), "skipped_rows": torch.zeros(1, dtype=torch.int64),
                    "positions": arguments["positions"].int(), "is_neox_style": False}) is True
    append = rotary_cases._append()
    assert _append(append) is True
    assert _append({**append, "query_output": append["query"], "destination_slots": append["destination_slots"].int(),
                    "cos_sin_cache": append["cos_sin_cache"].to(torch.bfloat16)}) is True
    arguments = attention_cases._arguments()
    assert _attend(arguments) is True
    assert _attend({**arguments, "query": torch.zeros(5, 4, 64, dtype=torch.bfloat16), "scale": 0.5,
                    "query_starts": torch.tensor([0, 2, 5])}) is True


@pytest.mark.parametrize("change", _parameters(rotary_cases.test_rotate_heads_refuses, "change"))
def test_rotate_heads_declines_what_python_refuses(change):
    arguments, _ = rotary_cases._heads()
    assert _rotate({**arguments, **change}) is None


@pytest.mark.parametrize("change", _parameters(rotary_cases.test_append_refuses, "change"))
def test_append_declines_what_python_refuses(change):
    assert _append({**rotary_cases._append(), **change}) is None


@pytest.mark.parametrize("change", [c for c in _parameters(attention_cases.test_paged_attention_refuses, "change")
                                    if "output" not in c])
def test_paged_attention_declines_what_python_refuses(change):
    assert _attend({**attention_cases._arguments(), **change}) is None


def test_overlaps_and_gradients_are_declined():
    append = rotary_cases._append()
    pool = append["key_buffer"]
    assert _append({**append, "key": pool[2:5]}) is None
    assert _append({**append, "value_buffer": pool}) is None
    assert _append({**append, "value": append["query"][:, :2], "query_output": append["query"]}) is None
    arguments, _ = rotary_cases._heads()
    query = arguments["query"]
    assert _rotate({**arguments, "key": query[:, 2:], "query_output": query}) is None
    assert _rotate({**arguments, "query_output": torch.zeros(3, 4, 32, dtype=torch.bfloat16)}) is None
    expanded = torch.zeros(1, 4, 32, dtype=torch.bfloat16).expand(3, 4, 32)
    assert _rotate({**arguments, "query": expanded}) is True
    assert _rotate({**arguments, "query": expanded, "query_output": expanded}) is None
    leaf = query.clone().requires_grad_()
    assert _rotate({**arguments, "query": leaf}) is None
    with torch.no_grad():
        assert _rotate({**arguments, "query": leaf}) is True
    attention = attention_cases._arguments()
    assert _attend({**attention, "query": attention["query"].clone().requires_grad_()}) is None


@pytest.mark.parametrize("arguments", [(), (1,), tuple(range(15)), tuple(range(18)), tuple(range(12)), (None,) * 15,
                                       (None,) * 18, (None,) * 12, ("x",) * 15, (0, 0, 0, *("x",) * 12),
                                       (0, 0, 0, *("x",) * 15), (0, 0, 0, 0, *("x",) * 8), (2 ** 70,) * 15])
def test_arguments_of_other_types_are_declined(arguments):
    for call in (_step_calls.rotate_heads, _step_calls.append, _step_calls.paged_attention):
        assert call(*arguments) is None


def test_the_operators_import_without_the_module(tmp_path):
    """As from a tree where it is not built: the Python checks take the calls."""

    code = ("import sys\nsys.modules['legolink_amd._step_calls'] = None\n"
            "from legolink_amd import head_rotary, paged_attention\n"
            "assert head_rotary._calls is None and paged_attention._calls is None\nprint('IMPORTED')\n")
    root = Path(__file__).resolve().parents[1]
    result = subprocess.run([sys.executable, "-c", code], cwd=tmp_path, capture_output=True, text=True, timeout=300,
                            env={**os.environ, "PYTHONPATH": str(root / "sglang-legolink_amd")})
    assert "IMPORTED" in result.stdout, result.stderr[-2000:]
