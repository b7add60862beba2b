"""Forward-mode tangents are refused as reverse-mode gradients are: the step's
operators would drop them (on the CPU: refusals only)."""

from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from legolink_amd.head_rotary import HeadRotaryError, append_rotated_kv_inplace, rotate_heads
from legolink_amd.paged_attention import PagedAttentionError, paged_attention
from tests.test_head_rotary import _append, _heads
from tests.test_paged_attention import _arguments
from tests.test_step_calls import _append as native_append
from tests.test_step_calls import _attend as native_attend
from tests.test_step_calls import _rotate as native_rotate


def _dual(tensor):
    return forward_ad.make_dual(tensor, torch.ones_like(tensor))


CALLS = {
    "rotate": (lambda: {**_heads()[0], "query_norm_weight": torch.ones(32)}, native_rotate, rotate_heads,
               HeadRotaryError, ["query", "key", "cos_sin_cache", "query_norm_weight"]),
    "append": (lambda: {**_append(), "key_norm_weight": torch.ones(32)}, native_append, append_rotated_kv_inplace,
               HeadRotaryError, ["query", "key", "value", "cos_sin_cache", "key_norm_weight", "key_buffer",
                                 "value_buffer"]),
    "attention": (_arguments, native_attend, paged_attention, PagedAttentionError,
                  ["query", "key_buffer", "value_buffer"]),
}


@pytest.mark.parametrize("call,name", [(call, name) for call, parts in CALLS.items() for name in parts[4]])
def test_tangents_are_refused(call, name):
    make, native, operator, error, _ = CALLS[call]
    for no_grad in (False, True):  # no_grad does not switch forward mode off
        with forward_ad.dual_level(), torch.set_grad_enabled(not no_grad):
            arguments = make()
            arguments[name] = _dual(arguments[name])
            assert native(arguments) is None
            with pytest.raises(error, match="no gradient"):
                operator(**arguments)


@pytest.mark.parametrize("call", list(CALLS))
def test_other_tensors_are_taken_inside_a_dual_level(call):
    make, native, operator, error, _ = CALLS[call]
    with forward_ad.dual_level():
        assert native(make()) is True
        with pytest.raises(error, match="device tensors are required"):
            operator(**make())
