"""Sizes that are no whole numbers are refused, not cut down to one."""

from __future__ import annotations

import pytest

from legolink_amd.head_rotary import HeadRotaryError, append_rotated_kv_inplace, rotate_heads
from legolink_amd.paged_attention import PagedAttentionError, paged_attention
from tests.test_head_rotary import _append, _heads
from tests.test_paged_attention import _arguments
from tests.test_step_calls import _append as native_append
from tests.test_step_calls import _attend as native_attend
from tests.test_step_calls import _rotate as native_rotate


@pytest.mark.parametrize("size", [8.5, 15.999, float("nan"), float("inf"), "8", None])
def test_sizes_are_whole_numbers(size):
    arguments = {**_arguments(), "page_size": size}
    assert native_attend(arguments) is None
    with pytest.raises(PagedAttentionError, match="page_size"):
        paged_attention(**arguments)
    for native, operator, arguments in ((native_rotate, rotate_heads, _heads()[0]),
                                        (native_append, append_rotated_kv_inplace, _append())):
        arguments["rotary_dim"] = size
        assert native(arguments) is None
        with pytest.raises(HeadRotaryError, match="rotary_dim"):
            operator(**arguments)


def test_a_whole_number_of_another_type_is_one():
    with pytest.raises(PagedAttentionError, match="device tensors are required"):
        paged_attention(**{**_arguments(), "page_size": 8.0})
    with pytest.raises(HeadRotaryError, match="device tensors are required"):
        rotate_heads(**{**_heads()[0], "rotary_dim": 32.0})
