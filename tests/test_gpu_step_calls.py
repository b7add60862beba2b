"""GPU tests of the native step calls: the results of the Python checks' calls,
bit for bit, and the same refusals."""

from __future__ import annotations

import pytest
import torch

from legolink_amd import _native, head_rotary, paged_attention
from tests.test_gpu_head_rotary import _case as heads_case
from tests.test_gpu_paged_attention import _case as attention_case

pytestmark = pytest.mark.gpu


@pytest.fixture(params=["native", "python"])
def path(request, monkeypatch):
    if request.param == "python":
        monkeypatch.setattr(head_rotary, "_calls", None)
        monkeypatch.setattr(paged_attention, "_calls", None)
    return request.param


def _both(monkeypatch, call):
    native = call()
    with monkeypatch.context() as patch:
        patch.setattr(head_rotary, "_calls", None)
        patch.setattr(paged_attention, "_calls", None)
        python = call()
    return native, python


@pytest.mark.parametrize("layout", ["fused", "by head", "odd"])
@pytest.mark.parametrize("weights", [None, torch.bfloat16])
def test_both_paths_give_the_same_heads(gpu_device, monkeypatch, layout, weights):
    arguments, value = heads_case(gpu_device, tokens=21, layout=layout, weights=weights)
    native, python = _both(monkeypatch, lambda: head_rotary.rotate_heads(**arguments))
    for a, b in zip(native, python):
        assert a.is_contiguous() and torch.equal(a.view(torch.int16), b.view(torch.int16))
    pools = []

    def append():
        pool = torch.zeros(2, 64, 2, 128, dtype=torch.bfloat16, device=gpu_device)
        pools.append(pool)
        return head_rotary.append_rotated_kv_inplace(key_buffer=pool[0], value_buffer=pool[1], value=value,
                                                     destination_slots=torch.arange(21, device=gpu_device) * 3,
                                                     **arguments)

    native, python = _both(monkeypatch, append)
    assert torch.equal(native, python) and torch.equal(pools[0], pools[1]) and bool(pools[0].any())


@pytest.mark.parametrize("queries", [None, [3, 40, 0]])
def test_both_paths_give_the_same_attention(gpu_device, monkeypatch, queries):
    case = attention_case(gpu_device, [700, 90, 2], queries, heads=(28, 4))
    native, python = _both(monkeypatch, lambda: paged_attention.paged_attention(**case, scale=0.07))
    assert torch.equal(native.view(torch.int16), python.view(torch.int16))
    assert torch.equal(paged_attention.paged_attention(**case),
                       paged_attention.paged_attention(**case, output=torch.empty_like(case["query"])))


def test_refusals_name_their_reason(gpu_device, path):
    arguments, _ = heads_case(gpu_device, tokens=3)
    with pytest.raises(head_rotary.HeadRotaryError, match="rotary_dim"):
        head_rotary.rotate_heads(**{**arguments, "rotary_dim": 130})
    with pytest.raises(head_rotary.HeadRotaryError, match="positions"):
        head_rotary.rotate_heads(**{**arguments, "positions": arguments["positions"].cpu()})
    case = attention_case(gpu_device, [5, 6], heads=(4, 2))
    with pytest.raises(paged_attention.PagedAttentionError, match="kv_lengths"):
        paged_attention.paged_attention(**{**case, "kv_lengths": case["kv_lengths"][:1]})
    with pytest.raises(paged_attention.PagedAttentionError, match="on the query's device"):
        paged_attention.paged_attention(**{**case, "page_table": case["page_table"].cpu()})
    with pytest.raises(paged_attention.PagedAttentionError, match="no gradient"):
        paged_attention.paged_attention(**{**case, "query": case["query"].clone().requires_grad_()})


def test_a_status_of_the_library_is_raised(gpu_device, path):
    """A table row of 2^30 keys is refused by the library's own check."""

    case = attention_case(gpu_device, [5], heads=(4, 2))
    with pytest.raises(_native.NativeCallError, match="table row"):
        paged_attention.paged_attention(**{**case, "page_size": 2 ** 30})
