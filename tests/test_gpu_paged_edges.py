"""GPU tests of paged attention at the edges of its ranges, against 64 bits."""

from __future__ import annotations

import pytest
import torch

from legolink_amd.paged_attention import paged_attention
from tests.gpu_helpers import report
from tests.test_gpu_paged_attention import _case, _check, _check_marked, _marked

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("queries", [None, [1, 40, 3, 65], [60, 128, 1, 70]])
@pytest.mark.parametrize("heads,dim,page", [((28, 4), 128, 16), ((14, 2), 64, 1), ((7, 1), 256, 32)])
def test_tables_of_at_most_128_keys(gpu_device, queries, heads, dim, page):
    """Calls that are never split: one chunk of 65 to 128 keys."""

    report(f"unsplit, queries {queries} heads {heads} dim {dim} page {page}")
    case = _case(gpu_device, [65, 128, 127, 100], queries, heads=heads, dim=dim, page=page, spare_columns=0)
    assert case["page_table"].shape[1] * page == 128
    _check(paged_attention(**case), case)
    _check_marked(paged_attention(**_marked(case)), case)


@pytest.mark.parametrize("queries", [None, [200, 1]])
@pytest.mark.parametrize("scale", [1e-37, 1e-30])
def test_the_smallest_scales_weigh_all_keys_alike(gpu_device, queries, scale):
    case = _case(gpu_device, [300, 64], queries, heads=(4, 2), dim=64, dtype=torch.bfloat16)
    _check(paged_attention(**case, scale=scale), case, scale=scale)
