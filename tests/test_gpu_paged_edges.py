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


@pytest.mark.parametrize("queries", [None, [130], [9]])
@pytest.mark.parametrize("length", [140, 900])
@pytest.mark.parametrize("dim,dtype", [(64, torch.bfloat16), (128, torch.float16), (256, torch.bfloat16)])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_scores_of_any_size_that_fp32_holds(gpu_device, queries, length, dim, dtype, sign):
    """Keys of equal largest scores share the weight alike, the others have none,
    whatever the scores: products that are exact in fp32, from 2^12 to 2^126 (fp16: to
    2^36), and scaled ones past its largest number."""

    report(f"score sizes, queries {queries} length {length} dim {dim} {dtype} sign {sign}")
    case = _case(gpu_device, [length], queries, heads=(4, 2), dim=dim, dtype=dtype, page=1)
    slots = case["page_table"][0, :length].long()
    tied = torch.tensor([0, 3, 5, 9], device=gpu_device)  # seen by every query
    keys = torch.full((length,), 0.75 if sign > 0 else 1.25, device=gpu_device)
    keys[tied] = 1.0
    want = case["value_buffer"][slots[tied]].double().mean(0).repeat_interleave(2, dim=0)  # [q heads, dim]
    bound = torch.finfo(dtype).eps / 2 * want.abs() + 8 * 2.0 ** -24 * 8  # the rounding, and sums in fp32
    # 2^power a query and a key: scores of dim 2^(2 power) scale.
    for power, scale in ((3, 1 / 3), (8, 1 / 3), (11, 1 / 3), (14, 1 / 3), *(
            ((30, 1 / 3), (59, 1 / 3), (59, 100.0)) if dtype == torch.bfloat16 else ((14, 1e28),))):
        case["query"].fill_(2.0 ** power)
        case["key_buffer"][slots] = (sign * 2.0 ** power * keys).to(dtype)[:, None, None]
        off = (paged_attention(**case, scale=scale).double() - want).abs()
        assert bool((off <= bound).all()), (power, scale, off.max().item())


@pytest.mark.parametrize("queries", [None, [40]])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_many_small_weights_beside_a_large_one(gpu_device, queries, dtype):
    """20,000 keys of weight 2^-26 beside one of weight 1, with values 64 times its:
    2 % of the result.  (256 KV heads: a workgroup takes all keys of one.)"""

    length, heads, dim = 20001, 256, 64
    case = _case(gpu_device, [length], queries, heads=(heads, heads), dim=dim, dtype=dtype, page=16)
    slot = int(case["page_table"][0, 0]) * 16  # key 0
    for name, first, rest in (("key_buffer", 0.0, -2.25), ("value_buffer", 1.0, 64.0)):
        case[name].fill_(rest)
        case[name][slot] = first
    case["query"].fill_(1.0)
    got = paged_attention(**case, scale=0.125).double()
    rows = got.shape[0]
    others = torch.arange(length - rows, length, dtype=torch.float64, device=gpu_device)  # that a query sees
    small = torch.exp(torch.tensor(-dim * 2.25 * 0.125, dtype=torch.float64, device=gpu_device))
    want = ((1.0 + small * others * 64.0) / (1.0 + small * others))[:, None, None]
    # The output's rounding; fp32 sums over the keys; of the small weights' part a
    # score's error (67 roundings of 18) and exp2's, and a weight's rounding: relative,
    # half a step, or in fp16's subnormal range 2^-25 on weights of up to 2^7.
    info = torch.finfo(dtype)
    bound = info.eps / 2 * want + (length + 64) * 2.0 ** -24 * want
    bound = bound + (want - 1.0) * (67 * 2.0 ** -24 * 18 + 2.0 ** -20 + info.eps / 2)
    if dtype == torch.float16:
        bound = bound + length * 2.0 ** -32 * 64.0
    assert bool(((got - want).abs() <= bound).all()), ((got - want).abs() / bound).max().item()
