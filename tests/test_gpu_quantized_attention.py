"""GPU tests of attention over an 8-bit pool, against 64 bits."""

from __future__ import annotations

import math

import pytest
import torch

from legolink_amd.paged_attention import paged_attention
from legolink_amd.quantized_pool import load_quantized_kv, quantized_paged_attention
from tests import quantized_pool_math as qm
from tests.gpu_helpers import report
from tests.paged_attention_math import allowed, attend

pytestmark = pytest.mark.gpu
POOL = ("key_buffer", "value_buffer", "key_scales", "value_scales", "scale_block")


def _case(device, lengths, queries=None, *, heads=(4, 2), dim=128, block=16, page=16, dtype=torch.bfloat16, seed=1,
          counts=torch.int32, extra_pages=3, spare_columns=2):
    """Requests of ``lengths`` keys and ``queries`` new tokens (None: one each);
    their pages in any order of a pool with pages of no request.  Values of about
    one, under scales of eight sizes."""

    generator = torch.Generator().manual_seed(seed)
    pages = [-(-n // page) for n in lengths]
    total = sum(pages) + extra_pages
    slots = total * page + (block if page > block else 0)  # the last rows are no whole page
    pool = {"scale_block": block}
    for name in ("key", "value"):
        scales = torch.randint(117, 125, (slots // block, heads[1]), generator=generator, dtype=torch.uint8)
        values = torch.randn(slots, heads[1], dim, generator=generator)
        codes = values / 2.0 ** (scales.float() - 127).repeat_interleave(block, 0)[..., None]
        pool[f"{name}_buffer"] = codes.clamp(-448, 448).to(torch.float8_e4m3fn).to(device)
        pool[f"{name}_scales"] = scales.view(torch.float8_e8m0fnu).to(device)
    order = torch.randperm(total, generator=generator).to(torch.int32)
    table = torch.full((len(lengths), max(pages, default=0) + spare_columns), 2 ** 31 - 1, dtype=torch.int32)
    taken = 0
    for request, count in enumerate(pages):
        table[request, :count] = order[taken:taken + count]
        taken += count
    rows = len(lengths) if queries is None else sum(queries)
    query = (1.5 * torch.randn(rows, heads[0], dim, generator=generator)).to(dtype).to(device)
    starts = None
    if queries is not None:
        starts = torch.tensor([0, *queries], device=device).cumsum(0).to(counts)
    return dict(query=query, **pool, page_table=table.to(device), query_starts=starts,
                kv_lengths=torch.tensor(lengths, device=device).to(counts), page_size=page)


def _check(got, case, scale=None):
    keys = qm.pool_values(case["key_buffer"], case["key_scales"], case["scale_block"])
    values = qm.pool_values(case["value_buffer"], case["value_scales"], case["scale_block"])
    want, size, reach = attend(case["query"], keys, values, case["page_table"], case["kv_lengths"].tolist(),
                               case["query_starts"], page=case["page_size"], scale=scale)
    covered = ~torch.isnan(want).any(-1).any(-1)
    longest = max([1, *case["kv_lengths"].tolist()])
    most = float(values[torch.isfinite(values)].abs().max()) if values.numel() else 0.0
    bound = allowed(want, size, reach, got.dtype, longest, most)[covered]
    off = (got.cpu().double() - want)[covered].abs()
    assert bool((off <= bound).all()), f"off by up to {(off / bound).max().item()} of the bound"


def _marked(case):
    """Uniform weights over values that mark each key's place: value d of key j is
    64 where j % dim == d, under a scale that differs from block to block."""

    page, dim, block = case["page_size"], case["query"].shape[2], case["scale_block"]
    case["query"].zero_()
    slots = case["value_buffer"].shape[0]
    marks = torch.full((slots, *case["value_buffer"].shape[1:]), 1024.0, device=case["query"].device)
    for request, length in enumerate(case["kv_lengths"].tolist()):
        place = torch.arange(length, device=case["query"].device)
        at = case["page_table"][request].long()[place // page] * page + place % page
        marks[at] = (torch.nn.functional.one_hot(place % dim, dim) * 64.0)[:, None]
    scales = (torch.arange(case["value_scales"].numel(), device=marks.device) % 5 + 129).view(case["value_scales"].shape)
    codes = marks / 2.0 ** (scales.float() - 127).repeat_interleave(block, 0)[..., None]
    case["value_buffer"].copy_(codes.to(torch.float8_e4m3fn))
    case["value_scales"].view(torch.uint8).copy_(scales)
    return case


def _check_marked(got, case):
    dim = case["query"].shape[2]
    lengths = case["kv_lengths"].tolist()
    starts = list(range(len(lengths) + 1)) if case["query_starts"] is None else case["query_starts"].tolist()
    got = got.cpu().double()
    for request, length in enumerate(lengths):
        for i in range(starts[request], starts[request + 1]):
            seen = max(0, length - (starts[request + 1] - 1 - i))
            counts = torch.bincount(torch.arange(seen) % dim, minlength=dim).double()
            read = got[i] * max(seen, 1) / 64.0
            # half a step of the output (2^-8 and 2^-11 of it) below half a key
            assert int(counts.max()) <= (100 if case["query"].dtype == torch.bfloat16 else 800)
            assert torch.equal(read.round(), counts.expand_as(read)), (request, i, seen)


LENGTHS = [1, 0, 15, 16, 17, 31, 32, 33, 64, 127, 128, 129, 640, 1023, 5000]


@pytest.mark.parametrize("heads,dim,block,page,dtype", [
    ((28, 4), 128, 16, 16, torch.bfloat16), ((28, 4), 128, 32, 32, torch.float16),
    ((64, 8), 128, 64, 64, torch.bfloat16), ((14, 2), 64, 16, 48, torch.float16),
    ((10, 10), 64, 128, 128, torch.bfloat16), ((7, 1), 256, 16, 16, torch.bfloat16),
    ((16, 2), 256, 128, 128, torch.float16), ((32, 1), 128, 16, 112, torch.bfloat16),
    ((96, 1), 64, 16, 16, torch.float16), ((2, 2), 256, 64, 192, torch.bfloat16),
])
def test_single_tokens(gpu_device, heads, dim, block, page, dtype):
    report(f"single tokens heads {heads} dim {dim} block {block} page {page} {dtype}")
    case = _case(gpu_device, LENGTHS, heads=heads, dim=dim, block=block, page=page, dtype=dtype)
    got = quantized_paged_attention(**case)
    _check(got, case)
    assert bool((got[1] == 0).all())  # no keys
    _check_marked(quantized_paged_attention(**_marked(case)), case)


CHUNKS = {
    "short": ([40, 3, 900, 17], [2, 3, 1, 4]),
    "eight": ([8, 300, 64, 65, 4500], [8, 8, 8, 7, 8]),
    "odd": ([701, 33, 1500, 129], [17, 33, 5, 129]),
    "prompt": ([517], [517]),
    "behind": ([1300, 2100], [260, 70]),
    "uneven": ([600, 40, 1, 900], [300, 0, 1, 2]),
    "mixed": ([700, 350, 64, 12, 1000, 31, 77, 500], [400, 1, 1, 1, 1, 1, 1, 1]),
    "too long": ([5, 0, 40], [9, 3, 40]),  # more new tokens than keys: the first see nothing
}


@pytest.mark.parametrize("chunks", list(CHUNKS))
@pytest.mark.parametrize("heads,dim,block,page,dtype", [
    ((28, 4), 128, 16, 16, torch.bfloat16), ((14, 2), 64, 16, 48, torch.float16), ((8, 8), 64, 64, 64, torch.bfloat16),
    ((16, 2), 256, 16, 16, torch.bfloat16), ((32, 1), 128, 32, 96, torch.float16), ((6, 6), 256, 128, 128, torch.float16),
])
def test_chunks(gpu_device, chunks, heads, dim, block, page, dtype):
    report(f"chunks {chunks} heads {heads} dim {dim} block {block} page {page} {dtype}")
    lengths, queries = CHUNKS[chunks]
    case = _case(gpu_device, lengths, queries, heads=heads, dim=dim, block=block, page=page, dtype=dtype,
                 counts=torch.int64)
    _check(quantized_paged_attention(**case), case)
    _check_marked(quantized_paged_attention(**_marked(case)), case)


@pytest.mark.parametrize("queries", [None, [40]])
@pytest.mark.parametrize("heads,dim,length", [((64, 64), 64, 30000), ((128, 128), 256, 16001), ((300, 300), 64, 9000)])
def test_chunks_longer_than_the_list_of_groups(gpu_device, queries, heads, dim, length):
    """With many KV heads a workgroup takes thousands of keys, and refills its list
    on the way."""

    report(f"long chunks, heads {heads} dim {dim} length {length} queries {queries}")
    case = _case(gpu_device, [length], queries, heads=heads, dim=dim, dtype=torch.float16)
    _check_marked(quantized_paged_attention(**_marked(case)), case)


@pytest.mark.parametrize("count,queries_of", [(150, lambda r: 1), (257, lambda r: 1), (1100, lambda r: 1),
                                              (2600, lambda r: r % 3), (300, lambda r: (7 * r) % 31)])
def test_many_requests(gpu_device, count, queries_of):
    queries = [queries_of(r) for r in range(count)]
    lengths = [0 if r % 53 == 17 else 1 + (29 * r) % 300 for r in range(count)]
    lengths[count // 2], lengths[count - 1] = 4097, 1500
    lengths = [max(length, n) if length else 0 for length, n in zip(lengths, queries)]
    single = all(n == 1 for n in queries)
    case = _marked(_case(gpu_device, lengths, None if single else queries, heads=(8, 2), dim=64))
    _check_marked(quantized_paged_attention(**case), case)


@pytest.mark.parametrize("count,spare", [(16, 600), (17, 0), (17, 600), (24, 600), (31, 600), (32, 0), (32, 600),
                                         (33, 600)])
@pytest.mark.parametrize("equal", [True, False])
def test_units_of_one_round_and_of_two(gpu_device, count, spare, equal):
    """Requests about a quarter and half of the places, in tables of few and of
    more than 8,192 keys."""

    report(f"{count} requests, {spare} spare columns, equal {equal}")
    lengths = [700] * count if equal else [(r * 397) % 1200 for r in range(count)]
    case = _case(gpu_device, lengths, heads=(16, 8), dim=128, spare_columns=spare)
    _check(quantized_paged_attention(**case), case)
    _check_marked(quantized_paged_attention(**_marked(case)), case)


@pytest.mark.parametrize("queries", [None, [1, 40, 3, 65], [60, 128, 1, 70]])
@pytest.mark.parametrize("heads,dim,page", [((28, 4), 128, 16), ((14, 2), 64, 32), ((7, 1), 256, 32)])
def test_tables_of_at_most_128_keys(gpu_device, queries, heads, dim, page):
    """Calls that are never split: one chunk of 65 to 128 keys."""

    report(f"unsplit, queries {queries} heads {heads} dim {dim} page {page}")
    case = _case(gpu_device, [65, 128, 127, 100], queries, heads=heads, dim=dim, page=page, spare_columns=0)
    assert case["page_table"].shape[1] * page == 128
    _check(quantized_paged_attention(**case), case)


@pytest.mark.parametrize("queries", [None, [70, 3, 1]])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_it_is_paged_attention_over_the_loaded_rows(gpu_device, queries, dtype):
    """Both are off by their roundings alone, each within the bound around 64 bits."""

    case = _case(gpu_device, [900, 65, 2000], queries, heads=(28, 4), dtype=dtype)
    keys, values = load_quantized_kv(**{name: case[name] for name in POOL}, dtype=dtype)
    other = paged_attention(case["query"], keys, values, case["page_table"], case["kv_lengths"],
                            page_size=case["page_size"], query_starts=case["query_starts"])
    _check(other, case)
    _check(quantized_paged_attention(**case), case)


@pytest.mark.parametrize("queries", [None, [3, 1, 2], [200, 5, 90]])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim,heads", [(64, (4, 2)), (128, (4, 2)), (256, (4, 2)), (64, (32, 32)), (64, (22, 22)),
                                       (128, (32, 32))])  # one, two and four heads a workgroup
def test_rows_that_are_not_seen_may_hold_anything(gpu_device, queries, dtype, dim, heads):
    """NaN behind a request's length, in pages of no request and in later tokens of a
    query's own chunk do not reach it, in codes and in scales."""

    report(f"unseen rows, queries {queries} {dtype} dim {dim} heads {heads}")
    lengths = [70, 31, 300] if queries != [200, 5, 90] else [270, 31, 300]
    case = _case(gpu_device, lengths, queries, heads=heads, dim=dim, dtype=dtype)
    want = quantized_paged_attention(**case)
    used = torch.zeros(case["key_buffer"].shape[0], dtype=torch.bool, device=gpu_device)
    for request, length in enumerate(lengths):
        place = torch.arange(length, device=gpu_device)
        used[case["page_table"][request].long()[place // 16] * 16 + place % 16] = True
    for name in ("key", "value"):
        case[f"{name}_buffer"].view(torch.uint8)[~used] = 0x7F
        case[f"{name}_scales"].view(torch.uint8)[~used.view(-1, 16).any(1)] = 255
    assert torch.equal(quantized_paged_attention(**case), want)
    if queries is None:
        return
    # The last key of each request: only its last query sees it.
    ends = case["query_starts"][1:].long() - 1
    others = torch.ones(case["query"].shape[0], dtype=torch.bool, device=gpu_device)
    others[ends] = False
    last = torch.tensor([int(case["page_table"][r, (n - 1) // 16]) * 16 + (n - 1) % 16 for r, n in enumerate(lengths)],
                        device=gpu_device)
    codes = case["value_buffer"].view(torch.uint8)
    kept = codes[last].clone()
    codes[last] = 0xFF
    got = quantized_paged_attention(**case)
    assert torch.equal(got[others], want[others]) and bool(torch.isnan(got[ends]).all())
    codes[last] = kept
    codes = case["key_buffer"].view(torch.uint8)
    kept = codes[last].clone()
    codes[last] = 0x7F
    got = quantized_paged_attention(**case)
    assert torch.equal(got[others], want[others]) and bool(torch.isnan(got[ends]).all())
    codes[last] = kept
    assert torch.equal(quantized_paged_attention(**case), want)


@pytest.mark.parametrize("queries", [[40], [300]])
@pytest.mark.parametrize("name", ["key_scales", "value_scales"])
def test_a_scale_of_nan_reaches_those_who_see_its_block(gpu_device, queries, name):
    """The request's last block, which its last queries see, in part or whole."""

    length = queries[0]
    case = _case(gpu_device, [length], queries, heads=(4, 2), dim=64)
    want = quantized_paged_attention(**case)
    first = (length - 1) // 16 * 16  # of the block's keys
    case[name].view(torch.uint8)[case["page_table"][0, first // 16].long(), 1] = 255
    got = quantized_paged_attention(**case)
    assert torch.equal(got[:first], want[:first]) and torch.equal(got[:, :2], want[:, :2])
    assert bool(torch.isnan(got[first:, 2:]).all())


@pytest.mark.parametrize("heads,dim", [((4, 2), 128), ((32, 16), 128), ((32, 16), 64), ((4, 2), 256)])
def test_single_tokens_over_a_scale_of_nan(gpu_device, heads, dim):
    case = _case(gpu_device, [100, 20], heads=heads, dim=dim)
    want = quantized_paged_attention(**case)
    case["value_scales"].view(torch.uint8)[case["page_table"][0, 6].long(), 0] = 255  # keys 96 to 99
    got = quantized_paged_attention(**case)
    assert bool(torch.isnan(got[0, :2]).all()) and torch.equal(got[0, 2:], want[0, 2:]) and torch.equal(got[1], want[1])


def test_fp16_takes_rows_past_its_range_as_infinities(gpu_device):
    """As load_quantized_kv gives them: seen they are infinite, unseen nothing."""

    for queries in (None, [50]):
        case = _case(gpu_device, [50], queries, heads=(2, 1), dim=64, dtype=torch.float16)
        want = quantized_paged_attention(**case)
        slot = int(case["page_table"][0, 2]) * 16 + 8  # key 40
        scales = case["value_scales"].view(torch.uint8)
        block = slot // 16
        case["value_buffer"].view(torch.uint8)[block * 16:block * 16 + 16, 0, 7] = 0
        scales[block, 0] = 127 + 9
        case["value_buffer"].view(torch.uint8)[slot, 0, 7] = 0x7E  # 448 * 2^9
        got = quantized_paged_attention(**case).cpu()
        if queries is None:
            assert bool((got[0, :, 7] == math.inf).all())
        else:
            assert torch.equal(got[:32], want[:32].cpu()) and bool((got[40:, :, 7] == math.inf).all())
            assert bool(torch.isfinite(got[32:40, :, 7]).all())


@pytest.mark.parametrize("queries", [None, [5, 40, 2], [150, 129, 1]])
def test_pages_outside_the_pool_are_invisible(gpu_device, queries):
    report(f"bad pages, queries {queries}")
    case = _case(gpu_device, [200, 129, 40], queries, heads=(6, 2), dim=64, page=32)
    pool_pages = case["key_buffer"].shape[0] // 32
    case["page_table"][0, 1] = -1
    case["page_table"][0, 5] = pool_pages  # the pool's last rows are no whole page
    case["page_table"][1, 0] = -2 ** 31
    case["page_table"][2, :] = 2 ** 31 - 1  # every page
    got = quantized_paged_attention(**case)
    _check(got, case)
    assert bool((got[-1] == 0).all())


def test_rows_of_no_request_keep_their_output(gpu_device):
    case = _case(gpu_device, [40, 70], [3, 5], heads=(4, 2), dim=64)
    query = torch.cat((case["query"], case["query"][:4]))
    output = torch.full_like(query, 7.0)
    got = quantized_paged_attention(**{**case, "query": query}, output=output)
    assert got is output and bool((output[8:] == 7).all())
    assert torch.equal(output[:8], quantized_paged_attention(**case))


def test_lengths_and_starts_outside_the_call_are_held_to_it(gpu_device):
    case = _case(gpu_device, [64, 64, 64], [4, 4, 4], heads=(4, 2), dim=64, spare_columns=0)
    want = quantized_paged_attention(**case)
    case["kv_lengths"].copy_(torch.tensor([2 ** 31 - 1, 64, -5]))
    got = quantized_paged_attention(**case)
    assert torch.equal(got[:8], want[:8]) and bool((got[8:] == 0).all())
    case["kv_lengths"].fill_(64)
    case["query_starts"].copy_(torch.tensor([-3, 4, 8, 2 ** 31 - 1]))
    assert torch.equal(quantized_paged_attention(**case), want)


@pytest.mark.parametrize("layout", ["fused", "by head", "odd"])
@pytest.mark.parametrize("queries", [None, [60, 2]])
def test_query_layouts(gpu_device, layout, queries):
    case = _case(gpu_device, [300, 77], queries, heads=(4, 2), dim=128)
    want = quantized_paged_attention(**case)
    query = case["query"]
    rows = query.shape[0]
    if layout == "fused":
        view = torch.zeros(rows, 8 * 128, dtype=query.dtype, device=gpu_device)[:, 2 * 128:6 * 128].unflatten(-1, (4, 128))
    elif layout == "by head":
        view = torch.zeros(4, rows, 128, dtype=query.dtype, device=gpu_device).transpose(0, 1)
    else:  # at an address that is no multiple of 16 bytes
        view = torch.zeros(rows * 4 * 128 + 1, dtype=query.dtype, device=gpu_device)[1:].view(rows, 4, 128)
    view.copy_(query)
    assert torch.equal(quantized_paged_attention(**{**case, "query": view}), want)


@pytest.mark.parametrize("scale", [1e-37, 1e-3, 1.0, 30.0])
@pytest.mark.parametrize("queries", [None, [70, 1]])
def test_scales(gpu_device, scale, queries):
    """Weights from uniform to nearly one-hot (scores of hundreds)."""

    case = _case(gpu_device, [900, 64], queries, heads=(4, 2), dim=64)
    if scale == 30.0:
        case["query"].div_(8)  # a score's error, exp(dim 2^-24 |score|), stays small
    _check(quantized_paged_attention(**case, scale=scale), case, scale=scale)


@pytest.mark.parametrize("queries", [None, [3], [200]])
def test_rising_scores(gpu_device, queries):
    """Keys whose scores rise (or fall) along the request by far more than the maximum's slack."""

    case = _case(gpu_device, [2000], queries, heads=(4, 1), dim=64)
    case["query"].fill_(1.0)
    case["key_scales"].view(torch.uint8).fill_(122)
    place = torch.arange(2000, device=gpu_device)
    slots = case["page_table"][0].long()[place // 16] * 16 + place % 16
    ramp = torch.linspace(-8, 8, 2000, device=gpu_device)[:, None, None].expand(2000, 1, 64) * 32
    for rows in (ramp, ramp.flip(0)):
        case["key_buffer"].view(torch.uint8)[slots] = rows.to(torch.float8_e4m3fn).view(torch.uint8)
        _check(quantized_paged_attention(**case), case)


@pytest.mark.parametrize("queries", [None, [130], [9]])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_scores_of_any_size_that_fp32_holds(gpu_device, queries, dim, sign):
    """Keys of equal largest scores share the weight alike, the others have none."""

    report(f"score sizes, queries {queries} dim {dim} sign {sign}")
    case = _case(gpu_device, [900], queries, heads=(4, 2), dim=dim)
    place = torch.arange(900, device=gpu_device)
    slots = case["page_table"][0].long()[place // 16] * 16 + place % 16
    tied = torch.tensor([0, 3, 5, 9], device=gpu_device)  # seen by every query
    keys = torch.full((900,), 0.75 if sign > 0 else 1.25, device=gpu_device)
    keys[tied] = 1.0
    rows = (sign * keys[:, None, None].expand(900, 2, dim)).to(torch.float8_e4m3fn)
    case["key_buffer"].view(torch.uint8)[slots] = rows.view(torch.uint8)
    values = qm.pool_values(case["value_buffer"], case["value_scales"], 16).to(gpu_device)
    want = values[slots[tied]].mean(0).repeat_interleave(2, dim=0)  # [q heads, dim]
    bound = torch.finfo(torch.bfloat16).eps / 2 * want.abs() + 8 * 2.0 ** -24 * 8  # the rounding, and sums in fp32
    for power, scale in ((8, 1 / 3), (14, 1 / 3), (30, 1 / 3), (59, 1 / 3), (59, 100.0)):
        case["query"].fill_(2.0 ** power)
        case["key_scales"].view(torch.uint8).fill_(127 + power)
        off = (quantized_paged_attention(**case, scale=scale).double() - want).abs()
        assert bool((off <= bound).all()), (power, scale, off.max().item())


def test_nothing_to_do(gpu_device):
    case = _case(gpu_device, [], heads=(4, 2), dim=64)
    assert quantized_paged_attention(**case).shape == (0, 4, 64)
    case = _case(gpu_device, [10, 20], [0, 0], heads=(4, 2), dim=64)
    assert quantized_paged_attention(**case).shape == (0, 4, 64)
    for slots in (0, 16):  # a pool without rows, and without a whole page: every key is invisible
        case = _case(gpu_device, [10, 20], heads=(4, 2), dim=64, page=32)
        for name in ("key", "value"):
            case[f"{name}_buffer"] = case[f"{name}_buffer"].view(torch.uint8)[:slots].clone().view(torch.float8_e4m3fn)
            case[f"{name}_scales"] = (case[f"{name}_scales"].view(torch.uint8)[:slots // 16].clone()
                                      .view(torch.float8_e8m0fnu))
        assert bool((quantized_paged_attention(**case) == 0).all())
    case = _case(gpu_device, [0, 0], heads=(4, 2), dim=64)
    case["page_table"] = case["page_table"][:, :0]
    assert bool((quantized_paged_attention(**case) == 0).all())


@pytest.mark.parametrize("starts", [None, [0, 100, 230]])
def test_pool_past_four_gib(gpu_device, starts):
    """Rows past 2^32 bytes: the same as those of a small pool."""

    slots = (1 << 32) // (2 * 128) + 4096
    far = {}
    small = qm.random_pool(512, 2, 128, 16, seed=3, low=117, high=121)
    for name, value in small.items():
        per = 16 if name.endswith("_scales") else 1
        big = torch.zeros(slots // per, *value.shape[1:], dtype=torch.uint8, device=gpu_device)
        big[-512 // per:] = value.view(torch.uint8).to(gpu_device)
        far[name] = big.view(value.dtype)
    table = torch.arange(32, dtype=torch.int32, device=gpu_device).flip(0).view(2, 16)
    rest = dict(page_size=16, scale_block=16, kv_lengths=torch.tensor([245, 250], device=gpu_device),
                query_starts=None if starts is None else torch.tensor(starts, device=gpu_device),
                query=torch.randn(2 if starts is None else 230, 4, 128, device=gpu_device).to(torch.bfloat16))
    got = quantized_paged_attention(**far, **rest, page_table=table + (slots - 512) // 16)
    near = {name: value.to(gpu_device) for name, value in small.items()}
    assert bool(got.any()) and torch.equal(got, quantized_paged_attention(**near, **rest, page_table=table))


@pytest.mark.parametrize("queries", [None, [6, 1, 9], [190, 64, 1]])
def test_a_captured_call_serves_other_lengths(gpu_device, queries):
    """One graph, replayed with other lengths, pages and starts, against eager calls."""

    case = _case(gpu_device, [700, 300, 512], queries, heads=(28, 4), dim=128)
    quantized_paged_attention(**case)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = quantized_paged_attention(**case)
    for lengths in ([700, 300, 512], [1, 0, 33], [129, 256, 500], [700, 1, 2]):
        case["kv_lengths"].copy_(torch.tensor(lengths))
        case["page_table"][0, :10] = case["page_table"][0, :10].flip(0)
        if queries is not None:
            total = case["query"].shape[0]
            case["query_starts"].copy_(torch.tensor([0, total // 3, total // 2, total]))
        captured.fill_(9)
        graph.replay()
        torch.cuda.synchronize()
        got = captured.clone()
        again = quantized_paged_attention(**case)
        torch.cuda.synchronize()
        assert torch.equal(got, again)
        _check(got, case)


def test_two_streams_at_once(gpu_device):
    """Calls in flight on two streams have workspaces of their own."""

    cases = [_case(gpu_device, [6000 + 100 * i], heads=(28, 4), seed=i) for i in range(2)]
    want = [quantized_paged_attention(**case) for case in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[], []]
    for _ in range(10):
        for i, (case, stream) in enumerate(zip(cases, streams)):
            with torch.cuda.stream(stream):
                got[i].append(quantized_paged_attention(**case))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(result, want[i]) for result in got[i])


@pytest.mark.parametrize("count", [8, 9, 13, 16])
@pytest.mark.parametrize("lengths", ["long", "just long", "just short", "short", "uneven"])
def test_rounds_go_by_the_lengths_of_the_call(gpu_device, count, lengths):
    """Calls in tables of long rows, from a quarter of the places to half of them:
    whichever target the lengths on the device make, every key counts once."""

    report(f"rounds, {count} requests, {lengths}")
    turn = math.ceil(500 * 1024 / count ** 2 / 64) * 64  # 32 places; 500 keys of 256 are 1,000 of 128
    of = {"long": lambda r: turn + 1200, "just long": lambda r: turn, "just short": lambda r: turn - 64,
          "short": lambda r: 40 + 61 * r, "uneven": lambda r: 0 if r % 5 == 3 else 9000 if r % 3 == 0 else 70}[lengths]
    case = _marked(_case(gpu_device, [of(r) for r in range(count)], heads=(16, 8), dim=256, spare_columns=300))
    _check_marked(quantized_paged_attention(**case), case)


def test_a_captured_call_turns_from_one_target_to_the_other(gpu_device):
    """One graph over tables of long rows, replayed with long and short lengths."""

    case = _marked(_case(gpu_device, [4200] * 14, heads=(16, 8), dim=256, spare_columns=100))
    quantized_paged_attention(**case)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = quantized_paged_attention(**case)
    for lengths in ([4200] * 14, [300] * 14, [4200] * 13 + [0], [1] * 14, [4200 - 13 * r for r in range(14)]):
        case["kv_lengths"].copy_(torch.tensor(lengths))
        captured.fill_(9)
        graph.replay()
        torch.cuda.synchronize()
        got = captured.clone()
        again = quantized_paged_attention(**case)
        torch.cuda.synchronize()
        assert torch.equal(got, again)
        _check_marked(got, case)
