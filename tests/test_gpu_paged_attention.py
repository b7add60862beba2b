"""GPU tests of paged attention against 64 bits."""

from __future__ import annotations

import math

import pytest
import torch

from legolink_amd.paged_attention import paged_attention
from tests.gpu_helpers import report
from tests.paged_attention_math import allowed, attend

pytestmark = pytest.mark.gpu


def _case(device, lengths, queries=None, *, heads=(4, 2), dim=128, page=16, dtype=torch.bfloat16, seed=1,
          counts=torch.int32, extra_pages=3, spare_columns=2):
    """Requests of ``lengths`` keys and ``queries`` new tokens (None: one each);
    their pages in any order of a pool with pages of no request."""

    generator = torch.Generator(device=device).manual_seed(seed)
    pages = [-(-n // page) for n in lengths]
    total = sum(pages) + extra_pages
    slots = total * page + (page // 2)  # the last rows are no whole page
    keys = torch.randn(slots, heads[1], dim, device=device, generator=generator).to(dtype)
    values = torch.randn(slots, heads[1], dim, device=device, generator=generator).to(dtype)
    order = torch.randperm(total, device=device, generator=generator).to(torch.int32)
    table = torch.full((len(lengths), max(pages, default=0) + spare_columns), 2 ** 31 - 1, dtype=torch.int32,
                       device=device)
    taken = 0
    for request, count in enumerate(pages):
        table[request, :count] = order[taken:taken + count]
        taken += count
    rows = len(lengths) if queries is None else sum(queries)
    query = (1.5 * torch.randn(rows, heads[0], dim, device=device, generator=generator)).to(dtype)
    starts = None
    if queries is not None:
        starts = torch.tensor([0, *queries], device=device).cumsum(0).to(counts)
    return dict(query=query, key_buffer=keys, value_buffer=values, page_table=table, query_starts=starts,
                kv_lengths=torch.tensor(lengths, device=device).to(counts), page_size=page)


def _check(got, case, scale=None):
    want, size, reach = attend(case["query"], case["key_buffer"], case["value_buffer"], case["page_table"],
                               case["kv_lengths"].tolist(), case["query_starts"], page=case["page_size"], scale=scale)
    covered = ~torch.isnan(want).any(-1).any(-1)
    longest = max([1, *case["kv_lengths"].tolist()])
    most = float(case["value_buffer"].float().abs().max()) if case["value_buffer"].numel() else 0.0
    bound = allowed(want, size, reach, got.dtype, longest, most)[covered]
    off = (got.cpu().double() - want)[covered].abs()
    assert bool((off <= bound).all()), f"off by up to {(off / bound).max().item()} of the bound"


def _marked(case):
    """Uniform weights (queries of zeros) over values that mark each key's place:
    value d of key j is 64 where j % dim == d.  Every query's count of keys by
    place can then be read off its output."""

    page, dim = case["page_size"], case["query"].shape[2]
    case["query"].zero_()
    case["value_buffer"].fill_(1000.0)  # rows of no request
    for request, length in enumerate(case["kv_lengths"].tolist()):
        place = torch.arange(length, device=case["query"].device)
        slots = case["page_table"][request].long()[place // page] * page + place % page
        rows = torch.nn.functional.one_hot(place % dim, dim) * 64.0
        case["value_buffer"][slots] = rows[:, None].to(case["value_buffer"].dtype)
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


LENGTHS = [1, 0, 31, 32, 33, 64, 127, 128, 129, 640, 1023, 5000]


@pytest.mark.parametrize("heads,dim,page,dtype", [
    ((28, 4), 128, 1, torch.bfloat16), ((28, 4), 128, 16, torch.float16), ((64, 8), 128, 64, torch.bfloat16),
    ((14, 2), 64, 48, torch.float16), ((10, 10), 64, 16, torch.bfloat16), ((7, 1), 256, 1, torch.bfloat16),
    ((16, 2), 256, 128, torch.float16), ((32, 1), 128, 7, torch.bfloat16), ((96, 1), 64, 16, torch.float16),
    ((2, 2), 256, 3, torch.bfloat16),
])
def test_single_tokens(gpu_device, heads, dim, page, dtype):
    report(f"single tokens heads {heads} dim {dim} page {page} {dtype}")
    case = _case(gpu_device, LENGTHS, heads=heads, dim=dim, page=page, dtype=dtype)
    got = paged_attention(**case)
    _check(got, case)
    assert bool((got[1] == 0).all())  # no keys
    _check_marked(paged_attention(**_marked(case)), case)


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
@pytest.mark.parametrize("heads,dim,page,dtype", [
    ((28, 4), 128, 16, torch.bfloat16), ((14, 2), 64, 1, torch.float16), ((8, 8), 64, 64, torch.bfloat16),
    ((16, 2), 256, 16, torch.bfloat16), ((32, 1), 128, 48, torch.float16), ((6, 6), 256, 5, torch.float16),
])
def test_chunks(gpu_device, chunks, heads, dim, page, dtype):
    report(f"chunks {chunks} heads {heads} dim {dim} page {page} {dtype}")
    lengths, queries = CHUNKS[chunks]
    case = _case(gpu_device, lengths, queries, heads=heads, dim=dim, page=page, dtype=dtype, counts=torch.int64)
    _check(paged_attention(**case), case)
    _check_marked(paged_attention(**_marked(case)), case)


@pytest.mark.parametrize("queries", [None, [40]])
@pytest.mark.parametrize("heads,dim,length", [((64, 64), 64, 30000), ((128, 128), 256, 16001), ((300, 300), 64, 9000)])
def test_chunks_longer_than_the_slot_list(gpu_device, queries, heads, dim, length):
    """With many KV heads a workgroup takes thousands of keys, and refills its list
    of slots on the way."""

    report(f"long chunks, heads {heads} dim {dim} length {length} queries {queries}")
    case = _case(gpu_device, [length], queries, heads=heads, dim=dim, page=16, dtype=torch.float16)
    _check_marked(paged_attention(**_marked(case)), case)


def test_more_requests_than_a_wave_scans_at_once(gpu_device):
    lengths = [(37 * i) % 211 for i in range(150)]
    lengths[70], lengths[149] = 4321, 1700
    case = _case(gpu_device, lengths, heads=(8, 2), dim=64)
    _check_marked(paged_attention(**_marked(case)), case)
    queries = [1 + (i % 3) for i in range(150)]
    case = _case(gpu_device, [max(n, q) for n, q in zip(lengths, queries)], queries, heads=(8, 2), dim=64)
    _check(paged_attention(**case), case)
    _check_marked(paged_attention(**_marked(case)), case)


@pytest.mark.parametrize("heads,dim", [((8, 1), 64), ((8, 1), 128), ((16, 2), 256)])
def test_chunks_of_more_requests_than_a_wave_orders_at_once(gpu_device, heads, dim):
    """150 requests of 0 to 30 queries over 0 to 449 keys, among them ones without
    queries, without keys, and many of the same length."""

    queries = [(7 * r) % 31 for r in range(150)]
    lengths = [0 if r % 23 == 5 else (3 * r if r < 150 // 2 else 64 * (r % 8)) for r in range(150)]
    lengths = [max(length, n) if length else 0 for length, n in zip(lengths, queries)]
    case = _marked(_case(gpu_device, lengths, queries, heads=heads, dim=dim, page=5))
    _check_marked(paged_attention(**case), case)


@pytest.mark.parametrize("count,queries_of", [
    (257, lambda r: 1), (1100, lambda r: 1), (2600, lambda r: r % 3), (300, lambda r: (7 * r) % 31),
    (1300, lambda r: 40 if r % 64 == 63 else 0)])
def test_requests_past_the_plan_s_threshold(gpu_device, count, queries_of):
    """Calls of many requests: short and long ones, ones without queries or keys."""

    queries = [queries_of(r) for r in range(count)]
    lengths = [0 if r % 53 == 17 else 1 + (29 * r) % 300 for r in range(count)]
    lengths[count // 2], lengths[count - 1] = 4097, 1500
    lengths = [max(length, n) if length else 0 for length, n in zip(lengths, queries)]
    single = all(n == 1 for n in queries)
    case = _marked(_case(gpu_device, lengths, None if single else queries, heads=(8, 2), dim=64, page=8))
    _check_marked(paged_attention(**case), case)


@pytest.mark.parametrize("queries", [None, [3, 1, 2], [200, 5, 90]])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_rows_that_are_not_seen_may_hold_anything(gpu_device, queries, dtype):
    """NaN and infinities behind a request's length, in pages of no request and in
    later tokens of a query's own chunk do not reach it."""

    lengths = [70, 31, 300] if queries != [200, 5, 90] else [270, 31, 300]
    case = _case(gpu_device, lengths, queries, heads=(4, 2), dtype=dtype, page=16)
    want = paged_attention(**case)
    used = torch.zeros(case["key_buffer"].shape[0], dtype=torch.bool, device=gpu_device)
    for request, length in enumerate(lengths):
        place = torch.arange(length, device=gpu_device)
        used[case["page_table"][request].long()[place // 16] * 16 + place % 16] = True
    for buffer in (case["key_buffer"], case["value_buffer"]):
        buffer[~used] = float("nan")
        buffer[(~used).nonzero()[::2, 0]] = float("inf")
    assert torch.equal(paged_attention(**case), want)
    if queries is None:
        return
    # The last key of each request: only its last query sees it.
    ends = case["query_starts"][1:].long() - 1
    others = torch.ones(case["query"].shape[0], dtype=torch.bool, device=gpu_device)
    others[ends] = False
    last = torch.tensor([int(case["page_table"][r, (n - 1) // 16]) * 16 + (n - 1) % 16 for r, n in enumerate(lengths)],
                        device=gpu_device)
    for bad in (float("nan"), float("inf"), -float("inf")):
        kept_k, kept_v = case["key_buffer"][last].clone(), case["value_buffer"][last].clone()
        case["value_buffer"][last] = bad
        got = paged_attention(**case)
        assert torch.equal(got[others], want[others])
        assert torch.equal(torch.nan_to_num(got[ends].float(), 1.0, 2.0, 3.0),
                           torch.nan_to_num(torch.full_like(got[ends], bad).float(), 1.0, 2.0, 3.0))
        case["value_buffer"][last] = kept_v
        case["key_buffer"][last] = bad
        assert torch.equal(paged_attention(**case)[others], want[others])
        case["key_buffer"][last] = kept_k
    assert torch.equal(paged_attention(**case), want)


def test_infinities_that_are_seen(gpu_device):
    """A seen value of infinity gives infinity in its dim, both kinds NaN."""

    case = _case(gpu_device, [50], [50], heads=(2, 1), dim=64, page=1)
    slots = case["page_table"][0, :50].long()
    case["value_buffer"][slots[10], 0, 3] = float("inf")
    case["value_buffer"][slots[20], 0, 3] = -float("inf")
    case["value_buffer"][slots[30], 0, 5] = float("nan")
    got = paged_attention(**case).float().cpu()
    assert bool(torch.isfinite(got[:10]).all())
    assert bool((got[10:20, :, 3] == math.inf).all()) and bool(torch.isnan(got[20:, :, 3]).all())
    assert bool(torch.isfinite(got[:30, :, 5]).all()) and bool(torch.isnan(got[30:, :, 5]).all())
    rest = [d for d in range(64) if d not in (3, 5)]
    assert bool(torch.isfinite(got[:, :, rest]).all())


@pytest.mark.parametrize("queries", [None, [5, 40, 2], [150, 129, 1]])
def test_pages_outside_the_pool_are_invisible(gpu_device, queries):
    report(f"bad pages, queries {queries}")
    lengths = [200, 129, 40]
    case = _case(gpu_device, lengths, queries, heads=(6, 2), dim=64, page=8)
    pool_pages = case["key_buffer"].shape[0] // 8
    case["page_table"][0, 3] = -1
    case["page_table"][0, 20] = pool_pages  # the pool's last rows are no whole page
    case["page_table"][1, 0] = -2 ** 31
    case["page_table"][2, :] = 2 ** 31 - 1  # every page
    got = paged_attention(**case)
    _check(got, case)
    assert bool((got[-1] == 0).all())


def test_rows_of_no_request_keep_their_output(gpu_device):
    case = _case(gpu_device, [40, 70], [3, 5], heads=(4, 2), dim=64)
    query = torch.cat((case["query"], case["query"][:4]))
    output = torch.full_like(query, 7.0)
    got = paged_attention(**{**case, "query": query}, output=output)
    assert got is output and bool((output[8:] == 7).all())
    assert torch.equal(output[:8], paged_attention(**case))
    # A request that begins later: the rows before it.
    starts = case["query_starts"] + 2
    output = torch.full_like(query, 7.0)
    paged_attention(**{**case, "query": query, "query_starts": starts}, output=output)
    assert bool((output[:2] == 7).all()) and bool((output[10:] == 7).all()) and bool((output[2:10] != 7).any(-1).all())


def test_lengths_and_starts_outside_the_call_are_held_to_it(gpu_device):
    """Longer than the table row, negative, starts past the queries: no access outside."""

    case = _case(gpu_device, [64, 64, 64], [4, 4, 4], heads=(4, 2), dim=64, page=16, spare_columns=0)
    want = paged_attention(**case)
    case["kv_lengths"].copy_(torch.tensor([2 ** 31 - 1, 64, -5]))
    got = paged_attention(**case)
    assert torch.equal(got[:8], want[:8]) and bool((got[8:] == 0).all())
    case["kv_lengths"].fill_(64)
    case["query_starts"].copy_(torch.tensor([-3, 4, 8, 2 ** 31 - 1]))
    assert torch.equal(paged_attention(**case), want)


@pytest.mark.parametrize("layout", ["fused", "by head", "odd"])
@pytest.mark.parametrize("queries", [None, [60, 2]])
def test_query_layouts(gpu_device, layout, queries):
    case = _case(gpu_device, [300, 77], queries, heads=(4, 2), dim=128)
    want = paged_attention(**case)
    query = case["query"]
    rows = query.shape[0]
    if layout == "fused":
        wide = torch.zeros(rows, 8 * 128, dtype=query.dtype, device=gpu_device)
        view = wide[:, 2 * 128:6 * 128].unflatten(-1, (4, 128))
    elif layout == "by head":
        view = torch.zeros(4, rows, 128, dtype=query.dtype, device=gpu_device).transpose(0, 1)
    else:  # at an address that is no multiple of 16 bytes
        view = torch.zeros(rows * 4 * 128 + 1, dtype=query.dtype, device=gpu_device)[1:].view(rows, 4, 128)
    view.copy_(query)
    assert torch.equal(paged_attention(**{**case, "query": view}), want)


def test_table_rows_with_a_stride(gpu_device):
    case = _case(gpu_device, [300, 77, 20], heads=(4, 2), dim=64, page=8)
    want = paged_attention(**case)
    wide = torch.full((6, 100), -9, dtype=torch.int32, device=gpu_device)
    view = wide[::2, 5:5 + case["page_table"].shape[1]]
    view.copy_(case["page_table"])
    assert torch.equal(paged_attention(**{**case, "page_table": view}), want)


@pytest.mark.parametrize("scale", [1e-3, 1.0, 30.0])
@pytest.mark.parametrize("queries", [None, [70, 1]])
def test_scales(gpu_device, scale, queries):
    """Weights from nearly uniform to nearly one-hot (scores of hundreds)."""

    case = _case(gpu_device, [900, 64], queries, heads=(4, 2), dim=64, dtype=torch.bfloat16)
    if scale == 30.0:
        case["query"].div_(8)  # a score's error, exp(dim 2^-24 |score|), stays small
    _check(paged_attention(**case, scale=scale), case, scale=scale)


def test_rising_scores(gpu_device):
    """Keys whose scores rise along the request by far more than the maximum's slack."""

    case = _case(gpu_device, [2000], [3], heads=(4, 1), dim=64, page=1)
    slots = case["page_table"][0, :2000].long()
    direction = torch.ones(64, device=gpu_device)
    case["query"].copy_(direction.expand_as(case["query"]))
    ramp = torch.linspace(-8, 8, 2000, device=gpu_device)[:, None] * direction
    case["key_buffer"][slots, 0] = ramp.to(torch.bfloat16)
    _check(paged_attention(**case), case)
    case["key_buffer"][slots, 0] = ramp.flip(0).to(torch.bfloat16)
    _check(paged_attention(**case), case)


def test_nothing_to_do(gpu_device):
    case = _case(gpu_device, [], heads=(4, 2), dim=64)
    assert paged_attention(**case).shape == (0, 4, 64)
    case = _case(gpu_device, [10, 20], [0, 0], heads=(4, 2), dim=64)
    assert paged_attention(**case).shape == (0, 4, 64)
    # A pool without rows, and without a whole page: every key is invisible.
    for slots in (0, 15):
        case = _case(gpu_device, [10, 20], heads=(4, 2), dim=64)
        case["key_buffer"] = case["key_buffer"][:slots].clone()
        case["value_buffer"] = case["value_buffer"][:slots].clone()
        assert bool((paged_attention(**case) == 0).all())
    case = _case(gpu_device, [0, 0], heads=(4, 2), dim=64)
    case["page_table"] = case["page_table"][:, :0]
    assert bool((paged_attention(**case) == 0).all())


def test_pool_past_four_gib(gpu_device):
    """Rows past 2^32 bytes, and a table of the pool's last pages."""

    slots = (1 << 32) // (2 * 128 * 2) + 4096
    keys = torch.zeros(slots, 2, 128, dtype=torch.bfloat16, device=gpu_device)
    values = torch.zeros_like(keys)
    generator = torch.Generator(device=gpu_device).manual_seed(3)
    for buffer in (keys, values):
        buffer[-4096:] = torch.randn(4096, 2, 128, device=gpu_device, generator=generator).to(torch.bfloat16)
        buffer[:4096] = torch.randn(4096, 2, 128, device=gpu_device, generator=generator).to(torch.bfloat16)
    pages = slots // 16
    table = torch.stack((torch.arange(pages - 20, pages, device=gpu_device), torch.arange(20, device=gpu_device)))
    case = dict(key_buffer=keys, value_buffer=values, page_table=table.to(torch.int32), page_size=16,
                kv_lengths=torch.tensor([317, 320], device=gpu_device), query_starts=None)
    near = dict(case, key_buffer=torch.cat((keys[-4096:], keys[:4096])),
                value_buffer=torch.cat((values[-4096:], values[:4096])),
                page_table=torch.stack((table[0] - (pages - 256), table[1] + 256)).to(torch.int32))
    for starts in (None, torch.tensor([0, 100, 230], device=gpu_device)):
        rows = 2 if starts is None else 230
        query = torch.randn(rows, 4, 128, device=gpu_device, generator=generator).to(torch.bfloat16)
        got = paged_attention(**{**case, "query": query, "query_starts": starts})
        assert torch.equal(got, paged_attention(**{**near, "query": query, "query_starts": starts}))
        assert bool(got.any())


@pytest.mark.parametrize("queries", [None, [6, 1, 9], [190, 64, 1]])
def test_a_captured_call_serves_other_lengths(gpu_device, queries):
    """One graph, replayed with other lengths, pages and starts, against eager calls."""

    most = [700, 300, 512]
    case = _case(gpu_device, most, queries, heads=(28, 4), dim=128, page=16)
    paged_attention(**case)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = paged_attention(**case)
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
        again = paged_attention(**case)
        torch.cuda.synchronize()
        assert torch.equal(got, again)
        _check(got, case)


def test_a_captured_call_of_many_requests_serves_other_lengths(gpu_device):
    """The sums over 200 requests are the replay's own, not the capture's."""

    count = 200
    case = _case(gpu_device, [600] * count, heads=(8, 2), dim=64, page=16)
    paged_attention(**case)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = paged_attention(**case)
    for step in range(3):
        case["kv_lengths"].copy_(torch.tensor([(97 * r * (step + 1)) % 601 for r in range(count)]))
        captured.fill_(9)
        graph.replay()
        torch.cuda.synchronize()
        got = captured.clone()
        assert torch.equal(got, paged_attention(**case))
        _check(got, case)


def test_two_streams_at_once(gpu_device):
    """Calls in flight on two streams have workspaces of their own."""

    cases = [_case(gpu_device, [6000 + 100 * i], heads=(28, 4), seed=i) for i in range(2)]
    want = [paged_attention(**case) for case in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[], []]
    for _ in range(20):
        for i, (stream, case) in enumerate(zip(streams, cases)):
            with torch.cuda.stream(stream):
                got[i].append(paged_attention(**case))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(out, want[i]) for out in got[i])


def test_repeated_calls_are_equal_bit_for_bit(gpu_device):
    case = _case(gpu_device, [9000, 50, 3000], [40, 2, 100], heads=(28, 4))
    want = paged_attention(**case)
    for _ in range(5):
        assert torch.equal(paged_attention(**case), want)
