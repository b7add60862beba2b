"""GPU tests of the 8-bit pool's writes and reads: codes and scales bit for bit
against the format's model in 64 bits."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from legolink_amd.quantized_pool import append_quantized_kv_inplace, link_quantized_kv_inplace, load_quantized_kv
from legolink_amd.rope import build_cos_sin_cache
from tests import quantized_pool_math as qm
from tests.gpu_helpers import report
from tests.head_rotary_math import allowed, turned

pytestmark = pytest.mark.gpu
POSITIONS = 512


def _pool(device, slots, heads, dim, block, *, seed=1, **options):
    return {**qm.random_pool(slots, heads, dim, block, seed=seed, device=device, **options), "scale_block": block}


def _state(pool):
    return [qm.host(pool[name]) for name in ("key_buffer", "key_scales", "value_buffer", "value_scales")]


def _check_pool(pool, before, block, slots, key_rows, value_rows, written):
    """The pool holds what the model stores into ``before``."""

    got = _state(pool)
    for half, rows in ((0, key_rows), (2, value_rows)):
        codes, scales = qm.stored(before[half], before[half + 1], block, slots, rows, written)
        name = "values" if half else "keys"
        assert np.array_equal(got[half + 1], scales), f"scales of the {name}"
        assert qm.same_codes(got[half], codes), f"codes of the {name}: {(got[half] != codes).sum()} differ"


def _append_case(device, slots_list, *, q_heads=4, kv_heads=2, dim=128, rotary=None, dtype=torch.bfloat16, block=16,
                 slots=256, table=torch.float32, weights=None, index=torch.int64, layout="fused", seed=1, **options):
    generator = torch.Generator().manual_seed(seed)
    tokens, rotary = len(slots_list), dim if rotary is None else rotary
    widths = [q_heads * dim, kv_heads * dim, kv_heads * dim]

    def normal(*shape):
        return (torch.randn(*shape, generator=generator) * 2).to(dtype).to(device)

    if layout == "by head":
        rows = [normal(h, tokens, dim).transpose(0, 1) for h in (q_heads, kv_heads, kv_heads)]
    else:
        odd = 1 if layout == "odd" else 0
        projected = normal(tokens, sum(widths) + odd)[:, odd:]
        rows = [part.unflatten(-1, (-1, dim)) for part in projected.split(widths, dim=-1)]
    norms = [None, None]
    if weights is not None:
        norms = [(1 + 0.4 * torch.randn(dim, generator=generator)).to(weights).to(device) for _ in range(2)]
    return dict(**_pool(device, slots, kv_heads, dim, block, seed=seed, **options), query=rows[0], key=rows[1],
                value=rows[2], destination_slots=torch.tensor(slots_list, device=device).to(index), rotary_dim=rotary,
                positions=torch.randint(POSITIONS, (tokens,), generator=generator).to(index).to(device),
                cos_sin_cache=build_cos_sin_cache(POSITIONS, rotary, dtype=table).to(device),
                query_norm_weight=norms[0], key_norm_weight=norms[1])


def _rows_of(case, neox, name):
    """The rows that an append writes, in 64 bits."""

    rows = case[name].cpu().double()
    if name == "key":
        rows, _ = turned(rows, torch.where(case["positions"].cpu() < 0, 0, case["positions"].cpu()).clamp(max=POSITIONS - 1),
                         case["cos_sin_cache"], rotary=case["rotary_dim"], neox=neox, weight=case["key_norm_weight"])
    return rows.numpy()


def _check_append(case, neox=True, **options):
    before = _state(case)
    query = case["query"].clone()
    got = append_quantized_kv_inplace(**case, is_neox_style=neox, **options)
    slots = case["destination_slots"].tolist()
    position = case["positions"].tolist()
    there = [0 <= p < POSITIONS for p in position]
    written = [ok and 0 <= s < case["key_buffer"].shape[0] for ok, s in zip(there, slots)]
    _check_pool(case, before, case["scale_block"], slots, _rows_of(case, neox, "key"), _rows_of(case, neox, "value"),
                written)
    want, size = turned(query, case["positions"].clamp(0, POSITIONS - 1), case["cos_sin_cache"], rotary=case["rotary_dim"],
                        neox=neox, weight=case["query_norm_weight"])
    off = (got.cpu().double() - want).abs()[there]
    assert bool((off <= allowed(want, size, got.dtype, query.shape[-1])[there]).all())
    return got


RUNS = {  # slots of a pool of 256
    "one": [37],
    "a row in each of some blocks": [5, 21, 47, 100, 240],
    "from the middle of a block on": list(range(90, 150)),
    "whole blocks": [*range(128, 192), *range(0, 64)],
    "rows of a block in any order": [3, 0, 7, 14, 9, 40, 33, 63, 130, 128, 129],
    "padded": [-1, -1, 200, 201, -1, 8, 9, -1, -5],
}


@pytest.mark.parametrize("runs", list(RUNS))
@pytest.mark.parametrize("dim,rotary,block", [(128, 128, 16), (64, 32, 16), (256, 256, 16), (128, 64, 64), (64, 64, 32),
                                              (256, 32, 128), (80, 48, 16), (112, 16, 8), (16, 16, 1), (240, 240, 64)])
@pytest.mark.parametrize("neox,dtype,weights", [(True, torch.bfloat16, None), (False, torch.float16, torch.float32),
                                                (True, torch.float16, torch.bfloat16)])
def test_append(gpu_device, runs, dim, rotary, block, neox, dtype, weights):
    report(f"append {runs}, dim {dim} rotary {rotary} block {block} neox {neox} {dtype} weights {weights}")
    case = _append_case(gpu_device, RUNS[runs], dim=dim, rotary=rotary, block=block, dtype=dtype, weights=weights,
                        q_heads=7, kv_heads=3)
    _check_append(case, neox)


@pytest.mark.parametrize("layout", ["fused", "by head", "odd"])
@pytest.mark.parametrize("table,index", [(torch.float32, torch.int32), (torch.bfloat16, torch.int64),
                                         (torch.float16, torch.int32)])
def test_append_layouts_and_tables(gpu_device, layout, table, index):
    report(f"append {layout} {table} {index}")
    case = _append_case(gpu_device, RUNS["from the middle of a block on"], layout=layout, table=table, index=index,
                        weights=torch.float16, q_heads=28, kv_heads=4)
    _check_append(case)


@pytest.mark.parametrize("stride,offset", [(67, 0), (64, 1), (80, 3)])
def test_append_tables_off_alignment(gpu_device, stride, offset):
    case = _append_case(gpu_device, [3, 4, 5, 20], dim=64, table=torch.bfloat16)
    wide = torch.zeros(POSITIONS * stride + offset, dtype=torch.bfloat16, device=gpu_device)
    table = wide.as_strided((POSITIONS, 64), (stride, 1), offset)
    table.copy_(case["cos_sin_cache"])
    _check_append({**case, "cos_sin_cache": table})


@pytest.mark.parametrize("tokens", [1, 2, 16, 700, 5000])
@pytest.mark.parametrize("kv_heads,block", [(1, 16), (5, 64), (8, 16)])
def test_append_many_tokens(gpu_device, tokens, kv_heads, block):
    """Chunks, and batches of single tokens of which each has a block: every count of
    tokens that a workgroup looks through."""

    report(f"append {tokens} tokens, {kv_heads} KV heads, block {block}")
    generator = torch.Generator().manual_seed(tokens)
    total = (tokens + 2 * block) // block * block + block
    chunk = [total - 1 - i for i in range(tokens)]  # from the end down
    case = _append_case(gpu_device, chunk, q_heads=kv_heads, kv_heads=kv_heads, dim=64, block=block, slots=total)
    _check_append(case)
    blocks = torch.randperm(tokens, generator=generator)
    single = (blocks * block + torch.randint(block, (tokens,), generator=generator)).tolist()
    case = _append_case(gpu_device, single, q_heads=kv_heads, kv_heads=kv_heads, dim=64, block=block,
                        slots=tokens * block)
    _check_append(case)


def test_append_grows_a_scale_and_never_lowers_it(gpu_device):
    """A block filled token by token: each size of the new rows against each scale."""

    for low, high in ((100, 101), (123, 124), (140, 141), (0, 1), (254, 255)):
        case = _append_case(gpu_device, [7], slots=32, low=low, high=high)
        for slot in (7, 0, 15, 8):
            case["destination_slots"].fill_(slot)
            case["value"].mul_(4)
            _check_append(case)
    # An empty pool's block: the scale is the rows', and a clearing makes it so again.
    case = _append_case(gpu_device, [2, 1], slots=32, empty=(0, 1))
    _check_append(case)
    case["value_scales"].view(torch.uint8)[0] = 0
    case["value"].mul_(2.0 ** -20)
    _check_append(case)
    assert int(case["value_scales"].view(torch.uint8)[0].max()) < 127 - 20


def test_append_values_of_any_size(gpu_device):
    """The largest and smallest numbers of the types, zeros, infinities and NaN."""

    for dtype in (torch.bfloat16, torch.float16):
        info = torch.finfo(dtype)
        for size in (info.max, info.smallest_normal, info.smallest_normal * info.eps, 0.0, 448.0, 449.0, 464.0, 480.0):
            case = _append_case(gpu_device, list(range(16, 32)), dtype=dtype, empty=range(16))
            case["value"].copy_((torch.randn(16, 2, 128).clamp(-1, 1) * size).to(dtype))
            case["value"][3, 1, 5] = -size
            case["key"].zero_()
            _check_append(case)
        case = _append_case(gpu_device, list(range(20, 26)), dtype=dtype)
        for row, bad in enumerate((float("inf"), -float("inf"), float("nan"))):
            case["value"][row, 0, 7 * row] = bad
        case["value"][4] = float("nan")
        _check_append(case)
        keys, values = load_quantized_kv(**{n: case[n] for n in ("key_buffer", "value_buffer", "key_scales", "value_scales",
                                                                 "scale_block")}, dtype=torch.float32)
        assert int(torch.isnan(values[20:26]).sum()) == 3 + 2 * 128 and bool(torch.isfinite(keys).all())


def test_append_to_a_block_whose_scale_is_nan(gpu_device):
    """It stays NaN while its rows are added to, and is new where all are written."""

    case = _append_case(gpu_device, [17, *range(32, 48)])
    for name in ("key_scales", "value_scales"):
        case[name].view(torch.uint8)[1:3] = 255
    append_quantized_kv_inplace(**case)
    for name in ("key_scales", "value_scales"):
        scales = case[name].view(torch.uint8).cpu()
        assert bool((scales[1] == 255).all()) and bool((scales[2] < 255).all())


@pytest.mark.parametrize("left_out", ["query_norm_weight", "key_norm_weight"])
@pytest.mark.parametrize("neox,rotary", [(True, 64), (False, 128)])
def test_append_with_one_norm(gpu_device, left_out, neox, rotary):
    case = _append_case(gpu_device, list(range(30, 60)), rotary=rotary, weights=torch.float32)
    _check_append({**case, left_out: None}, neox)


def test_append_nothing(gpu_device):
    case = _append_case(gpu_device, [3], slots=32)
    before = _state(case)
    empty = {name: case[name][:0] for name in ("query", "key", "value", "positions", "destination_slots")}
    assert append_quantized_kv_inplace(**{**case, **empty}).shape == (0, 4, 128)
    assert all(np.array_equal(a, b) for a, b in zip(_state(case), before))


def test_runs_that_windows_cut(gpu_device):
    """Runs of every length from 1 to 17 one after another, padding between some: windows
    of all widths begin and end inside them."""

    for block, tokens in ((16, 2500), (64, 2500), (128, 1500), (8, 400)):
        slots, length, at = [], 1, 0
        while len(slots) < tokens:
            begin = at * block + (length % 3 if block > length + 3 else 0)
            slots += list(range(begin, begin + min(length, block)))
            slots += [-1] * (length % 2)
            length, at = length % 17 + 1, at + 1
        report(f"runs of 1 to 17, block {block}, {len(slots)} tokens")
        case = _append_case(gpu_device, slots, q_heads=2, kv_heads=2, dim=64, block=block, slots=(at + 1) * block)
        _check_append(case)


def test_append_leaves_out_and_counts(gpu_device):
    slots = [3, 4, 5, 300, 301, -1, 20, 21, 22, 256]
    case = _append_case(gpu_device, slots, q_heads=28)
    case["positions"][1], case["positions"][6], case["positions"][5] = POSITIONS, -1, -7
    skipped = torch.full((1,), 5, dtype=torch.int64, device=gpu_device)
    output = torch.full((10, 28, 128), 9.0, dtype=torch.bfloat16, device=gpu_device)
    got = _check_append(case, skipped_rows=skipped, query_output=output)
    assert got is output and bool((output[[1, 5, 6]] == 9).all())
    assert int(skipped) == 5 + 6  # three positions, three slots past the pool


def test_append_in_place_queries(gpu_device):
    case = _append_case(gpu_device, [3, 4, 90])
    want = append_quantized_kv_inplace(**case)
    other = _append_case(gpu_device, [3, 4, 90])
    got = append_quantized_kv_inplace(**other, query_output=other["query"])
    assert got is other["query"] and torch.equal(got, want)
    assert torch.equal(other["key"], case["key"]) and torch.equal(other["value"], case["value"])


# -- link --------------------------------------------------------------------


def _link_case(device, sources, destinations, *, kv_heads=2, dim=128, rotary=None, block=16, slots=512,
               table=torch.float32, index=torch.int64, seed=1, repair=False, **options):
    generator = torch.Generator().manual_seed(seed)
    rotary, tokens = dim if rotary is None else rotary, len(sources)

    def positions():
        return torch.randint(POSITIONS, (tokens,), generator=generator).to(index).to(device)

    mask = (torch.rand(tokens, generator=generator) < 0.3).to(device) if repair else None
    return dict(**_pool(device, slots, kv_heads, dim, block, seed=seed, **options), rotary_dim=rotary,
                source_slots=torch.tensor(sources, device=device).to(index),
                destination_slots=torch.tensor(destinations, device=device).to(index), local_positions=positions(),
                global_positions=positions(), cos_sin_cache=build_cos_sin_cache(POSITIONS, rotary, dtype=table).to(device),
                repair_mask=mask)


def _check_link(case, neox=True, prefix=0, **options):
    before = _state(case)
    link_quantized_kv_inplace(**case, is_neox_style=neox, prefix_token_count=prefix, **options)
    block, slots, pool_slots = case["scale_block"], case["destination_slots"].tolist(), case["key_buffer"].shape[0]
    source, old, new = (case[name].cpu().numpy() for name in ("source_slots", "local_positions", "global_positions"))
    turns = np.arange(len(slots)) >= prefix
    in_table = (old >= 0) & (old < POSITIONS) & (new >= 0) & (new < POSITIONS)
    written = (source >= 0) & (source < pool_slots) & (in_table | ~turns)
    written &= (np.array(slots) >= 0) & (np.array(slots) < pool_slots)
    if case["repair_mask"] is not None:
        written &= ~case["repair_mask"].cpu().numpy().astype(bool)
    safe = np.clip(source, 0, pool_slots - 1)
    keys, values = (qm.values_of(before[i], before[i + 1], block)[safe] for i in (0, 2))
    table = case["cos_sin_cache"].cpu().double().numpy()
    half = case["rotary_dim"] // 2
    c, s = (table[np.clip(old, 0, POSITIONS - 1)][:, None, i * half:(i + 1) * half] for i in (0, 1))
    cn, sn = (table[np.clip(new, 0, POSITIONS - 1)][:, None, i * half:(i + 1) * half] for i in (0, 1))
    moved = qm.turned_rows(keys, cn * c + sn * s, sn * c - cn * s, neox)
    _check_pool(case, before, block, slots, np.where(turns[:, None, None], moved, keys), values, written)
    return written


@pytest.mark.parametrize("dim,rotary,block", [(128, 128, 16), (64, 32, 16), (256, 256, 16), (128, 64, 64), (64, 64, 32),
                                              (256, 32, 128), (80, 48, 16), (112, 16, 8), (16, 16, 1), (240, 240, 64)])
@pytest.mark.parametrize("neox,repair,prefix", [(True, False, 0), (False, True, 7), (True, True, 60)])
def test_link(gpu_device, dim, rotary, block, neox, repair, prefix):
    report(f"link dim {dim} rotary {rotary} block {block} neox {neox} repair {repair} prefix {prefix}")
    # Runs of cached rows, some twice, to whole and partial blocks.
    sources = [*range(3, 40), *range(100, 101), *range(7, 90)]
    destinations = [*range(256, 256 + len(sources) - 20), *range(400, 420)]
    case = _link_case(gpu_device, sources, destinations, dim=dim, rotary=rotary, block=block, repair=repair, kv_heads=3)
    _check_link(case, neox, prefix)


@pytest.mark.parametrize("table,index", [(torch.float32, torch.int32), (torch.bfloat16, torch.int64),
                                         (torch.float16, torch.int32)])
def test_link_tables_and_empty_blocks(gpu_device, table, index):
    case = _link_case(gpu_device, list(range(5, 55)), list(range(300, 350)), table=table, index=index,
                      empty=range(18, 22), repair=True)
    case["repair_mask"] = case["repair_mask"].to(torch.uint8)
    _check_link(case)


@pytest.mark.parametrize("tokens", [1, 33, 6000])
def test_link_many_tokens(gpu_device, tokens):
    report(f"link {tokens} tokens")
    generator = torch.Generator().manual_seed(tokens)
    sources = torch.randint(4096, (tokens,), generator=generator).tolist()
    blocks = torch.randperm(400, generator=generator)
    place = torch.arange(tokens)
    destinations = (4096 + blocks[place // 16] * 16 + place % 16).tolist()
    _check_link(_link_case(gpu_device, sources, destinations, slots=4096 + 400 * 16, dim=64, empty=range(256, 656)))


def test_link_leaves_out_and_counts(gpu_device):
    sources = [0, 1, -1, 512, 4, 5, 6, 7, 8, 9]
    destinations = [300, 301, 302, 303, 304, 512, -3, 306, 307, 305]
    case = _link_case(gpu_device, sources, destinations)
    case["local_positions"][1], case["global_positions"][4], case["local_positions"][7] = POSITIONS, -1, -1
    case["repair_mask"] = torch.tensor([0, 0, 0, 0, 0, 0, 0, 1, 0, 0], dtype=torch.bool, device=gpu_device)
    skipped = torch.zeros(1, dtype=torch.int64, device=gpu_device)
    written = _check_link(case, skipped_rows=skipped)
    assert int(skipped) == 5 and written.sum() == 3  # two sources, two positions, a slot past the pool
    # Below the prefix no position is read.
    case = _link_case(gpu_device, [0, 1], [300, 301])
    case["local_positions"].fill_(-1)
    assert _check_link(case, prefix=2).all()


def test_link_moves_nan(gpu_device):
    case = _link_case(gpu_device, [0, 17, 34], [300, 301, 302])
    case["key_scales"].view(torch.uint8)[1] = 255
    case["value_buffer"].view(torch.uint8)[34, 1, 3] = 0x7F
    _check_link(case)


# -- load --------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("heads,dim,block", [(4, 128, 16), (1, 64, 128), (2, 256, 64), (3, 80, 8), (5, 16, 1)])
@pytest.mark.parametrize("index", [None, torch.int32, torch.int64])
def test_load(gpu_device, dtype, heads, dim, block, index):
    report(f"load {dtype} heads {heads} dim {dim} block {block} slots {index}")
    pool = _pool(gpu_device, 384, heads, dim, block, low=0, high=256)
    slots = None
    if index is not None:
        slots = torch.randint(-3, 400, (301,), generator=torch.Generator().manual_seed(4)).to(index).to(gpu_device)
    got = load_quantized_kv(**pool, slots=slots, dtype=dtype)
    for name, rows in zip(("key", "value"), got):
        want = qm.pool_values(pool[f"{name}_buffer"], pool[f"{name}_scales"], block).float()  # exact (or an overflow)
        if slots is not None:
            at = slots.cpu().long()
            there = (at >= 0) & (at < 384)
            want = torch.where(there[:, None, None], want[torch.where(there, at, 0)], 0.0)
        assert rows.is_contiguous() and rows.dtype == dtype
        assert torch.equal(torch.nan_to_num(rows.cpu().float(), 1.5, 2e38, -2e38),
                           torch.nan_to_num(want.to(dtype).float(), 1.5, 2e38, -2e38))
        assert torch.equal(torch.isnan(rows.cpu()), torch.isnan(want))


def test_load_into_given_rows(gpu_device):
    pool = _pool(gpu_device, 64, 2, 64, 16)
    slots = torch.tensor([5, 63, 0], device=gpu_device)
    want = load_quantized_kv(**pool, slots=slots)
    outputs = [torch.full((3, 2, 64), 7.0, dtype=torch.bfloat16, device=gpu_device) for _ in range(2)]
    got = load_quantized_kv(**pool, slots=slots, key_output=outputs[0], value_output=outputs[1])
    assert got[0] is outputs[0] and got[1] is outputs[1]
    assert torch.equal(outputs[0], want[0]) and torch.equal(outputs[1], want[1])
    assert load_quantized_kv(**pool, slots=slots[:0])[0].shape == (0, 2, 64)


def test_pool_past_four_gib(gpu_device):
    """Codes past 2^32 bytes: appended, linked and loaded."""

    slots = (1 << 32) // 128 + 4096
    pool = {name: torch.zeros(slots, 1, 128, dtype=torch.uint8, device=gpu_device).view(torch.float8_e4m3fn)
            for name in ("key_buffer", "value_buffer")}
    for name in ("key_scales", "value_scales"):
        pool[name] = torch.zeros(slots // 16, 1, dtype=torch.uint8, device=gpu_device).view(torch.float8_e8m0fnu)
    far, near = list(range(slots - 40, slots - 20)), list(range(8, 28))
    kept = None
    for rows in (near, far):
        case = _append_case(gpu_device, rows, kv_heads=1, slots=16)
        case.update(pool, scale_block=16)
        append_quantized_kv_inplace(**case)
        got = load_quantized_kv(**pool, scale_block=16, slots=case["destination_slots"])
        assert kept is None or all(torch.equal(a, b) for a, b in zip(got, kept))
        kept = got
    index = torch.tensor(far, device=gpu_device)
    positions = torch.arange(20, device=gpu_device)
    link_quantized_kv_inplace(**pool, scale_block=16, source_slots=index, destination_slots=index - 640,
                              local_positions=positions, global_positions=positions, prefix_token_count=20,
                              cos_sin_cache=build_cos_sin_cache(POSITIONS, 128).to(gpu_device), rotary_dim=128)
    got = load_quantized_kv(**pool, scale_block=16, slots=index - 640)
    assert all(torch.equal(a, b) for a, b in zip(got, kept))


def test_captured_calls_replay_with_other_inputs(gpu_device):
    """Append, link and load in one graph, replayed over changing inputs, against eager calls."""

    case = _append_case(gpu_device, list(range(16, 40)), slots=512)
    twin = {name: value.clone() if name.endswith(("_buffer", "_scales")) else value for name, value in case.items()}
    positions = torch.arange(24, device=gpu_device)

    def step(arguments):
        query = append_quantized_kv_inplace(**arguments)
        pool = {name: arguments[name] for name in ("key_buffer", "value_buffer", "key_scales", "value_scales",
                                                   "scale_block")}
        link_quantized_kv_inplace(**pool, source_slots=arguments["destination_slots"],
                                  destination_slots=arguments["destination_slots"] + 256, local_positions=positions,
                                  global_positions=positions + 100, cos_sin_cache=arguments["cos_sin_cache"],
                                  rotary_dim=128)
        return (query, *load_quantized_kv(**pool))

    step(case)
    step(twin)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(case)
    generator = torch.Generator(device=gpu_device).manual_seed(9)
    for turn in range(3):
        case["key"].copy_(torch.randn(case["key"].shape, device=gpu_device, generator=generator) * 3 ** turn)
        case["value"].copy_(torch.randn(case["value"].shape, device=gpu_device, generator=generator) * 5 ** turn)
        case["destination_slots"].add_(11)
        graph.replay()
        torch.cuda.synchronize()
        want = step(twin)
        torch.cuda.synchronize()
        for a, b in zip(captured, want):
            assert torch.equal(a, b)
        for name in ("key_buffer", "value_buffer", "key_scales", "value_scales"):
            assert torch.equal(case[name].view(torch.uint8), twin[name].view(torch.uint8))


def test_calls_on_another_stream(gpu_device):
    case = _append_case(gpu_device, RUNS["from the middle of a block on"])
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    before = _state(case)
    with torch.cuda.stream(stream):
        append_quantized_kv_inplace(**case)
    stream.synchronize()
    slots = case["destination_slots"].tolist()
    _check_pool(case, before, 16, slots, _rows_of(case, True, "key"), _rows_of(case, True, "value"), [True] * len(slots))


# -- padding within a block's rows ---------------------------------------------

PADDED = {  # slots of a pool of 512; 512 and more are past it
    "one": [0, -1, 1],
    "past the pool": [0, 512, 1, 7, 2 ** 31 - 1, 3],
    "two blocks": [133, -1, -9, 130, 600, 128, -1, 300, -1, 257],
    "every second": [s for pair in zip(range(256, 384), [-1, 512] * 64) for s in pair],
    "a few": [s for i in range(140) for s in ([-1] * (i % 23 == 5) + [140 + i])],
    "long": [40, *[-1] * 700, 41, *[-5] * 1500, 47, *[-1] * 64, 200, *[512] * 3000, 207, 204],
    "in front": [*[-1] * 1200, 384, *[-1] * 600, 385, 386],
    "behind": [17, 18, 19, *[-1] * 2045],
    "alone": [-1] * 1000 + [511] + [-1] * 200,
    "nothing": [-1, 512] * 300,
}


@pytest.mark.parametrize("runs", list(PADDED))
@pytest.mark.parametrize("dim,block", [(128, 16), (64, 64), (128, 32), (256, 128), (64, 128), (16, 128), (80, 8)])
def test_append_with_padding_within_a_block(gpu_device, runs, dim, block):
    """A block's scale and codes are of all its rows in the call, whatever padding of
    whatever length stands between them."""

    report(f"append padded {runs}, dim {dim} block {block}")
    slots = PADDED[runs]
    case = _append_case(gpu_device, slots, dim=dim, block=block, slots=512, kv_heads=2, q_heads=2, rotary=16)
    case["key"].mul_(torch.linspace(0.1, 30.0, len(slots), device=gpu_device).to(case["key"].dtype)[:, None, None])
    case["value"].mul_(torch.linspace(20.0, 0.1, len(slots), device=gpu_device).to(case["key"].dtype)[:, None, None])
    skipped = torch.zeros(1, dtype=torch.int64, device=gpu_device)
    _check_append(case, skipped_rows=skipped)
    assert int(skipped) == sum(s >= 512 for s in slots)


@pytest.mark.parametrize("runs", list(PADDED))
@pytest.mark.parametrize("dim,block", [(128, 16), (128, 64), (64, 128), (256, 32), (256, 128)])
def test_link_with_padding_within_a_block(gpu_device, runs, dim, block):
    report(f"link padded {runs}, dim {dim} block {block}")
    slots = PADDED[runs]
    sources = [1024 + (5 * i) % 512 for i in range(len(slots))]
    case = _link_case(gpu_device, sources, [s if s < 512 else 1536 + s for s in slots], dim=dim, block=block, slots=1536,
                      rotary=32, repair=True, index=torch.int64)
    skipped = torch.zeros(1, dtype=torch.int64, device=gpu_device)
    _check_link(case, skipped_rows=skipped)
    masked = case["repair_mask"].tolist()
    assert int(skipped) == sum(s >= 512 and not m for s, m in zip(slots, masked))


@pytest.mark.parametrize("block", [16, 32, 64, 128])
@pytest.mark.parametrize("tokens", [40, 700, 5000])
def test_padding_anywhere_in_a_large_append(gpu_device, block, tokens):
    """Windows of every width: rows of many blocks in any order within each, and padding
    of any length between any two of them."""

    report(f"padding anywhere, {tokens} tokens, block {block}")
    generator = torch.Generator().manual_seed(tokens + block)

    def draw(high):
        return int(torch.randint(high, (1,), generator=generator))

    slots, blocks = [], iter(torch.randperm(tokens, generator=generator).tolist())
    while len(slots) < tokens:
        base = next(blocks) * block
        for offset in torch.randperm(block, generator=generator)[:1 + draw(block)].tolist():
            if draw(9) == 0:
                slots += [-1] * (1 + draw(3) * draw(3) * draw(90))
            slots.append(base + offset)
    case = _append_case(gpu_device, slots, q_heads=2, kv_heads=3, dim=64, block=block, slots=tokens * block)
    _check_append(case)


# -- every kernel that the dispatch by dim and block sends calls to ------------------

VARIANTS = [(128, 128, 32), (128, 64, 128), (256, 128, 32), (256, 256, 8), (64, 64, 64), (64, 32, 128), (144, 16, 16)]


@pytest.mark.parametrize("runs", list(RUNS))
@pytest.mark.parametrize("dim,rotary,block", VARIANTS)
def test_append_other_blocks(gpu_device, runs, dim, rotary, block):
    report(f"append {runs}, dim {dim} rotary {rotary} block {block}")
    for neox, dtype, weights in ((True, torch.bfloat16, None), (False, torch.float16, torch.float32)):
        case = _append_case(gpu_device, RUNS[runs], dim=dim, rotary=rotary, block=block, dtype=dtype, weights=weights,
                            q_heads=7, kv_heads=3)
        _check_append(case, neox)


@pytest.mark.parametrize("dim,rotary,block", VARIANTS)
@pytest.mark.parametrize("neox,repair,prefix", [(True, False, 0), (False, True, 7), (True, True, 60)])
def test_link_other_blocks(gpu_device, dim, rotary, block, neox, repair, prefix):
    report(f"link dim {dim} rotary {rotary} block {block} neox {neox} repair {repair} prefix {prefix}")
    sources = [*range(3, 40), *range(100, 101), *range(7, 90)]
    destinations = [*range(256, 256 + len(sources) - 20), *range(400, 420)]
    case = _link_case(gpu_device, sources, destinations, dim=dim, rotary=rotary, block=block, repair=repair, kv_heads=3)
    _check_link(case, neox, prefix)


@pytest.mark.parametrize("dim", [128, 256])
@pytest.mark.parametrize("block,tokens", [(8, 400), (32, 1500), (128, 1500)])
def test_runs_that_windows_cut_of_other_dims(gpu_device, dim, block, tokens):
    slots, length, at = [], 1, 0
    while len(slots) < tokens:
        begin = at * block + (length % 3 if block > length + 3 else 0)
        slots += list(range(begin, begin + min(length, block)))
        slots += [-1] * (length % 2)
        length, at = length % 17 + 1, at + 1
    report(f"runs of 1 to 17, dim {dim} block {block}, {len(slots)} tokens")
    case = _append_case(gpu_device, slots, q_heads=2, kv_heads=2, dim=dim, block=block, slots=(at + 1) * block)
    _check_append(case)


@pytest.mark.parametrize("heads,dim,block,tokens", [
    ((28, 1), 128, 16, 8192), ((28, 1), 128, 16, 8193), ((28, 1), 128, 64, 4096), ((28, 1), 128, 64, 4097),
    ((33, 2), 64, 32, 11000), ((9, 1), 256, 128, 6000)])  # 32,768 waves of queries or more, 16,384 in large blocks
def test_append_with_queries_of_either_launch(gpu_device, heads, dim, block, tokens):
    """Padding, counting, norms and the queries' own rows as output, whichever launch turns the queries."""

    report(f"append {tokens} tokens, heads {heads} of {dim}, block {block}")
    total = (tokens // block + 2) * block
    slots = [total - 1 - i for i in range(tokens)]
    slots[100:103], slots[tokens - 2], slots[tokens - 1] = [-1, -7, -1], total, total + 12345
    case = _append_case(gpu_device, slots, q_heads=heads[0], kv_heads=heads[1], dim=dim, block=block, slots=total,
                        weights=torch.float32, rotary=32)
    case["positions"][5], case["positions"][tokens // 2], case["positions"][101] = POSITIONS, -1, 2 ** 40
    skipped = torch.full((1,), 3, dtype=torch.int64, device=gpu_device)
    query = case["query"].clone()
    got = _check_append(case, query_output=case["query"], skipped_rows=skipped)
    assert int(skipped) == 3 + 5  # three positions, two slots past the pool
    left_out = [5, tokens // 2, 101]
    assert got is case["query"] and torch.equal(got[left_out], query[left_out])


# -- blocks of an earlier owner ------------------------------------------------------


@pytest.mark.parametrize("block", [16, 64])
def test_rows_added_to_used_blocks_need_cleared_scales(gpu_device, block):
    """A link that leaves rows out, and a prompt's last block: their blocks' scales are the
    rows' own where their bytes were cleared, and else no less than the earlier owner's."""

    sources, destinations = list(range(70)), list(range(256, 326))
    for cleared in (True, False):
        case = _link_case(gpu_device, sources, destinations, block=block, repair=True, low=110, high=111)
        for name in ("key_scales", "value_scales"):
            case[name].view(torch.uint8)[256 // block:] = 0 if cleared else 200
        assert bool(case["repair_mask"].view(torch.uint8)[:64].view(-1, block).any(1).all())  # in every block
        _check_link(case)
        for name in ("key_scales", "value_scales"):
            of_blocks = case[name].view(torch.uint8)[256 // block:-(-326 // block)]
            assert bool(((of_blocks > 0) & (of_blocks < 115)).all() if cleared else (of_blocks == 200).all())
        case = _append_case(gpu_device, list(range(block + 3)), block=block)
        for name in ("key_scales", "value_scales"):
            case[name].view(torch.uint8)[:] = 0 if cleared else 200
        _check_append(case)
        for name in ("key_scales", "value_scales"):
            scales = case[name].view(torch.uint8)[:2]
            assert bool((scales[0] < 130).all()) and bool((scales[1] < 130).all() if cleared else (scales[1] == 200).all())


@pytest.mark.parametrize("runs", list(PADDED))
def test_padding_in_slots_of_32_bits(gpu_device, runs):
    slots = PADDED[runs]
    case = _append_case(gpu_device, slots, dim=64, slots=512, kv_heads=1, q_heads=1, index=torch.int32)
    _check_append(case)
    sources = [1024 + (7 * i) % 512 for i in range(len(slots))]
    case = _link_case(gpu_device, sources, [s if s < 512 else 1536 for s in slots], dim=64, slots=1536, index=torch.int32)
    _check_link(case)


def test_a_captured_append_replays_with_other_padding(gpu_device):
    """One graph of a padded batch, replayed with its padding elsewhere, against eager calls."""

    tokens = 600
    case = _append_case(gpu_device, [-1] * tokens, slots=tokens * 16, q_heads=2)
    twin = {name: value.clone() if name.endswith(("_buffer", "_scales")) else value for name, value in case.items()}
    append_quantized_kv_inplace(**case)
    append_quantized_kv_inplace(**twin)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = append_quantized_kv_inplace(**case)
    for turn, gaps in enumerate(([], [3, 4, 300], range(100, 590), range(1, tokens, 2), range(0, 599))):
        slots = torch.arange(tokens) + 37 * turn
        slots[list(gaps)] = -1
        case["destination_slots"].copy_(slots)
        graph.replay()
        torch.cuda.synchronize()
        before = _state(twin)
        want = append_quantized_kv_inplace(**twin)
        torch.cuda.synchronize()
        assert torch.equal(captured, want)
        _check_pool(twin, before, 16, slots.tolist(), _rows_of(twin, True, "key"), _rows_of(twin, True, "value"),
                    (slots >= 0).tolist())
        assert all(np.array_equal(a, b) for a, b in zip(_state(case), _state(twin)))
