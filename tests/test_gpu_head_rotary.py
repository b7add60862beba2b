"""GPU tests of the norm-and-rotate and append operators against 64 bits."""

from __future__ import annotations

import pytest
import torch

from legolink_amd.head_rotary import append_rotated_kv_inplace, rotate_heads
from legolink_amd.rope import build_cos_sin_cache
from tests.gpu_helpers import report
from tests.head_rotary_math import allowed, turned

pytestmark = pytest.mark.gpu
POSITIONS = 4096


def _case(device, *, tokens, q_heads=4, kv_heads=2, dim=128, rotary=None, dtype=torch.bfloat16,
          table=torch.float32, weights=None, index=torch.int64, layout="fused", value_dim=None, seed=1):
    generator = torch.Generator(device=device).manual_seed(seed)
    value_dim = dim if value_dim is None else value_dim
    widths = [q_heads * dim, kv_heads * dim, kv_heads * value_dim]

    def normal(*shape):
        return (torch.randn(*shape, device=device, generator=generator) * 2).to(dtype)

    if layout == "by head":  # [heads, tokens, dim] storage
        rows = [normal(h, tokens, d).transpose(0, 1) for h, d in ((q_heads, dim), (kv_heads, dim), (kv_heads, value_dim))]
    else:
        # "fused": views of one projection; "odd": at an address that is no multiple of 16 bytes.
        odd = 1 if layout == "odd" else 0
        projected = normal(tokens, sum(widths) + odd)[:, odd:]
        rows = [part.unflatten(-1, (-1, d)) for part, d in zip(projected.split(widths, dim=-1), (dim, dim, value_dim))]
    rotary = dim if rotary is None else rotary
    norms = [None, None]
    if weights is not None:
        norms = [(1 + 0.4 * torch.randn(dim, device=device, generator=generator)).to(weights) for _ in range(2)]
    arguments = dict(query=rows[0], key=rows[1], rotary_dim=rotary, query_norm_weight=norms[0],
                     key_norm_weight=norms[1],
                     positions=torch.randint(POSITIONS, (tokens,), device=device, generator=generator).to(index),
                     cos_sin_cache=build_cos_sin_cache(POSITIONS, rotary, dtype=table).to(device))
    return arguments, rows[2]


def _close(got, rows, arguments, weight, neox):
    want, size = turned(rows, arguments["positions"], arguments["cos_sin_cache"], rotary=arguments["rotary_dim"],
                        neox=neox, weight=weight)
    off = (got.detach().cpu().double() - want).abs()
    bound = allowed(want, size, got.dtype, rows.shape[-1])
    assert bool((off <= bound).all()), f"off by up to {(off / bound).max().item()} of the bound"


SHAPES = [  # dim, rotary: the vector kernel's groups of 1 to 16 lanes (5 and 7 used of 8), then the element kernel's
    (128, 128), (128, 64), (64, 64), (64, 32), (256, 256), (256, 32), (16, 16), (32, 16), (80, 80), (112, 32),
    (40, 16), (24, 24), (128, 8), (6, 2), (2, 2), (129, 128), (200, 90),
]


@pytest.mark.parametrize("dim,rotary", SHAPES)
@pytest.mark.parametrize("neox", [True, False])
@pytest.mark.parametrize("dtype,weights", [(torch.bfloat16, None), (torch.bfloat16, torch.bfloat16),
                                           (torch.float16, torch.float32)])
def test_rotate_heads_matches_64_bits(gpu_device, dim, rotary, neox, dtype, weights):
    report(f"rotate_heads dim {dim} rotary {rotary} neox {neox} {dtype} weights {weights}")
    arguments, _ = _case(gpu_device, tokens=5, q_heads=7, kv_heads=3, dim=dim, rotary=rotary, dtype=dtype,
                         weights=weights)
    query, key = rotate_heads(**arguments, is_neox_style=neox)
    assert query.is_contiguous() and key.is_contiguous()
    _close(query, arguments["query"], arguments, arguments["query_norm_weight"], neox)
    _close(key, arguments["key"], arguments, arguments["key_norm_weight"], neox)


@pytest.mark.parametrize("layout", ["fused", "by head", "odd"])
@pytest.mark.parametrize("tokens", [1, 2, 67, 300])
@pytest.mark.parametrize("table,index", [(torch.float32, torch.int32), (torch.bfloat16, torch.int64),
                                         (torch.float16, torch.int64)])
def test_rotate_heads_layouts_and_tables(gpu_device, layout, tokens, table, index):
    report(f"rotate_heads {layout} tokens {tokens} table {table}")
    arguments, _ = _case(gpu_device, tokens=tokens, q_heads=28, kv_heads=4, table=table, index=index, layout=layout,
                         weights=torch.float16)
    query, key = rotate_heads(**arguments)
    _close(query, arguments["query"], arguments, arguments["query_norm_weight"], True)
    _close(key, arguments["key"], arguments, arguments["key_norm_weight"], True)


def test_one_norm_alone(gpu_device):
    arguments, _ = _case(gpu_device, tokens=9, weights=torch.float32)
    for kept in ("query_norm_weight", "key_norm_weight"):
        only = {**arguments, "query_norm_weight": None, "key_norm_weight": None, kept: arguments[kept]}
        query, key = rotate_heads(**only)
        _close(query, arguments["query"], arguments, only["query_norm_weight"], True)
        _close(key, arguments["key"], arguments, only["key_norm_weight"], True)


@pytest.mark.parametrize("dim,rotary,layout", [(128, 128, "fused"), (128, 128, "by head"), (40, 16, "fused"),
                                               (200, 90, "odd")])
@pytest.mark.parametrize("neox", [True, False])
def test_in_place_equals_out_of_place(gpu_device, dim, rotary, layout, neox):
    report(f"rotate_heads in place dim {dim} {layout} neox {neox}")
    arguments, value = _case(gpu_device, tokens=33, dim=dim, rotary=rotary, layout=layout, weights=torch.bfloat16)
    value_before = value.clone()
    want = rotate_heads(**arguments, is_neox_style=neox)
    got = rotate_heads(**arguments, is_neox_style=neox, query_output=arguments["query"],
                       key_output=arguments["key"])
    assert got[0] is arguments["query"] and got[1] is arguments["key"]
    for a, b in zip(got, want):
        assert torch.equal(a.contiguous().view(torch.int16), b.view(torch.int16))
    assert torch.equal(value, value_before)  # the rows between them


def test_rows_of_special_values(gpu_device):
    """Infinities and NaN stay in their own pair (no norm), zeros give zeros (eps holds the norm)."""

    arguments, _ = _case(gpu_device, tokens=4, dim=64)
    rows = arguments["query"]
    rows[0, 0, 3], rows[1, 1, 7] = float("nan"), float("inf")
    query, _ = rotate_heads(**arguments)
    bad = ~torch.isfinite(query).cpu()
    assert set(map(tuple, bad.nonzero().tolist())) <= {(0, 0, 3), (0, 0, 35), (1, 1, 7), (1, 1, 39)}
    assert bool(bad[0, 0, 3]) and bool(bad[0, 0, 35])
    rows.zero_()
    weight = torch.ones(64, device=gpu_device)
    query, _ = rotate_heads(**{**arguments, "query_norm_weight": weight})
    assert bool((query == 0).all())


@pytest.mark.parametrize("dim", [128, 40])
def test_positions_outside_the_table_are_left_out_and_counted(gpu_device, dim):
    arguments, _ = _case(gpu_device, tokens=9, dim=dim, rotary=16)
    bad = torch.tensor([2, 5, 8], device=gpu_device)
    arguments["positions"][bad] = torch.tensor([-1, POSITIONS, 2 ** 40], device=gpu_device)
    outputs = [torch.full_like(arguments[name].contiguous(), 3.0) for name in ("query", "key")]
    counter = torch.zeros(1, dtype=torch.int64, device=gpu_device)
    query, key = rotate_heads(**arguments, query_output=outputs[0], key_output=outputs[1], skipped_rows=counter)
    assert int(counter) == 3
    assert bool((query[bad] == 3).all()) and bool((key[bad] == 3).all())
    kept = torch.tensor([0, 1, 3, 4, 6, 7], device=gpu_device)
    part = {**arguments, "positions": arguments["positions"][kept]}
    _close(query[kept], arguments["query"][kept], part, None, True)
    _close(key[kept], arguments["key"][kept], part, None, True)


@pytest.mark.parametrize("dim,value_dim,rotary,dtype", [
    (128, 128, 128, torch.bfloat16), (128, 64, 128, torch.float16), (256, 256, 64, torch.bfloat16),
    (64, 64, 64, torch.float16), (80, 80, 80, torch.bfloat16), (40, 24, 16, torch.bfloat16), (96, 7, 96, torch.float16),
])
@pytest.mark.parametrize("tokens,index", [(1, torch.int64), (37, torch.int32), (260, torch.int64)])
def test_append_writes_its_slots_and_nothing_else(gpu_device, dim, value_dim, rotary, dtype, tokens, index):
    report(f"append dim {dim}/{value_dim} tokens {tokens}")
    arguments, value = _case(gpu_device, tokens=tokens, q_heads=7, kv_heads=3, dim=dim, value_dim=value_dim,
                             rotary=rotary, dtype=dtype, weights=torch.float32, index=index)
    slots_held = 600
    generator = torch.Generator(device=gpu_device).manual_seed(4)
    keys = torch.randn(slots_held, 3, dim, device=gpu_device, generator=generator).to(dtype)
    values = torch.randn(slots_held, 3, value_dim, device=gpu_device, generator=generator).to(dtype)
    before_k, before_v = keys.clone(), values.clone()
    slots = torch.randperm(slots_held, device=gpu_device, generator=generator)[:tokens].to(index)
    # Every seventh token is padding or has a slot past the pool.
    away = torch.arange(6, max(tokens, 6), 7, device=gpu_device)
    slots[away] = torch.where(away % 2 == 0, -1, slots_held + 5).to(index)
    counter = torch.zeros(1, dtype=torch.int64, device=gpu_device)
    query = append_rotated_kv_inplace(key_buffer=keys, value_buffer=values, destination_slots=slots, value=value,
                                      skipped_rows=counter, **arguments)
    assert int(counter) == int((slots >= slots_held).sum())
    _close(query, arguments["query"], arguments, arguments["query_norm_weight"], True)
    there = (slots >= 0) & (slots < slots_held)
    at = slots[there].long()
    part = {**arguments, "positions": arguments["positions"][there]}
    _close(keys[at], arguments["key"][there], part, arguments["key_norm_weight"], True)
    assert torch.equal(values[at].view(torch.int16), value[there].contiguous().view(torch.int16))
    rest = torch.ones(slots_held, dtype=torch.bool, device=gpu_device)
    rest[at] = False
    assert torch.equal(keys[rest].view(torch.int16), before_k[rest].view(torch.int16))
    assert torch.equal(values[rest].view(torch.int16), before_v[rest].view(torch.int16))


def test_append_equals_rotate_heads_bit_for_bit(gpu_device):
    arguments, value = _case(gpu_device, tokens=130, q_heads=28, kv_heads=4, weights=torch.bfloat16)
    query, key = rotate_heads(**arguments)
    keys = torch.zeros(256, 4, 128, dtype=torch.bfloat16, device=gpu_device)
    values = torch.zeros_like(keys)
    slots = torch.randperm(256, device=gpu_device)[:130]
    got = append_rotated_kv_inplace(key_buffer=keys, value_buffer=values, destination_slots=slots, value=value,
                                    query_output=arguments["query"], **arguments)
    assert got is arguments["query"]
    assert torch.equal(got.contiguous().view(torch.int16), query.view(torch.int16))
    assert torch.equal(keys[slots].view(torch.int16), key.view(torch.int16))


def test_append_with_a_position_outside_the_table_writes_nothing_of_the_token(gpu_device):
    arguments, value = _case(gpu_device, tokens=3)
    arguments["positions"][1] = POSITIONS
    keys = torch.full((8, 2, 128), 5.0, dtype=torch.bfloat16, device=gpu_device)
    values = keys.clone()
    counter = torch.zeros(1, dtype=torch.int64, device=gpu_device)
    append_rotated_kv_inplace(key_buffer=keys, value_buffer=values, value=value, skipped_rows=counter,
                              destination_slots=torch.tensor([4, 8, 6], device=gpu_device), **arguments)
    assert int(counter) == 1  # bad in both ways, counted once
    untouched = torch.tensor([0, 1, 2, 3, 5, 7], device=gpu_device)
    assert bool((keys[untouched] == 5).all()) and bool((values[untouched] == 5).all())
    assert torch.equal(values[6], value[2])


def test_no_tokens(gpu_device):
    arguments, value = _case(gpu_device, tokens=0)
    query, key = rotate_heads(**arguments)
    assert query.shape == (0, 4, 128) and key.shape == (0, 2, 128)
    keys = torch.zeros(4, 2, 128, dtype=torch.bfloat16, device=gpu_device)
    append_rotated_kv_inplace(key_buffer=keys, value_buffer=keys.clone(), value=value,
                              destination_slots=torch.zeros(0, dtype=torch.int64, device=gpu_device), **arguments)
    empty = torch.zeros(0, 2, 128, dtype=torch.bfloat16, device=gpu_device)  # a pool without rows
    arguments, value = _case(gpu_device, tokens=2)
    counter = torch.zeros(1, dtype=torch.int64, device=gpu_device)
    query = append_rotated_kv_inplace(key_buffer=empty, value_buffer=empty.clone(), value=value, skipped_rows=counter,
                                      destination_slots=torch.tensor([0, -1], device=gpu_device), **arguments)
    assert int(counter) == 1
    _close(query, arguments["query"], arguments, None, True)


def test_append_past_four_gib(gpu_device):
    """A pool whose last rows lie past 2^32 bytes."""

    slots = (1 << 32) // (2 * 128 * 2) + 64
    keys = torch.zeros(slots, 2, 128, dtype=torch.bfloat16, device=gpu_device)
    values = torch.zeros_like(keys)
    arguments, value = _case(gpu_device, tokens=3)
    at = torch.tensor([slots - 1, 0, slots - 40], device=gpu_device)
    append_rotated_kv_inplace(key_buffer=keys, value_buffer=values, destination_slots=at, value=value, **arguments)
    _close(keys[at], arguments["key"], arguments, None, True)
    assert torch.equal(values[at], value)
    assert int((keys != 0).any(-1).any(-1).sum()) == 3


def test_captured_append_replays(gpu_device):
    arguments, value = _case(gpu_device, tokens=17, weights=torch.bfloat16)
    keys = torch.zeros(64, 2, 128, dtype=torch.bfloat16, device=gpu_device)
    values = torch.zeros_like(keys)
    slots = torch.arange(17, device=gpu_device)

    def step():
        return append_rotated_kv_inplace(key_buffer=keys, value_buffer=values, destination_slots=slots, value=value,
                                         **arguments)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for replay in range(3):
        arguments["positions"].copy_((arguments["positions"] + 11 * replay) % POSITIONS)
        slots.copy_(torch.randperm(64, device=gpu_device)[:17])
        keys.zero_()
        values.zero_()
        graph.replay()
        torch.cuda.synchronize()
        got, got_keys, got_values = captured.clone(), keys.clone(), values.clone()
        keys.zero_()
        values.zero_()
        assert torch.equal(got, step())
        assert torch.equal(got_keys, keys) and torch.equal(got_values, values)


def test_another_stream(gpu_device):
    arguments, _ = _case(gpu_device, tokens=50)
    want = rotate_heads(**arguments)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = rotate_heads(**arguments)
    stream.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
