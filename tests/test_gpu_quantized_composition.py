"""GPU tests of the 8-bit pool's calls one after another, as a serving step makes them."""

from __future__ import annotations

import pytest
import torch

from legolink_amd.quantized_pool import (append_quantized_kv_inplace, link_quantized_kv_inplace, load_quantized_kv,
                                         quantized_paged_attention)
from legolink_amd.repair_attention import RepairAttentionPlan
from legolink_amd.rope import build_cos_sin_cache
from tests import quantized_pool_math as qm
from tests.gpu_helpers import report
from tests.head_rotary_math import turned
from tests.paged_attention_math import allowed, attend

pytestmark = pytest.mark.gpu
POSITIONS = 4096


def _empty_pool(device, slots, heads, dim, block):
    pool = {"scale_block": block}
    for name in ("key", "value"):
        pool[f"{name}_buffer"] = torch.zeros(slots, heads, dim, dtype=torch.uint8, device=device).view(torch.float8_e4m3fn)
        pool[f"{name}_scales"] = (torch.zeros(slots // block, heads, dtype=torch.uint8, device=device)
                                  .view(torch.float8_e8m0fnu))
    return pool


class _Model:
    """One layer's projections and table."""

    def __init__(self, device, q_heads, kv_heads, dim, dtype, seed=5):
        self.device, self.heads, self.dim, self.dtype = device, (q_heads, kv_heads), dim, dtype
        self.generator = torch.Generator(device=device).manual_seed(seed)
        self.table = build_cos_sin_cache(POSITIONS, dim).to(device)

    def rows(self, tokens):
        q_heads, kv_heads = self.heads
        projected = torch.randn(tokens, (q_heads + 2 * kv_heads) * self.dim, device=self.device,
                                generator=self.generator).to(self.dtype)
        widths = [q_heads * self.dim, kv_heads * self.dim, kv_heads * self.dim]
        return [part.unflatten(-1, (-1, self.dim)) for part in projected.split(widths, dim=-1)]

    def step(self, pool, slots, positions):
        query, key, value = self.rows(len(slots))
        as_device = lambda values: torch.tensor(values, device=self.device)  # noqa: E731
        rotated = append_quantized_kv_inplace(**pool, destination_slots=as_device(slots), query=query, key=key,
                                              value=value, positions=as_device(positions), cos_sin_cache=self.table,
                                              rotary_dim=self.dim)
        return rotated, key, value


def _slots(pages, page, begin, end):
    return [pages[j // page] * page + j % page for j in range(begin, end)]


def _check_attention(got, query, pool, pages, lengths, starts, page):
    keys = qm.pool_values(pool["key_buffer"], pool["key_scales"], pool["scale_block"])
    values = qm.pool_values(pool["value_buffer"], pool["value_scales"], pool["scale_block"])
    want, size, reach = attend(query, keys, values, pages, lengths, starts, page=page)
    bound = allowed(want, size, reach, got.dtype, max(lengths), float(values.abs().max()))
    assert bool(((got.cpu().double() - want).abs() <= bound).all())


@pytest.mark.parametrize("dtype,dim,block,page", [(torch.bfloat16, 128, 16, 32), (torch.float16, 64, 32, 32),
                                                  (torch.bfloat16, 256, 16, 16)])
def test_a_prompt_and_its_decode(gpu_device, dtype, dim, block, page):
    """Two requests' prompts in one call, then tokens one at a time: the pool holds
    each key and value to half a code's step of its block's scale (twice that where
    the scale grew under it), and attention is that over what the pool holds."""

    report(f"prompt and decode, {dtype} dim {dim} block {block} page {page}")
    model = _Model(gpu_device, 8, 2, dim, dtype)
    pool = _empty_pool(gpu_device, 32 * page, 2, dim, block)
    order = torch.randperm(32, generator=torch.Generator().manual_seed(2)).tolist()
    pages, lengths = [order[:9], order[9:18]], [100, 37]
    table = torch.tensor(pages, dtype=torch.int32, device=gpu_device)
    keys, values = [[], []], [[], []]

    def record(key, value, places):
        at = 0
        for request, positions in places:
            rows = key[at:at + len(positions)]
            where = torch.tensor(positions, device=gpu_device)
            want, _ = turned(rows, where, model.table, rotary=dim, neox=True)
            keys[request].append(want)
            values[request].append(value[at:at + len(positions)].cpu().double())
            at += len(positions)

    places = [(r, list(range(n))) for r, n in enumerate(lengths)]
    slots = [s for r, n in enumerate(lengths) for s in _slots(pages[r], page, 0, n)]
    query, key, value = model.step(pool, slots, [j for _, positions in places for j in positions])
    record(key, value, places)
    starts = torch.tensor([0, lengths[0], sum(lengths)], device=gpu_device)
    counts = torch.tensor(lengths, dtype=torch.int32, device=gpu_device)
    got = quantized_paged_attention(query, **pool, page_table=table, kv_lengths=counts, page_size=page,
                                    query_starts=starts)
    _check_attention(got, query, pool, table, lengths, starts, page)
    for _ in range(20):
        places = [(r, [n]) for r, n in enumerate(lengths)]
        slots = [_slots(pages[r], page, n, n + 1)[0] for r, n in enumerate(lengths)]
        query, key, value = model.step(pool, slots, lengths)
        record(key, value, places)
        lengths = [n + 1 for n in lengths]
        counts += 1
        got = quantized_paged_attention(query, **pool, page_table=table, kv_lengths=counts, page_size=page)
    _check_attention(got, query, pool, table, lengths, None, page)
    for r in range(2):
        at = torch.tensor(_slots(pages[r], page, 0, lengths[r]))
        for rows, name in ((keys[r], "key"), (values[r], "value")):
            held = qm.pool_values(pool[f"{name}_buffer"], pool[f"{name}_scales"], block)[at]
            scale = 2.0 ** (qm.host(pool[f"{name}_scales"]).astype(float) - 127)
            least = torch.from_numpy(scale)[at // block][..., None] * 2.0 ** -10  # half of e4m3's least step
            want = torch.cat(rows)
            # e4m3: half a step is 2^-4 of the value; rounded again under a scale that grew, in its subnormal range.
            assert bool(((held - want).abs() <= 2.0 ** -4 * want.abs() + 2 * least).all())


def test_linked_rows_are_attended_and_repaired(gpu_device):
    """Cached blocks linked to a new request, its boundary rows left to the repair pass,
    which reads the linked rows in 16 bits, and a chunk of new tokens behind them."""

    dim, block, page, cached, linked = 128, 16, 16, 160, 130
    model = _Model(gpu_device, 8, 2, dim, torch.bfloat16)
    pool = _empty_pool(gpu_device, 40 * page, 2, dim, block)
    model.step(pool, list(range(cached)), list(range(cached)))  # compiled once, at positions of its own
    source = torch.cat((torch.arange(20, 90), torch.arange(100, 160))).to(gpu_device)
    pages = torch.randperm(30, generator=torch.Generator().manual_seed(8))[:12] + 10  # apart from the cached ones
    place = torch.arange(linked + 40)
    slots = (pages[place // page] * page + place % page).to(gpu_device)
    mask = torch.zeros(linked, dtype=torch.bool, device=gpu_device)
    mask[70:78] = True  # the seam
    positions = torch.arange(linked, device=gpu_device)
    link_quantized_kv_inplace(**pool, source_slots=source, destination_slots=slots[:linked], local_positions=source,
                              global_positions=positions, cos_sin_cache=model.table, rotary_dim=dim, repair_mask=mask)
    # The seam's rows, recomputed: appended where the link left room.
    repaired, *_ = model.step(pool, slots[70:78].tolist(), list(range(70, 78)))
    keys, values = load_quantized_kv(**pool, slots=slots[:linked])
    plan = RepairAttentionPlan([(torch.arange(linked, dtype=torch.int32, device=gpu_device), 70, 78)],
                               num_q_heads=8, num_kv_heads=2, head_dim=dim, pool_size=linked)
    out = plan.run(repaired, keys, values)
    want, size, reach = attend(repaired, keys, values, torch.arange(linked)[None], [78], [0, 8], page=1)
    bound = allowed(want, size, reach, out.dtype, 78, float(values.float().abs().max()))
    assert bool(((out.cpu().double() - want).abs() <= bound).all())
    # New tokens behind the linked context.
    query, *_ = model.step(pool, slots[linked:].tolist(), list(range(linked, linked + 40)))
    table = pages.to(torch.int32)[None].to(gpu_device)
    got = quantized_paged_attention(query, **pool, page_table=table, page_size=page,
                                    kv_lengths=torch.tensor([linked + 40], device=gpu_device),
                                    query_starts=torch.tensor([0, 40], device=gpu_device))
    _check_attention(got, query, pool, table, [linked + 40], [0, 40], page)
    # The cached rows are as they were: linked again elsewhere, unturned, they are the same values.
    again = torch.arange(36 * page, 36 * page + 60, device=gpu_device)
    link_quantized_kv_inplace(**pool, source_slots=torch.arange(32, 92, device=gpu_device), destination_slots=again,
                              local_positions=again % 64, global_positions=again % 64, cos_sin_cache=model.table,
                              rotary_dim=dim, prefix_token_count=60)
    assert all(torch.equal(a, b) for a, b in zip(
        load_quantized_kv(**pool, slots=again[:48]), load_quantized_kv(**pool, slots=torch.arange(32, 80, device=gpu_device))))


def test_a_captured_decode_step(gpu_device):
    """Append and attention of a decode batch in one graph, replayed token by token,
    against eager steps on a pool of its own."""

    dim, block, page, requests = 128, 16, 16, 3
    tables = torch.randperm(60, generator=torch.Generator().manual_seed(3)).view(3, 20).to(torch.int32).to(gpu_device)
    pools = [_empty_pool(gpu_device, 60 * page, 4, dim, block) for _ in range(2)]
    table = build_cos_sin_cache(POSITIONS, dim).to(gpu_device)
    lengths = torch.tensor([0, 17, 250], dtype=torch.int64, device=gpu_device)
    rows = [torch.zeros(requests, heads, dim, dtype=torch.bfloat16, device=gpu_device) for heads in (28, 4, 4)]

    def step(pool):
        counts = lengths + 1
        page_of = torch.gather(tables, 1, (lengths // page)[:, None])[:, 0].long()
        query = append_quantized_kv_inplace(**pool, destination_slots=page_of * page + lengths % page, query=rows[0],
                                            key=rows[1], value=rows[2], positions=lengths, cos_sin_cache=table,
                                            rotary_dim=dim)
        return quantized_paged_attention(query, **pool, page_table=tables, kv_lengths=counts, page_size=page)

    for pool in pools:
        step(pool)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(pools[0])
    generator = torch.Generator(device=gpu_device).manual_seed(4)
    for turn in range(40):
        lengths.add_(1)
        for part in rows:
            part.copy_(torch.randn(part.shape, device=gpu_device, generator=generator) * (1 + turn % 7))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(captured, step(pools[1]))
        torch.cuda.synchronize()
    for name in ("key_buffer", "value_buffer", "key_scales", "value_scales"):
        assert torch.equal(*(pool[name].view(torch.uint8) for pool in pools))
