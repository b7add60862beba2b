"""A model's steps over the pool that a link filled, as a program runs them: the
rest of the prompt as one chunk, then single tokens of a batch, each layer's new
keys and values appended before its attention reads them."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from legolink_amd import kv_link
from legolink_amd.head_rotary import append_rotated_kv_inplace, rotate_heads
from legolink_amd.link_runtime import KVPool
from legolink_amd.paged_attention import paged_attention
from legolink_amd.rope import build_cos_sin_cache
from legolink_amd.workloads import QWEN25_7B, scaled_single_request
from tests.gpu_helpers import report
from tests.head_rotary_math import allowed as rotary_allowed
from tests.head_rotary_math import turned
from tests.paged_attention_math import allowed, attend

pytestmark = pytest.mark.gpu
Q_HEADS, KV_HEADS, DIM, LAYERS = 28, 4, 128, 2


def _projection(generator, tokens, device):
    """A step's fused projection and its query, key and value views."""

    widths = [Q_HEADS * DIM, KV_HEADS * DIM, KV_HEADS * DIM]
    rows = torch.randn(tokens, sum(widths), device=device, generator=generator).to(torch.bfloat16)
    return [part.unflatten(-1, (-1, DIM)) for part in rows.split(widths, dim=-1)]


def _check_attention(got, query, pool, layer, table, lengths, starts, page):
    keys, values = pool.get_key_buffer(layer), pool.get_value_buffer(layer)
    want, size, reach = attend(query, keys, values, table, lengths, starts, page=page)
    bound = allowed(want, size, reach, got.dtype, max(lengths), float(values.float().abs().max()))
    off = (got.cpu().double() - want).abs()
    assert bool((off <= bound).all()), f"off by up to {(off / bound).max().item()} of the bound"


def test_chunk_and_tokens_behind_a_link(gpu_device):
    generator = torch.Generator(device=gpu_device).manual_seed(11)
    workload = scaled_single_request(shape=QWEN25_7B, num_slots=4096, block_lengths=[200, 300, 150], imp_per_seam=0,
                                     delta_range=512, name="step")
    pool = KVPool.allocate(num_slots=4096, num_layers=LAYERS, num_heads=KV_HEADS, head_dim=DIM, device=gpu_device)
    for buffer in (*pool.k_buffer, *pool.v_buffer):
        buffer.copy_(torch.randn(buffer.shape, device=gpu_device, generator=generator))
    cos_sin = build_cos_sin_cache(workload.max_position + 1024, DIM).to(gpu_device)

    def device_of(array):
        return torch.from_numpy(np.ascontiguousarray(array)).to(gpu_device)

    kv_link.fused_kv_link_layers_inplace(
        key_buffers=pool.k_buffer, value_buffers=pool.v_buffer, source_slots=device_of(workload.source_slots),
        destination_slots=device_of(workload.destination_slots), local_positions=device_of(workload.local_positions),
        global_positions=device_of(workload.global_positions), cos_sin_cache=cos_sin,
        prefix_token_count=workload.prefix_token_count, rotary_dim=DIM, is_neox_style=True)

    # The linked request and a second one without a past, as rows of slots (pages of one).
    linked = workload.tokens
    used = set(workload.source_slots.tolist()) | set(workload.destination_slots.tolist())
    free = torch.tensor([s for s in range(4096) if s not in used], device=gpu_device)
    free = free[torch.randperm(free.numel(), device=gpu_device, generator=generator)]
    table = torch.full((2, linked + 400), -1, dtype=torch.int32, device=gpu_device)
    table[0, :linked] = device_of(workload.destination_slots).to(torch.int32)
    table[0, linked:] = free[:400].to(torch.int32)
    table[1, :300] = free[400:700].to(torch.int32)
    norms = [(1 + 0.2 * torch.randn(DIM, device=gpu_device, generator=generator)).to(torch.bfloat16) for _ in range(2)]

    lengths = [linked, 0]
    for new in ([173, 90], [1, 1], [1, 1], [4, 1]):
        report(f"step of {new} tokens behind {lengths}")
        positions = torch.cat([torch.arange(n, n + count) for n, count in zip(lengths, new)]).to(gpu_device)
        slots = torch.cat([table[r, n:n + count] for r, (n, count) in enumerate(zip(lengths, new))])
        lengths = [n + count for n, count in zip(lengths, new)]
        single = new == [1, 1]
        starts = None if single else torch.tensor([0, new[0], sum(new)], dtype=torch.int32, device=gpu_device)
        device_lengths = torch.tensor(lengths, dtype=torch.int32, device=gpu_device)
        for layer in range(LAYERS):
            query, key, value = _projection(generator, sum(new), gpu_device)
            before = pool.get_key_buffer(layer).clone()
            rotated = append_rotated_kv_inplace(
                key_buffer=pool.get_key_buffer(layer), value_buffer=pool.get_value_buffer(layer),
                destination_slots=slots, query=query, key=key, value=value, positions=positions,
                cos_sin_cache=cos_sin, rotary_dim=DIM, query_norm_weight=norms[0], key_norm_weight=norms[1])
            out = paged_attention(rotated, pool.get_key_buffer(layer), pool.get_value_buffer(layer), table,
                                  device_lengths, query_starts=starts)
            for rows, got, weight in ((query, rotated, norms[0]),
                                      (key, pool.get_key_buffer(layer)[slots.long()], norms[1])):
                want, size = turned(rows, positions, cos_sin, rotary=DIM, neox=True, weight=weight)
                assert bool(((got.cpu().double() - want).abs() <= rotary_allowed(want, size, got.dtype, DIM)).all())
            assert torch.equal(pool.get_value_buffer(layer)[slots.long()], value)
            rest = torch.ones(4096, dtype=torch.bool, device=gpu_device)
            rest[slots.long()] = False
            assert torch.equal(pool.get_key_buffer(layer)[rest], before[rest])
            _check_attention(out, rotated, pool, layer, table, lengths, None if starts is None else starts, 1)


def test_rotated_heads_and_the_pools_own_write(gpu_device):
    """``rotate_heads`` with ``KVPool.set_kv_buffer`` leaves what one append does."""

    generator = torch.Generator(device=gpu_device).manual_seed(2)
    pools = [KVPool.allocate(num_slots=64, num_layers=1, num_heads=KV_HEADS, head_dim=DIM, device=gpu_device)
             for _ in range(2)]
    for pool in pools:
        for buffer in (*pool.k_buffer, *pool.v_buffer):
            buffer.zero_()
    query, key, value = _projection(generator, 9, gpu_device)
    cos_sin = build_cos_sin_cache(100, DIM).to(gpu_device)
    options = dict(positions=torch.arange(50, 59, device=gpu_device), cos_sin_cache=cos_sin, rotary_dim=DIM)
    slots = torch.randperm(64, device=gpu_device)[:9]
    first, turned_key = rotate_heads(query, key, **options)
    pools[0].set_kv_buffer(0, slots, turned_key, value)
    second = append_rotated_kv_inplace(key_buffer=pools[1].k_buffer[0], value_buffer=pools[1].v_buffer[0],
                                       destination_slots=slots, query=query, key=key, value=value, **options)
    assert torch.equal(first, second)
    assert torch.equal(pools[0].k_buffer[0], pools[1].k_buffer[0])
    assert torch.equal(pools[0].v_buffer[0], pools[1].v_buffer[0])


def test_a_captured_decode_loop(gpu_device):
    """One graph of a batch's step (a padded request among them), replayed token
    after token with eager work between, against the same steps made eagerly."""

    page, requests = 16, 3
    generator = torch.Generator(device=gpu_device).manual_seed(5)
    slots_held = 40 * page
    pools = []
    for _ in range(2):
        pool = KVPool.allocate(num_slots=slots_held, num_layers=LAYERS, num_heads=KV_HEADS, head_dim=DIM,
                               device=gpu_device)
        pools.append(pool)
    for layer in range(LAYERS):
        for name in ("k_buffer", "v_buffer"):
            rows = torch.randn(slots_held, KV_HEADS, DIM, device=gpu_device, generator=generator).to(torch.bfloat16)
            for pool in pools:
                getattr(pool, name)[layer].copy_(rows)
    cos_sin = build_cos_sin_cache(600, DIM).to(gpu_device)
    pages = torch.randperm(40, device=gpu_device, generator=generator).to(torch.int32)
    table = pages[:36].view(requests, 12)
    projected = torch.zeros(requests, (Q_HEADS + 2 * KV_HEADS) * DIM, dtype=torch.bfloat16, device=gpu_device)
    lengths = torch.zeros(requests, dtype=torch.int32, device=gpu_device)
    positions = torch.zeros(requests, dtype=torch.int64, device=gpu_device)
    slots = torch.zeros(requests, dtype=torch.int64, device=gpu_device)

    def step(pool):
        query, key, value = (part.unflatten(-1, (-1, DIM)) for part in
                             projected.split([Q_HEADS * DIM, KV_HEADS * DIM, KV_HEADS * DIM], dim=-1))
        outputs = []
        for layer in range(LAYERS):
            rotated = append_rotated_kv_inplace(
                key_buffer=pool.k_buffer[layer], value_buffer=pool.v_buffer[layer], destination_slots=slots,
                query=query, key=key, value=value, positions=positions, cos_sin_cache=cos_sin, rotary_dim=DIM)
            outputs.append(paged_attention(rotated, pool.k_buffer[layer], pool.v_buffer[layer], table, lengths,
                                           page_size=page))
        return outputs

    slots.fill_(-1)
    step(pools[0])  # padding alone: nothing is written
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(pools[0])
    counts = [130, 15, 0]  # keys before the first step; the last request is padding
    for token in range(5):
        projected.copy_(torch.randn(projected.shape, device=gpu_device, generator=generator))
        places = torch.tensor(counts[:2], device=gpu_device)
        positions[:2] = places
        slots[:2] = table[torch.arange(2, device=gpu_device), places // page].long() * page + places % page
        lengths[:2] = (places + 1).to(torch.int32)
        counts[:2] = [n + 1 for n in counts[:2]]
        graph.replay()
        torch.cuda.synchronize()
        got = [out.clone() for out in captured]
        want = step(pools[1])
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b) and bool((a[2] == 0).all()) and bool(a[:2].any())
        for layer in range(LAYERS):
            assert torch.equal(pools[0].k_buffer[layer], pools[1].k_buffer[layer])
            assert torch.equal(pools[0].v_buffer[layer], pools[1].v_buffer[layer])
