"""Performance cases of the operators of a paged pool held in 8 bits.

One layer's pool holds keys and values as 8-bit floats (e4m3) with a scale, a
power of two held in 8 bits (e8m0), for each head of every ``block`` tokens.
Four kinds of call:

* ``append``: a step's new tokens into the pool: norms for each head, rotation,
  quantisation (``append_quantized_kv_inplace``);
* ``link``: cached rows to a new request's slots, their keys turned to their new
  positions (``link_quantized_kv_inplace``);
* ``load``: rows of the pool in 16 or 32 bits (``load_quantized_kv``);
* ``attention``: each request's new tokens over its pages
  (``quantized_paged_attention``), single tokens and chunks.

A call that writes the pool returns it as the values it stands for.  Where
``own`` is false everything is computed from elementary torch operations in 32
bits.  A case fixes everything that the amount of work depends on; the seed draws
the pages, the slots, the positions and the values.
"""

from __future__ import annotations

import functools
import math
import sys
from pathlib import Path

import torch

# The framework's package, imported by the calls that are made of it.
_PACKAGE = str(Path.cwd() / "sglang-legolink_amd")
if _PACKAGE not in sys.path:
    sys.path.insert(0, _PACKAGE)

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32,
          "int32": torch.int32, "int64": torch.int64}
SIZES = {"bf16": 2, "fp16": 2, "fp32": 4, "int32": 4, "int64": 8}
NORM_EPS = 1e-6
ROPE_THETA = 1_000_000.0
CONTEXT = 131072  # rows of the cos/sin table
MOST_CODE = 448.0  # e4m3's largest
REPAIR_EVERY = 24  # tokens of a linked context for one that the repair pass recomputes


def _append(**options):
    """``tokens`` new tokens of ``requests`` requests, behind what their blocks hold."""

    case = {"kind": "append", "tokens": 64, "requests": 64, "block": 16, "page": 16, "q_heads": 28, "kv_heads": 4,
            "dim": 128, "rotary": 128, "norm": False, "neox": True, "dtype": "bf16", "table": "fp32", "index": "int64"}
    return {**case, **options}


def _link(**options):
    """``tokens`` linked tokens in runs of ``run`` of a catalogue of ``cached`` tokens."""

    case = {"kind": "link", "tokens": 32768, "run": 512, "cached": 8192, "block": 16, "kv_heads": 4, "dim": 128,
            "rotary": 128, "neox": True, "repair": True, "dtype": "bf16", "table": "fp32", "index": "int64"}
    return {**case, **options}


def _load(**options):
    case = {"kind": "load", "tokens": 32768, "block": 16, "kv_heads": 4, "dim": 128, "dtype": "bf16",
            "index": "int64"}
    return {**case, **options}


def _attention(**options):
    """``queries`` new tokens of each of ``requests`` requests (the shortest has
    ``least_queries``), over keys that count ``least_keys`` to ``keys``, their
    own among them."""

    case = {"kind": "attention", "requests": 1, "queries": 1, "least_queries": 1, "keys": 2048, "least_keys": 2048,
            "block": 16, "page": 16, "q_heads": 28, "kv_heads": 4, "dim": 128, "dtype": "bf16"}
    return {**case, **options}


def listed():
    return [
        # A decode step of 64 requests: each one's new key and value behind those of its block.
        _append(name="append_64_tokens"),
        # A linked request's tail, prefilled in one chunk, of a model with norms.
        _append(name="append_16k_tokens", tokens=16384, requests=1, norm=True),
        # A short context of a small model in fp16 from a few cached blocks: the link where latency counts.
        _link(name="link_1k_tokens", tokens=1237, run=211, cached=1024, kv_heads=2, dim=64, rotary=64, dtype="fp16",
              index="int32"),
        # c2's length, linked from a catalogue that several requests share.
        _link(name="link_32k_tokens"),
        # The rows that a repair pass of a few hundred tokens reads.
        _load(name="load_701_rows", tokens=701),
        # A linked context of wide heads on its way to a 16-bit pool.
        _load(name="load_32k_rows", kv_heads=2, dim=256, block=64, dtype="fp16", index="int32"),
        # The next token of a short chat (c1's length): the latency of one layer's attention.
        _attention(name="decode_2k_keys"),
        # The next token over the longest context.
        _attention(name="decode_131k_keys", keys=131072, least_keys=131072),
        # A serving batch of uneven requests in larger pages.
        _attention(name="decode_batch_of_64", requests=64, keys=32768, least_keys=500, page=64, block=64, q_heads=64,
                   kv_heads=8),
        # A chunk of 2,048 new tokens behind a linked 30k-token context (c2's length).
        _attention(name="chunk_behind_32k_keys", queries=2048, least_queries=2048, keys=32768, least_keys=32768),
        # Short chunks of several requests of a small model, uneven on both sides.
        _attention(name="chunks_of_6", requests=6, queries=701, least_queries=5, keys=9000, least_keys=300, page=48,
                   q_heads=14, kv_heads=2, dim=64, dtype="fp16"),
        # A whole prompt of a model with wide heads, nothing cached before it.
        _attention(name="prompt_wide_heads", queries=4099, least_queries=4099, keys=4099, least_keys=4099, page=128,
                   block=64, q_heads=16, kv_heads=2, dim=256),
    ]


# What a drawn case may have at most, so that it costs no more than the listed
# ones: bytes moved, multiplications, and values of the plain form's padded
# scores and keys.
_MOST_BYTES = 4 * 10 ** 8
_MOST_READ = 64 * 32768 * 2 * 8 * 128 // 4
_MOST_FLOPS = 4 * 128 * 28 * 2048 * 30000
_MOST_SCORES = 2048 * 28 * 32768
_MOST_PADDED = 64 * 32768 * 8 * 128

_HEADS = [(28, 4), (28, 4), (64, 8), (14, 2), (7, 1), (10, 10), (16, 2), (32, 1)]
_DIMS = [(128, 128), (128, 64), (64, 64), (64, 32), (256, 256)]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["append", "append", "link", "link", "load", "attention", "attention", "attention"])
    while True:
        q_heads, kv_heads = rng.choice(_HEADS)
        dtype = rng.choice(["bf16", "bf16", "fp16"])
        block = rng.choice([16, 16, 32, 64, 128])
        dim, rotary = rng.choice(_DIMS)
        if kind == "append":
            tokens = _log(rng, 1, 16384)
            case = _append(tokens=tokens, requests=rng.choice([min(tokens, 2048), _log(rng, 1, min(tokens, 64))]),
                           block=block, page=block * rng.choice([1, 1, 2, 3]), q_heads=q_heads, kv_heads=kv_heads,
                           dim=dim, rotary=rotary, norm=rng.random() < 0.6, neox=rng.random() < 0.8, dtype=dtype,
                           table=rng.choice(["fp32", "fp32", "bf16", "fp16"]), index=rng.choice(["int64", "int32"]))
        elif kind == "link":
            tokens = _log(rng, 1, 32768)
            case = _link(tokens=tokens, run=_log(rng, 1, 2000), cached=_log(rng, 64, 16384), block=block,
                         kv_heads=kv_heads, dim=dim, rotary=rotary, neox=rng.random() < 0.8,
                         repair=rng.random() < 0.7, dtype=dtype, table=rng.choice(["fp32", "fp32", "bf16", "fp16"]),
                         index=rng.choice(["int64", "int32"]))
        elif kind == "load":
            case = _load(tokens=_log(rng, 1, 65536), block=block, kv_heads=kv_heads, dim=dim,
                         dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]), index=rng.choice(["int64", "int32"]))
        if kind != "attention":
            if work(case)["bytes"] <= _MOST_BYTES:
                return case
            continue
        requests = rng.choice([1, 1, _log(rng, 2, 64), _log(rng, 2, 64)])
        least_queries = queries = 1
        if rng.random() < 0.6:  # a chunk
            queries = _log(rng, 2, 4096)
            least_queries = _log(rng, 1, queries)
        keys = max(queries, _log(rng, 16, CONTEXT))
        least_keys = max(queries, _log(rng, max(1, min(16, keys)), keys))
        case = _attention(requests=requests, queries=queries, least_queries=least_queries, keys=keys,
                          least_keys=min(least_keys, keys), block=block, page=block * rng.choice([1, 1, 2, 3]),
                          q_heads=q_heads, kv_heads=kv_heads, dim=dim, dtype=dtype)
        cost = work(case)
        if (cost["bytes"] <= _MOST_READ and cost["flops"] <= _MOST_FLOPS
                and requests * queries * q_heads * keys <= _MOST_SCORES
                and requests * keys * kv_heads * dim <= _MOST_PADDED):
            return case


# -- what the cases hold ----------------------------------------------------


def _spread(low, high, count):
    """``count`` sizes between ``low`` and ``high``, spread over their logarithm
    in an order that is not sorted; the first is ``high``."""

    sizes = [round(low * (high / low) ** ((0.618 * i + 0.31) % 1.0)) for i in range(count)]
    return [high, *sizes[1:]]


def _queries(case):
    return _spread(case["least_queries"], case["queries"], case["requests"])


def _keys(case):
    return [max(keys, queries) for keys, queries in
            zip(_spread(case["least_keys"], case["keys"], case["requests"]), _queries(case))]


def _new_tokens(case):
    """The requests' new tokens: uneven, ``tokens`` in all."""

    tokens, requests = case["tokens"], case["requests"]
    if tokens == requests:
        return [1] * requests
    weights = [1 + (0.618 * i) % 1.0 for i in range(requests)]
    counts = [int((tokens - requests) * weight / sum(weights)) + 1 for weight in weights]
    counts[0] += tokens - sum(counts)
    return counts


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _normal(generator, *shape, dtype):
    return torch.randn(*shape, dtype=dtype, device="cuda", generator=generator)


def _whole(generator, low, high, *shape, dtype=torch.int64):
    return torch.randint(low, high, shape, device="cuda", generator=generator, dtype=dtype)


@functools.lru_cache(maxsize=8)
def _table(rotary, dtype):
    """The model's cos/sin table, built once per program: cos in the first half
    of a row, sin in the second, from angles in 64 bits."""

    frequencies = ROPE_THETA ** (-torch.arange(0, rotary, 2, dtype=torch.float64, device="cuda") / rotary)
    angles = torch.arange(CONTEXT, dtype=torch.float64, device="cuda")[:, None] * frequencies
    return torch.cat((angles.cos(), angles.sin()), dim=-1).to(DTYPES[dtype])


def _pool(generator, slots, heads, dim, block):
    """Codes that fill e4m3's range as a block's largest value does, and scales
    that make them values of about one."""

    codes = (80 * _normal(generator, slots, heads, dim, dtype=torch.bfloat16)).clamp_(-MOST_CODE, MOST_CODE)
    scales = _whole(generator, 119, 123, slots // block, heads, dtype=torch.uint8)
    return codes.to(torch.float8_e4m3fn), scales.view(torch.float8_e8m0fnu)


def _both_pools(generator, slots, heads, dim, block):
    key_buffer, key_scales = _pool(generator, slots, heads, dim, block)
    value_buffer, value_scales = _pool(generator, slots, heads, dim, block)
    return {"key_buffer": key_buffer, "value_buffer": value_buffer, "key_scales": key_scales,
            "value_scales": value_scales, "scale_block": block}


def prepare(case, seed):
    return {"append": _prepare_append, "link": _prepare_link, "load": _prepare_load,
            "attention": _prepare_attention}[case["kind"]](case, seed)


def _prepare_append(case, seed):
    generator = _generator(seed)
    tokens, dim, block, page, dtype = case["tokens"], case["dim"], case["block"], case["page"], DTYPES[case["dtype"]]
    counts = torch.tensor(_new_tokens(case), device="cuda")
    requests = counts.numel()
    # Each request's first token comes behind what its page holds already (a long prompt's at a page's begin).
    begin = _whole(generator, 0, page, requests) if case["requests"] > 1 else torch.zeros_like(counts)
    pages = (begin + counts + page - 1) // page
    first_page = pages.cumsum(0) - pages
    total = sum(-(-(page - 1 + count) // page) for count in _new_tokens(case)) + 2
    order = torch.randperm(total, device="cuda", generator=generator)
    request = torch.repeat_interleave(torch.arange(requests, device="cuda"), counts, output_size=tokens)
    place = torch.arange(tokens, device="cuda") - (counts.cumsum(0) - counts)[request] + begin[request]
    slots = order[first_page[request] + place // page] * page + place % page
    heads = case["q_heads"] + 2 * case["kv_heads"]
    # The model's fused projection of a step's tokens; channels of different scale.
    projected = _normal(generator, tokens, heads * dim, dtype=dtype)
    projected *= torch.linspace(0.25, 4.0, heads * dim, device="cuda").to(dtype)
    state = {**_both_pools(generator, total * page, case["kv_heads"], dim, block), "kind": "append",
             "projected": projected, "q_heads": case["q_heads"], "kv_heads": case["kv_heads"], "dim": dim,
             "rotary": case["rotary"], "neox": case["neox"], "query_norm": None, "key_norm": None, "dtype": dtype,
             "table": _table(case["rotary"], case["table"]), "slots": slots.to(DTYPES[case["index"]]),
             "positions": _whole(generator, 0, CONTEXT, tokens).to(DTYPES[case["index"]])}
    if case["norm"]:
        state["query_norm"] = (1.0 + 0.3 * _normal(generator, dim, dtype=torch.float32)).to(dtype)
        state["key_norm"] = (1.0 + 0.3 * _normal(generator, dim, dtype=torch.float32)).to(dtype)
    return state


def _prepare_link(case, seed):
    generator = _generator(seed)
    tokens, block, index = case["tokens"], case["block"], DTYPES[case["index"]]
    cached, linked = -(-case["cached"] // block), -(-tokens // block)
    state = _both_pools(generator, (cached + linked) * block, case["kv_heads"], case["dim"], block)
    # Runs of the catalogue, each from anywhere in it; the request's blocks are new ones, in any order.
    run = min(case["run"], cached * block)
    runs = -(-tokens // run)
    offset = torch.arange(tokens, device="cuda")
    source = _whole(generator, 0, cached * block - run + 1, runs)[offset // run] + offset % run
    blocks = cached + torch.randperm(linked, device="cuda", generator=generator)
    for scales in (state["key_scales"], state["value_scales"]):
        scales.view(torch.uint8)[cached:] = 0
    repair = torch.rand(tokens, device="cuda", generator=generator) * REPAIR_EVERY < 1 if case["repair"] else None
    return {**state, "kind": "link", "rotary": case["rotary"], "neox": case["neox"], "dtype": DTYPES[case["dtype"]],
            "table": _table(case["rotary"], case["table"]), "source": source.to(index),
            "slots": (blocks[offset // block] * block + offset % block).to(index), "repair": repair,
            "local": (source % 4096).to(index), "global": (offset + 2048).to(index)}


def _prepare_load(case, seed):
    generator = _generator(seed)
    tokens, block = case["tokens"], case["block"]
    blocks = -(-tokens // block) + 16
    order = torch.randperm(blocks, device="cuda", generator=generator)
    place = torch.arange(tokens, device="cuda")
    return {**_both_pools(generator, blocks * block, case["kv_heads"], case["dim"], block), "kind": "load",
            "slots": (order[place // block] * block + place % block).to(DTYPES[case["index"]]),
            "dtype": DTYPES[case["dtype"]]}


def _prepare_attention(case, seed):
    generator = _generator(seed)
    dtype, page, dim = DTYPES[case["dtype"]], case["page"], case["dim"]
    queries, keys = _queries(case), _keys(case)
    pages = [-(-count // page) for count in keys]
    total = sum(pages) + max(8, sum(pages) // 16)
    state = _both_pools(generator, total * page, case["kv_heads"], dim, case["block"])
    query = (1.5 * _normal(generator, sum(queries), case["q_heads"], dim, dtype=torch.float32)).to(dtype)
    # Every request's pages, in any order of the pool; entries behind its last page are left over from others.
    order = torch.randperm(total, device="cuda", generator=generator).to(torch.int32)
    table = _whole(generator, 0, total, case["requests"], max(pages), dtype=torch.int32)
    taken = 0
    for request, count in enumerate(pages):
        table[request, :count] = order[taken:taken + count]
        taken += count
    starts = torch.tensor([0, *queries], device="cuda").cumsum(0).to(torch.int32)
    return {**state, "kind": "attention", "query": query, "table": table, "page": page,
            "lengths": torch.tensor(keys, dtype=torch.int32, device="cuda"),
            "starts": None if case["queries"] == 1 else starts, "most_queries": max(queries), "most_keys": max(keys)}


# -- one pass ---------------------------------------------------------------


def run(state):
    return {"append": _run_append, "link": _run_link, "load": _run_load, "attention": _run_attention}[
        state["kind"]](state)


def _pool_of(state):
    return {name: state[name] for name in ("key_buffer", "value_buffer", "key_scales", "value_scales", "scale_block")}


def _split(state):
    q_width, kv_width = state["q_heads"] * state["dim"], state["kv_heads"] * state["dim"]
    return [part.unflatten(-1, (-1, state["dim"])) for part in
            state["projected"].split([q_width, kv_width, kv_width], dim=-1)]


def _run_append(state):
    query, key, value = _split(state)
    if own:
        from legolink_amd.quantized_pool import append_quantized_kv_inplace, load_quantized_kv

        rotated = append_quantized_kv_inplace(
            **_pool_of(state), destination_slots=state["slots"], query=query, key=key, value=value,
            positions=state["positions"], cos_sin_cache=state["table"], rotary_dim=state["rotary"],
            is_neox_style=state["neox"], query_norm_weight=state["query_norm"], key_norm_weight=state["key_norm"],
            norm_eps=NORM_EPS)
        return rotated, *load_quantized_kv(**_pool_of(state), dtype=state["dtype"])
    row = state["table"][state["positions"].long()].float()[:, None]
    cos, sin = row.chunk(2, dim=-1)
    rotated = _plain_turn(_plain_norm(query, state["query_norm"]), cos, sin, state["neox"]).to(query.dtype)
    keys = _plain_turn(_plain_norm(key, state["key_norm"]), cos, sin, state["neox"])
    slots = state["slots"].long()
    _plain_store(state["key_buffer"], state["key_scales"], state["scale_block"], slots, keys)
    _plain_store(state["value_buffer"], state["value_scales"], state["scale_block"], slots, value.float())
    return rotated, *_plain_values(state)


def _run_link(state):
    if own:
        from legolink_amd.quantized_pool import link_quantized_kv_inplace, load_quantized_kv

        link_quantized_kv_inplace(
            **_pool_of(state), source_slots=state["source"], destination_slots=state["slots"],
            local_positions=state["local"], global_positions=state["global"], cos_sin_cache=state["table"],
            rotary_dim=state["rotary"], is_neox_style=state["neox"], repair_mask=state["repair"])
        return load_quantized_kv(**_pool_of(state), dtype=state["dtype"])
    block, source, slots = state["scale_block"], state["source"].long(), state["slots"].long()
    cos_from, sin_from = state["table"][state["local"].long()].float()[:, None].chunk(2, dim=-1)
    cos_to, sin_to = state["table"][state["global"].long()].float()[:, None].chunk(2, dim=-1)
    cos, sin = cos_to * cos_from + sin_to * sin_from, sin_to * cos_from - cos_to * sin_from
    keys = _plain_turn(_plain_rows(state["key_buffer"], state["key_scales"], block, source), cos, sin, state["neox"])
    values = _plain_rows(state["value_buffer"], state["value_scales"], block, source)
    written = None if state["repair"] is None else ~state["repair"]
    _plain_store(state["key_buffer"], state["key_scales"], block, slots, keys, written)
    _plain_store(state["value_buffer"], state["value_scales"], block, slots, values, written)
    return _plain_values(state)


def _run_load(state):
    if own:
        from legolink_amd.quantized_pool import load_quantized_kv

        return load_quantized_kv(**_pool_of(state), slots=state["slots"], dtype=state["dtype"])
    block, slots = state["scale_block"], state["slots"].long()
    return (_plain_rows(state["key_buffer"], state["key_scales"], block, slots).to(state["dtype"]),
            _plain_rows(state["value_buffer"], state["value_scales"], block, slots).to(state["dtype"]))


def _plain_power(exponents):
    """2^exponents, exactly, by e8m0's bits."""

    return (exponents + 127).clamp(min=0).to(torch.uint8).view(torch.float8_e8m0fnu).float()


def _plain_rows(codes, scales, block, slots):
    return codes.view(torch.uint8)[slots].view(codes.dtype).float() * scales.float()[slots // block][..., None]


def _plain_values(state):
    """The whole pool as the values it stands for."""

    block = state["scale_block"]
    return [(state[codes].float().unflatten(0, (-1, block)) * state[scales].float()[:, None, :, None])
            .flatten(0, 1).to(state["dtype"])
            for codes, scales in (("key_buffer", "key_scales"), ("value_buffer", "value_scales"))]


def _plain_norm(rows, weight):
    out = rows.float()
    return out if weight is None else out * torch.rsqrt((out * out).mean(-1, keepdim=True) + NORM_EPS) * weight.float()


def _plain_turn(rows, cos, sin, neox):
    """Rows [tokens, heads, dim] whose first dims are turned by angles of these cos and sin [tokens, 1, pairs]."""

    half = cos.shape[-1]
    if neox:
        first, second = rows[..., :half], rows[..., half:2 * half]
        turned = torch.cat((first * cos - second * sin, second * cos + first * sin), dim=-1)
    else:
        first, second = rows[..., 0:2 * half:2], rows[..., 1:2 * half:2]
        turned = torch.stack((first * cos - second * sin, second * cos + first * sin), dim=-1).flatten(-2)
    return torch.cat((turned, rows[..., 2 * half:]), dim=-1)


def _plain_store(codes, scales, block, slots, rows, written=None):
    """Rows [tokens, heads, dim] to their slots.  A block's scale is the least
    that holds its new rows, and no less than it was unless every row of the
    block is written; the other rows are rounded to a scale that has grown."""

    magnitude, count = rows.abs().amax(-1), torch.ones_like(slots)
    if written is not None:
        magnitude, count = magnitude * written[:, None], count * written
    blocks, held = slots // block, scales.view(torch.uint8).int()
    most = torch.zeros(held.shape, device=codes.device).index_reduce_(0, blocks, magnitude, "amax")
    full = torch.zeros(held.shape[0], dtype=torch.int64, device=codes.device).index_add_(0, blocks, count) == block
    fraction, exponent = torch.frexp(most)  # most <= 448 2^e from e = exponent - 9 (+ 1 past 0.875) on
    needed = (exponent - 9 + (fraction > 0.875).int() + 127).clamp(0, 254) * (most > 0)
    grown = torch.where(full[:, None], needed, torch.maximum(held, needed))
    ratio = _plain_power(torch.clamp(held - grown, max=0))
    moved = (codes.float().unflatten(0, (-1, block)) * ratio[:, None, :, None]).flatten(0, 1).to(codes.dtype)
    new = (rows * _plain_power(127 - grown)[blocks][..., None]).clamp(-MOST_CODE, MOST_CODE).to(codes.dtype)
    if written is not None:
        new = torch.where(written[:, None, None], new.view(torch.uint8), moved.view(torch.uint8)[slots])
    codes.copy_(moved)
    codes.view(torch.uint8)[slots] = new.view(torch.uint8)
    scales.view(torch.uint8).copy_(grown)


def _run_attention(state):
    query, keys, values = state["query"], state["key_buffer"], state["value_buffer"]
    if own:
        from legolink_amd.quantized_pool import quantized_paged_attention

        return quantized_paged_attention(query, keys, values, state["key_scales"], state["value_scales"],
                                         state["table"], state["lengths"], scale_block=state["scale_block"],
                                         page_size=state["page"], query_starts=state["starts"])
    # Every request padded to the longest: its keys by its pages, its queries by their starts.
    page, most_keys, most_queries = state["page"], state["most_keys"], state["most_queries"]
    requests, (q_heads, dim), kv_heads = state["table"].shape[0], query.shape[1:], keys.shape[1]
    place = torch.arange(most_keys, device="cuda")
    slots = state["table"][:, place // page].long() * page + place % page  # [requests, keys]
    lengths = state["lengths"].long()
    if state["starts"] is None:
        starts, counts = torch.arange(requests, device="cuda"), torch.ones_like(lengths)
    else:
        starts = state["starts"][:-1].long()
        counts = state["starts"][1:].long() - starts
    offset = torch.arange(most_queries, device="cuda")
    valid = offset < counts[:, None]
    rows = torch.where(valid, starts[:, None] + offset, 0)  # [requests, queries]
    position = (lengths - counts)[:, None] + offset
    group = q_heads // kv_heads
    padded = query[rows].float().view(requests, most_queries, kv_heads, group, dim)
    padded = padded.permute(0, 2, 3, 1, 4).reshape(requests, kv_heads, group * most_queries, dim).contiguous()
    seen_keys = _plain_rows(keys, state["key_scales"], state["scale_block"], slots)
    seen_keys = seen_keys.permute(0, 2, 3, 1).contiguous()  # [requests, heads, dim, keys]
    scores = torch.matmul(padded, seen_keys).mul_(1.0 / math.sqrt(dim))
    del seen_keys
    hidden = place > position[..., None]  # [requests, queries, keys]
    scores.view(requests, kv_heads, group, most_queries, most_keys).masked_fill_(hidden[:, None, None], -math.inf)
    scores = scores.sub_(scores.amax(-1, keepdim=True)).exp_()
    sums = scores.sum(-1, keepdim=True)
    seen_values = _plain_rows(values, state["value_scales"], state["scale_block"], slots)
    seen_values.masked_fill_((place >= lengths[:, None])[..., None, None], 0.0)
    out = torch.matmul(scores, seen_values.permute(0, 2, 1, 3).contiguous()) / sums
    out = out.view(requests, kv_heads, group, most_queries, dim).permute(0, 3, 1, 2, 4)
    return out.reshape(requests, most_queries, q_heads, dim)[valid].to(query.dtype)


def work(case):
    kv_heads, dim, block = case["kv_heads"], case["dim"], case["block"]
    row = 2 * kv_heads * dim  # a token's codes
    if case["kind"] == "attention":
        queries, keys = _queries(case), _keys(case)
        pairs = sum(n * (k - n) + n * (n + 1) // 2 for n, k in zip(queries, keys))
        pages = sum(-(-count // case["page"]) for count in keys)
        return {"bytes": sum(keys) * row + sum(-(-count // block) for count in keys) * 2 * kv_heads
                + 2 * sum(queries) * case["q_heads"] * dim * 2 + 4 * (pages + 2 * case["requests"]),
                "flops": 4 * dim * case["q_heads"] * pairs}
    tokens, size, index = case["tokens"], SIZES[case["dtype"]], SIZES[case["index"]]
    if case["kind"] == "load":
        return {"bytes": tokens * (row + size * row + index) + -(-tokens // block) * 2 * kv_heads,
                "flops": tokens * row}
    if case["kind"] == "append":
        slots = (sum(-(-(case["page"] - 1 + count) // case["page"]) for count in _new_tokens(case)) + 2) * case["page"]
        turned, maps = case["q_heads"] + kv_heads, 2
        moved = tokens * (2 * case["q_heads"] * dim * size + row * size)  # queries both ways, keys and values
        flops = tokens * turned * (3 * case["rotary"] + (4 * dim if case["norm"] else 0))
    else:
        slots = (-(-case["cached"] // block) + -(-tokens // block)) * block
        turned, maps = kv_heads, 4
        moved = tokens * (row + (1 if case["repair"] else 0))
        flops = tokens * turned * 3 * case["rotary"]
    # The rows that are written, and the whole pool as the values it stands for.
    moved += tokens * row + slots * row * (1 + size)
    table = (maps // 2) * min(tokens, CONTEXT) * case["rotary"] * SIZES[case["table"]]
    return {"bytes": moved + table + tokens * maps * index, "flops": flops + slots * row}


# -- the same in 64 bits ----------------------------------------------------


def exact(case, seed):
    return {"append": _exact_append, "link": _exact_link, "load": _exact_load, "attention": _exact_attention}[
        case["kind"]](case, seed)


def _two_to(exponents):
    """2^exponents in 64 bits, exactly (a power function rounds, and a tie would fall elsewhere)."""

    return ((exponents.long() + 1023) << 52).view(torch.float64)


def _held(state):
    """The values of keys and of values [blocks, block, heads, dim], and their scales' exponents."""

    pools = []
    for codes, scales in ((state["key_buffer"], state["key_scales"]), (state["value_buffer"], state["value_scales"])):
        exponents = scales.view(torch.uint8).long() - 127
        values = codes.to(torch.float64).unflatten(0, (-1, state["scale_block"]))
        pools.append((values * _two_to(exponents)[:, None, :, None], exponents))
    return pools


def _to_grid(values, exponents):
    """Values rounded to even on e4m3's grid under scales 2^exponents."""

    scaled = values * _two_to(-exponents)
    steps = torch.frexp(scaled.abs())[1].clamp(min=-5) - 4  # four bits from the leading one on, none below 2^-9
    return torch.round(scaled * _two_to(-steps)) * _two_to(steps + exponents)


def _turned(rows, turn, neox):
    """Pairs of dims as complex numbers, multiplied by those of ``turn`` [tokens, pairs]."""

    half = turn.shape[-1]
    low = torch.arange(half, device="cuda") * (1 if neox else 2)
    high = low + (half if neox else 1)
    rows = rows.clone()
    pairs = torch.complex(rows[..., low].contiguous(), rows[..., high].contiguous()) * turn[:, None]
    rows[..., low], rows[..., high] = pairs.real, pairs.imag
    return rows


def _turn_at(state, positions):
    cos, sin = state["table"].double()[state[positions].long()].chunk(2, dim=-1)
    return torch.complex(cos.contiguous(), sin.contiguous())


def _stored(pool, exponents, slots, rows, dtype):
    """The pool [slots, heads, dim] once ``rows`` went to ``slots``."""

    block = pool.shape[1]
    blocks, inverse = torch.unique(slots // block, return_inverse=True)
    touched = torch.zeros(blocks.numel(), *pool.shape[1:], dtype=torch.float64, device="cuda")
    new = torch.zeros(touched.shape[:2], dtype=torch.bool, device="cuda")
    touched[inverse, slots % block], new[inverse, slots % block] = rows, True
    most = touched.abs().amax((1, 3))
    needed = torch.where(most > 0, torch.ceil(torch.log2(most / MOST_CODE)), -127.0).long().clamp(-127, 127)
    needed += (most > MOST_CODE * _two_to(needed)).long()
    needed -= ((most > 0) & (most <= MOST_CODE * _two_to(needed - 1))).long()
    grown = torch.where(new.all(1)[:, None], needed, torch.maximum(exponents[blocks], needed))
    touched = torch.where(new[..., None, None], touched, pool[blocks])
    pool = pool.clone()
    pool[blocks] = _to_grid(touched, grown[:, None, :, None])
    return pool.flatten(0, 1)


def _exact_append(case, seed):
    state = _prepare_append(case, seed)
    q_heads, kv_heads, dim = case["q_heads"], case["kv_heads"], case["dim"]
    rows = state["projected"].double().view(case["tokens"], q_heads + 2 * kv_heads, dim)
    turn = _turn_at(state, "positions")

    def headed(part, weight):
        if weight is not None:
            part = part / (part.pow(2).sum(-1, keepdim=True) / dim + NORM_EPS).sqrt() * weight.double()
        return _turned(part, turn, case["neox"])

    (keys, key_exponents), (values, value_exponents) = _held(state)
    slots = state["slots"].long()
    key_rows = headed(rows[:, q_heads:q_heads + kv_heads], state["key_norm"])
    return (headed(rows[:, :q_heads], state["query_norm"]),
            _stored(keys, key_exponents, slots, key_rows, state["dtype"]),
            _stored(values, value_exponents, slots, rows[:, q_heads + kv_heads:], state["dtype"]))


def _exact_link(case, seed):
    state = _prepare_link(case, seed)
    (keys, key_exponents), (values, value_exponents) = _held(state)
    # Turned back from where it was compiled, and on to where it goes.
    turn = _turn_at(state, "global") * _turn_at(state, "local").conj()
    source, slots = state["source"].long(), state["slots"].long()
    key_rows = _turned(keys.flatten(0, 1)[source], turn, case["neox"])
    value_rows = values.flatten(0, 1)[source]
    if state["repair"] is not None:
        kept = ~state["repair"]
        slots, key_rows, value_rows = slots[kept], key_rows[kept], value_rows[kept]
    return [_stored(keys, key_exponents, slots, key_rows, state["dtype"]),
            _stored(values, value_exponents, slots, value_rows, state["dtype"])]


def _exact_load(case, seed):
    state = _prepare_load(case, seed)
    (keys, _), (values, _) = _held(state)
    slots = state["slots"].long()
    return keys.flatten(0, 1)[slots], values.flatten(0, 1)[slots]


def _exact_attention(case, seed):
    state = _prepare_attention(case, seed)
    page, dim, block, group = case["page"], case["dim"], case["block"], case["q_heads"] // case["kv_heads"]
    query = state["query"].double()
    out = torch.empty_like(query)

    def rows_of(name, slots, head):
        exponents = state[name + "_scales"].view(torch.uint8).long()[slots // block, head] - 127
        return state[name + "_buffer"][:, head].contiguous().double()[slots] * _two_to(exponents)[:, None]

    begin = 0
    for request, (count, length) in enumerate(zip(_queries(case), _keys(case))):
        entries = state["table"][request, :-(-length // page)].long()
        slots = (entries[:, None] * page + torch.arange(page, device="cuda")).flatten()[:length]
        for head in range(case["kv_heads"]):
            key, value = rows_of("key", slots, head), rows_of("value", slots, head)
            heads = slice(head * group, (head + 1) * group)
            for first in range(0, count, 512):
                last = min(first + 512, count)
                part = query[begin + first:begin + last, heads].reshape(-1, dim)
                seen = length - count + last
                scores = part @ key[:seen].t() / math.sqrt(dim)
                at = torch.arange(length - count + first, seen, device="cuda").repeat_interleave(group)
                scores.masked_fill_(torch.arange(seen, device="cuda") > at[:, None], -math.inf)
                weights = torch.softmax(scores, dim=-1)
                out[begin + first:begin + last, heads] = (weights @ value[:seen]).view(-1, group, dim)
        begin += count
    return out
