"""Performance cases of the operators of a model's step over the paged pool.

Three kinds of call, each one layer's:

* ``rotate``: the norms of the queries and keys for each head and their
  position rotation, in one pass (``rotate_heads``);
* ``append``: the same for a step's new tokens, whose keys and values go to
  their slots of the pool on the way (``append_rotated_kv_inplace``);
* ``attention``: the attention of each request's new tokens over its pages of
  the pool (``paged_attention``), in its form for single tokens and for chunks.

Where ``own`` is false they are computed from elementary torch operations in
32 bits.  A case fixes everything that the amount of work depends on (how many
tokens each request has and adds); the seed draws the pages, the slots, the
positions and the values.
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
NORM_EPS = 1e-6
ROPE_THETA = 1_000_000.0
CONTEXT = 131072  # rows of the cos/sin table


def _rotate(**options):
    case = {"kind": "rotate", "tokens": 8192, "q_heads": 28, "kv_heads": 4, "dim": 128, "rotary": 128, "norm": True,
            "neox": True, "dtype": "bf16", "table": "fp32", "index": "int64"}
    return {**case, **options}


def _append(**options):
    case = {"kind": "append", "tokens": 64, "q_heads": 28, "kv_heads": 4, "dim": 128, "rotary": 128, "norm": False,
            "neox": True, "dtype": "bf16", "table": "fp32", "index": "int64"}
    return {**case, **options}


def _attention(**options):
    """``queries`` new tokens of each of ``requests`` requests (the shortest has
    ``least_queries``), over keys that count ``least_keys`` to ``keys``, their
    own among them."""

    case = {"kind": "attention", "requests": 1, "queries": 1, "least_queries": 1, "keys": 2048, "least_keys": 2048,
            "page": 1, "q_heads": 28, "kv_heads": 4, "dim": 128, "dtype": "bf16"}
    return {**case, **options}


def listed():
    return [
        # One new token's queries and keys, normed and rotated: the smallest call, where latency is the cost.
        _rotate(name="rotate_one_token", tokens=1),
        # A long prompt's, of a model with many heads.
        _rotate(name="rotate_8k_tokens", q_heads=64, kv_heads=8),
        # An odd number of tokens of a small model that rotates half of its dims and has no norms.
        _rotate(name="rotate_half_rotary", tokens=1237, q_heads=14, kv_heads=2, dim=64, rotary=32, norm=False,
                dtype="fp16", table="bf16", index="int32"),
        # A decode step of 64 requests: each one's new key and value to its slot.
        _append(name="append_64_tokens"),
        # A linked request's tail, prefilled in one chunk.
        _append(name="append_16k_tokens", tokens=16384, norm=True),
        # An odd chunk of a model with wide heads and neighbouring pairs.
        _append(name="append_wide_heads", tokens=2011, q_heads=16, kv_heads=2, dim=256, rotary=256, neox=False,
                dtype="fp16", index="int32"),
        # The next token of a short chat (c1's length): the latency of one layer's attention.
        _attention(name="decode_2k_keys"),
        # The next token over the longest context.
        _attention(name="decode_131k_keys", keys=131072, least_keys=131072),
        # A serving batch of uneven requests in pages of 16.
        _attention(name="decode_batch_of_64", requests=64, keys=32768, least_keys=500, page=16, q_heads=64,
                   kv_heads=8),
        # A chunk of 2,048 new tokens behind a linked 30k-token context (c2's length).
        _attention(name="chunk_behind_32k_keys", queries=2048, least_queries=2048, keys=32768, least_keys=32768),
        # Short chunks of several requests of a small model, uneven on both sides.
        _attention(name="chunks_of_6", requests=6, queries=701, least_queries=5, keys=9000, least_keys=300, page=16,
                   q_heads=14, kv_heads=2, dim=64, dtype="fp16"),
        # A whole prompt of a model with wide heads, nothing cached before it.
        _attention(name="prompt_wide_heads", queries=4099, least_queries=4099, keys=4099, least_keys=4099, page=64,
                   q_heads=16, kv_heads=2, dim=256),
    ]


# What a drawn case may have at most, so that it costs no more than the listed
# ones: bytes of the pool's rows, multiplications, and values of the plain
# form's padded scores and keys.
_MOST_BYTES = 64 * 32768 * 2 * 8 * 128 * 2 // 4
_MOST_FLOPS = 4 * 128 * 28 * 2048 * 30000
_MOST_SCORES = 2048 * 28 * 32768
_MOST_PADDED = 64 * 32768 * 8 * 128

_HEADS = [(28, 4), (28, 4), (64, 8), (14, 2), (7, 1), (10, 10), (16, 2), (32, 1)]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["rotate", "append", "attention", "attention", "attention"])
    while True:
        q_heads, kv_heads = rng.choice(_HEADS)
        dtype = rng.choice(["bf16", "bf16", "fp16"])
        if kind in ("rotate", "append"):
            dim, rotary = rng.choice([(128, 128), (128, 64), (64, 64), (64, 32), (256, 256), (80, 80), (112, 32)])
            make = _rotate if kind == "rotate" else _append
            case = make(tokens=_log(rng, 1, 16384), q_heads=q_heads, kv_heads=kv_heads, dim=dim, rotary=rotary,
                        norm=rng.random() < 0.6, neox=rng.random() < 0.8, dtype=dtype,
                        table=rng.choice(["fp32", "fp32", "bf16", "fp16"]), index=rng.choice(["int64", "int32"]))
            if work(case)["bytes"] <= 1.2e9:
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
                          least_keys=min(least_keys, keys), page=rng.choice([1, 1, 16, 48, 64, 128]),
                          q_heads=q_heads, kv_heads=kv_heads, dim=rng.choice([64, 128, 128, 256]), dtype=dtype)
        cost = work(case)
        if (cost["bytes"] <= _MOST_BYTES and cost["flops"] <= _MOST_FLOPS
                and requests * queries * q_heads * keys <= _MOST_SCORES
                and requests * keys * kv_heads * case["dim"] <= _MOST_PADDED):
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


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _normal(generator, *shape, dtype):
    return torch.randn(*shape, dtype=dtype, device="cuda", generator=generator)


@functools.lru_cache(maxsize=8)
def _table(rotary, dtype):
    """The model's cos/sin table, built once per program: cos in the first half
    of a row, sin in the second, from angles in 64 bits."""

    frequencies = ROPE_THETA ** (-torch.arange(0, rotary, 2, dtype=torch.float64, device="cuda") / rotary)
    angles = torch.arange(CONTEXT, dtype=torch.float64, device="cuda")[:, None] * frequencies
    return torch.cat((angles.cos(), angles.sin()), dim=-1).to(DTYPES[dtype])


def prepare(case, seed):
    return _prepare_attention(case, seed) if case["kind"] == "attention" else _prepare_heads(case, seed)


def _prepare_heads(case, seed):
    generator = _generator(seed)
    tokens, dim, dtype = case["tokens"], case["dim"], DTYPES[case["dtype"]]
    heads = case["q_heads"] + 2 * case["kv_heads"]
    # The model's fused projection of a step's tokens; channels of different scale.
    projected = _normal(generator, tokens, heads * dim, dtype=dtype)
    projected *= torch.linspace(0.25, 4.0, heads * dim, device="cuda").to(dtype)
    index = DTYPES[case["index"]]
    state = {"kind": case["kind"], "projected": projected, "q_heads": case["q_heads"], "kv_heads": case["kv_heads"],
             "dim": dim, "rotary": case["rotary"], "neox": case["neox"], "query_norm": None, "key_norm": None,
             "table": _table(case["rotary"], case["table"]),
             # Decode steps of many requests and chunks alike: positions anywhere in the context.
             "positions": torch.randint(CONTEXT, (tokens,), device="cuda", generator=generator).to(index)}
    if case["norm"]:
        state["query_norm"] = (1.0 + 0.3 * _normal(generator, dim, dtype=torch.float32)).to(dtype)
        state["key_norm"] = (1.0 + 0.3 * _normal(generator, dim, dtype=torch.float32)).to(dtype)
    if case["kind"] == "append":
        slots = max(4096, 2 * tokens + 7)
        state["key_buffer"] = _normal(generator, slots, case["kv_heads"], dim, dtype=dtype)
        state["value_buffer"] = _normal(generator, slots, case["kv_heads"], dim, dtype=dtype)
        state["slots"] = torch.randperm(slots, device="cuda", generator=generator)[:tokens].to(index)
    return state


def _prepare_attention(case, seed):
    generator = _generator(seed)
    dtype, page, dim = DTYPES[case["dtype"]], case["page"], case["dim"]
    queries, keys = _queries(case), _keys(case)
    pages = [-(-count // page) for count in keys]
    total = sum(pages) + max(8, sum(pages) // 16)
    slots = total * page
    key_buffer = _normal(generator, slots, case["kv_heads"], dim, dtype=dtype)
    value_buffer = _normal(generator, slots, case["kv_heads"], dim, dtype=dtype)
    query = (1.5 * _normal(generator, sum(queries), case["q_heads"], dim, dtype=torch.float32)).to(dtype)
    # Every request's pages, in any order of the pool; entries behind its last page are left over from others.
    order = torch.randperm(total, device="cuda", generator=generator).to(torch.int32)
    table = torch.randint(total, (case["requests"], max(pages)), device="cuda", generator=generator,
                          dtype=torch.int32)
    taken = 0
    for request, count in enumerate(pages):
        table[request, :count] = order[taken:taken + count]
        taken += count
    starts = torch.tensor([0, *queries], device="cuda").cumsum(0).to(torch.int32)
    return {"kind": "attention", "query": query, "key_buffer": key_buffer, "value_buffer": value_buffer,
            "table": table, "page": page, "lengths": torch.tensor(keys, dtype=torch.int32, device="cuda"),
            "starts": None if case["queries"] == 1 else starts, "most_queries": max(queries),
            "most_keys": max(keys)}


def run(state):
    if state["kind"] == "attention":
        return _run_attention(state)
    q_width, kv_width = state["q_heads"] * state["dim"], state["kv_heads"] * state["dim"]
    query, key, value = (part.unflatten(-1, (-1, state["dim"])) for part in
                         state["projected"].split([q_width, kv_width, kv_width], dim=-1))
    if own:
        from legolink_amd.head_rotary import append_rotated_kv_inplace, rotate_heads

        options = dict(positions=state["positions"], cos_sin_cache=state["table"], rotary_dim=state["rotary"],
                       is_neox_style=state["neox"], query_norm_weight=state["query_norm"],
                       key_norm_weight=state["key_norm"], norm_eps=NORM_EPS)
        if state["kind"] == "rotate":
            return rotate_heads(query, key, **options)
        rotated = append_rotated_kv_inplace(key_buffer=state["key_buffer"], value_buffer=state["value_buffer"],
                                            destination_slots=state["slots"], query=query, key=key, value=value,
                                            **options)
        return rotated, state["key_buffer"], state["value_buffer"]
    row = state["table"][state["positions"].long()].float()[:, None]
    rotated = _plain_heads(query, state["query_norm"], row, state["rotary"], state["neox"])
    keys = _plain_heads(key, state["key_norm"], row, state["rotary"], state["neox"])
    if state["kind"] == "rotate":
        return rotated, keys
    slots = state["slots"].long()
    state["key_buffer"][slots] = keys
    state["value_buffer"][slots] = value
    return rotated, state["key_buffer"], state["value_buffer"]


def _plain_heads(rows, weight, table, rotary, neox):
    """Rows [tokens, heads, dim] normed by their head and turned by the table's rows."""

    out = rows.float()
    if weight is not None:
        out = out * torch.rsqrt((out * out).mean(-1, keepdim=True) + NORM_EPS) * weight.float()
    half = rotary // 2
    cos, sin = table[..., :half], table[..., half:]
    if neox:
        first, second = out[..., :half], out[..., half:rotary]
        turned = torch.cat((first * cos - second * sin, second * cos + first * sin), dim=-1)
    else:
        first, second = out[..., 0:rotary:2], out[..., 1:rotary:2]
        turned = torch.stack((first * cos - second * sin, second * cos + first * sin), dim=-1).flatten(-2)
    return torch.cat((turned, out[..., rotary:]), dim=-1).to(rows.dtype)


def _run_attention(state):
    query, keys, values = state["query"], state["key_buffer"], state["value_buffer"]
    if own:
        from legolink_amd.paged_attention import paged_attention

        return paged_attention(query, keys, values, state["table"], state["lengths"], page_size=state["page"],
                               query_starts=state["starts"])
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
    seen_keys = keys[slots].float().permute(0, 2, 3, 1).contiguous()  # [requests, heads, dim, keys]
    scores = torch.matmul(padded, seen_keys).mul_(1.0 / math.sqrt(dim))
    del seen_keys
    hidden = place > position[..., None]  # [requests, queries, keys]
    scores.view(requests, kv_heads, group, most_queries, most_keys).masked_fill_(hidden[:, None, None], -math.inf)
    scores = scores.sub_(scores.amax(-1, keepdim=True)).exp_()
    sums = scores.sum(-1, keepdim=True)
    seen_values = values[slots].float().masked_fill_((place >= lengths[:, None])[..., None, None], 0.0)
    out = torch.matmul(scores, seen_values.permute(0, 2, 1, 3).contiguous()) / sums
    out = out.view(requests, kv_heads, group, most_queries, dim).permute(0, 3, 1, 2, 4)
    return out.reshape(requests, most_queries, q_heads, dim)[valid].to(query.dtype)


def work(case):
    size, q_heads, kv_heads, dim = 2, case["q_heads"], case["kv_heads"], case["dim"]
    if case["kind"] == "attention":
        queries, keys = _queries(case), _keys(case)
        pairs = sum(n * (k - n) + n * (n + 1) // 2 for n, k in zip(queries, keys))
        pages = sum(-(-count // case["page"]) for count in keys)
        return {"bytes": sum(keys) * 2 * kv_heads * dim * size + 2 * sum(queries) * q_heads * dim * size
                + 4 * (pages + 2 * case["requests"]),
                "flops": 4 * dim * q_heads * pairs}
    index = 4 if case["index"] == "int32" else 8
    tokens, turned = case["tokens"], q_heads + kv_heads
    moved = 2 * tokens * turned * dim * size
    table = min(tokens, CONTEXT) * case["rotary"] * (4 if case["table"] == "fp32" else 2)
    flops = tokens * turned * (3 * case["rotary"] + (4 * dim if case["norm"] else 0))
    if case["kind"] == "append":
        moved += 2 * tokens * kv_heads * dim * size + tokens * index
    return {"bytes": moved + table + tokens * index + (2 * dim * size if case["norm"] else 0), "flops": flops}


# -- the same in 64 bits ----------------------------------------------------


def exact(case, seed):
    return _exact_attention(case, seed) if case["kind"] == "attention" else _exact_heads(case, seed)


def _exact_heads(case, seed):
    state = _prepare_heads(case, seed)
    q_heads, kv_heads, dim, half = case["q_heads"], case["kv_heads"], case["dim"], case["rotary"] // 2
    rows = state["projected"].double().view(case["tokens"], q_heads + 2 * kv_heads, dim)
    # A pair of dims as one complex number, multiplied by exp(i angle) of the table.
    at = state["table"].double()[state["positions"].long()]
    turn = torch.complex(at[:, :half].contiguous(), at[:, half:].contiguous())[:, None]
    low = torch.arange(half, device="cuda") * (1 if case["neox"] else 2)
    high = low + (half if case["neox"] else 1)

    def turned(part, weight):
        part = part.clone()
        if weight is not None:
            part = part / (part.pow(2).sum(-1, keepdim=True) / dim + NORM_EPS).sqrt() * weight.double()
        pairs = torch.complex(part[..., low].contiguous(), part[..., high].contiguous()) * turn
        part[..., low], part[..., high] = pairs.real, pairs.imag
        return part

    query = turned(rows[:, :q_heads], state["query_norm"])
    key = turned(rows[:, q_heads:q_heads + kv_heads], state["key_norm"])
    if case["kind"] == "rotate":
        return query, key
    slots = state["slots"].long()
    key_buffer, value_buffer = state["key_buffer"].double(), state["value_buffer"].double()
    key_buffer.index_copy_(0, slots, key)
    value_buffer.index_copy_(0, slots, rows[:, q_heads + kv_heads:].contiguous())
    return query, key_buffer, value_buffer


def _exact_attention(case, seed):
    state = _prepare_attention(case, seed)
    page, dim, group = case["page"], case["dim"], case["q_heads"] // case["kv_heads"]
    query = state["query"].double()
    out = torch.empty_like(query)
    begin = 0
    for request, (count, length) in enumerate(zip(_queries(case), _keys(case))):
        entries = state["table"][request, :-(-length // page)].long()
        slots = (entries[:, None] * page + torch.arange(page, device="cuda")).flatten()[:length]
        for head in range(case["kv_heads"]):
            key, value = state["key_buffer"][slots, head].double(), state["value_buffer"][slots, head].double()
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
