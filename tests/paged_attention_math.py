"""Attention over pages in 64 bits on the CPU, and how far a kernel may be off."""

from __future__ import annotations

import math

import torch


def slots_of(table_row, length, page):
    """(slots, valid) of a request's keys; a page entry may be outside the pool."""

    place = torch.arange(length)
    entries = table_row.cpu().long()[place // page]
    return entries * page + place % page, entries


def attend(query, keys, values, table, lengths, starts, *, page, scale=None):
    """(result, size, weights) in float64: ``size`` is the weighted sum of |values|,
    ``weights`` the largest sum |q k| scale of a query's scores.  ``starts`` None: one
    query a request.  Rows of no request are NaN."""

    q, k, v = query.cpu().double(), keys.cpu().double(), values.cpu().double()
    dim, group = q.shape[2], q.shape[1] // k.shape[1]
    scale = 1 / math.sqrt(dim) if scale is None else scale
    pages = k.shape[0] // page
    out = torch.full_like(q, math.nan)
    size, reach = torch.zeros_like(q), torch.zeros(q.shape[:2], dtype=torch.float64)
    starts = list(range(len(lengths) + 1)) if starts is None else [int(s) for s in starts]
    for request, length in enumerate(int(n) for n in lengths):
        begin, count = starts[request], starts[request + 1] - starts[request]
        if count <= 0:
            continue
        slots, entries = slots_of(table[request], length, page)
        there = (entries >= 0) & (entries < pages)
        safe = torch.where(there, slots, 0)
        seen = there & (torch.arange(length) <= torch.arange(length - count, length)[:, None])  # [queries, keys]
        for head in range(k.shape[1]):
            heads = slice(head * group, (head + 1) * group)
            part = q[begin:begin + count, heads]  # [queries, group, dim]
            key, value = k[safe, head], v[safe, head]
            scores = torch.einsum("qgd,kd->qgk", part, key) * scale
            shown = seen[:, None].expand_as(scores)
            scores = torch.where(shown, scores, -math.inf)
            top = scores.amax(-1, keepdim=True) if length else torch.zeros(count, group, 1, dtype=torch.float64)
            weights = torch.where(shown, (scores - torch.where(top == -math.inf, 0.0, top)).exp(), 0.0)
            total = weights.sum(-1, keepdim=True)
            weights = weights / torch.where(total == 0, 1.0, total)
            # Unseen values do not count, whatever they hold: only seen rows are multiplied.
            alone = bool(torch.isfinite(value).all())
            if alone:
                out[begin:begin + count, heads] = torch.einsum("qgk,kd->qgd", weights, value)
                size[begin:begin + count, heads] = torch.einsum("qgk,kd->qgd", weights, value.abs())
            else:
                for i in range(count):
                    rows = seen[i]
                    out[begin + i, heads] = weights[i][:, rows] @ value[rows]
                    size[begin + i, heads] = weights[i][:, rows] @ value[rows].abs()
            magnitude = torch.einsum("qgd,kd->qgk", part.abs(), key.abs()) * scale
            if length:
                reach[begin:begin + count, heads] = torch.where(shown, magnitude, 0.0).amax(-1)
    return out, size, reach


def allowed(want, size, reach, dtype, longest, value_most):
    """The sum over j of p_j v_j over that of p_j, relative to ``size`` + |want|:
    half a step of the KV type for each weight; the scores' fp32 sums of ``dim``
    products (dim + 3 roundings of 2^-24 of ``reach``, as an error of the
    exponent) and exp2 with its argument (2^-20 of a weight for exponents below
    16, which hold all that counts); and fp32 sums over the keys (a rounding of
    2^-24 each).  Then the output's rounding.  Weights below fp16's normal range
    are off by 2^-25 of the largest weight at most, which is one or more."""

    info = torch.finfo(dtype)
    dim = want.shape[-1]
    relative = info.eps / 2 + (dim + 3) * 2.0 ** -24 * reach[..., None] + 2.0 ** -20 + (longest + 64) * 2.0 ** -24
    bound = relative * (size + want.abs()) + info.eps / 2 * want.abs() + info.smallest_normal * info.eps / 2
    if dtype == torch.float16:
        bound = bound + longest * 2.0 ** -25 * value_most
    return bound * (1 + 2.0 ** -6)  # products of the above
