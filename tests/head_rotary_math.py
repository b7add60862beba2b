"""Norms and rotation of heads in 64 bits, and how far a kernel may be off.

Written from the formulas: y = x / sqrt(mean(x^2) + eps) * w, then each rotary
pair turned by its angle.
"""

from __future__ import annotations

import torch


def turned(rows, positions, table, *, rotary, neox, weight=None, eps=1e-6):
    """(result, size) of rows [tokens, heads, dim] in float64 on the CPU; ``size``
    is the sum of the magnitudes that each result was added from."""

    x = rows.detach().cpu().double()
    if weight is not None:
        x = x / (x.pow(2).mean(-1, keepdim=True) + eps).sqrt() * weight.detach().cpu().double()
    at = table.detach().cpu().double()[positions.detach().cpu().long()][:, None]
    half = rotary // 2
    cos, sin = at[..., :half], at[..., half:rotary]
    low = torch.arange(half) if neox else 2 * torch.arange(half)
    high = low + (half if neox else 1)
    out, size = x.clone(), x.abs()
    a, b = x[..., low], x[..., high]
    out[..., low], out[..., high] = a * cos - b * sin, b * cos + a * sin
    size[..., low] = (a * cos).abs() + (b * sin).abs()
    size[..., high] = (b * cos).abs() + (a * sin).abs()
    return out, size


def allowed(want, size, dtype, dim):
    """A rounding to ``dtype`` (half a step, relative, or half the smallest
    subnormal) and the fp32 work before it, relative to ``size``: the two
    products and the sum of a pair (3 roundings), the norm's three products,
    square root and quotient by the count (2 units each at most), and half of
    the relative error of a sum of ``dim`` squares added up in any order (at most
    dim + 1 roundings), all of 2^-24."""

    info = torch.finfo(dtype)
    work = (3 + 8 + (dim + 1) / 2) * 2.0 ** -24
    return info.eps / 2 * (want.abs() + work * size) + work * size + info.smallest_normal * info.eps / 2
