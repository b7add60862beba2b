"""The 8-bit pool's format and what the calls write to it, on the CPU in 64 bits.

Written from the format: a value is its code (e4m3: sign, 4 bits of exponent with
bias 7, 3 of fraction, 0x7f NaN) times 2^(scale byte - 127).
"""

from __future__ import annotations

import numpy as np
import torch

_CODES = np.arange(127)
_SIZES = np.where(_CODES < 8, _CODES * 2.0 ** -9, (1 + _CODES % 8 / 8) * 2.0 ** (_CODES // 8 - 7.0))  # 0 .. 448
_MIDDLES = (_SIZES[1:] + _SIZES[:-1]) / 2
VALUES = np.concatenate((_SIZES, [np.nan], -_SIZES, [np.nan]))  # of the 256 codes


def encoded(values):
    """float64 -> codes, to nearest even; not finite: NaN with the sign."""

    size = np.abs(values)
    below = np.searchsorted(_MIDDLES, size, side="left")  # ties: the middle's lower neighbour
    tie = (below < 126) & (size == _MIDDLES[np.minimum(below, 125)])
    codes = np.where(tie & (below % 2 == 1), below + 1, below)
    codes = np.where(np.isfinite(values), codes, 127)
    return (codes + np.where(np.signbit(values), 128, 0)).astype(np.uint8)


def host(tensor):
    return tensor.detach().cpu().contiguous().view(torch.uint8).numpy().copy()


def values_of(codes, scales, block):
    """Codes [slots, heads, dim] and scale bytes [blocks, heads] as float64."""

    scale = np.where(scales == 255, np.nan, np.ldexp(1.0, scales.astype(int) - 127))
    return VALUES[codes] * np.repeat(scale, block, axis=0)[..., None]


def pool_values(buffer, scales, block):
    return torch.from_numpy(values_of(host(buffer), host(scales), block))


def least_byte(most):
    byte = 0
    while most > np.ldexp(448.0, byte - 127):
        byte += 1
    return byte


def stored(codes, scales, block, slots, rows, written):
    """The pool's (codes, scales) once ``rows`` [tokens, heads, dim] (float64) went
    to ``slots`` where ``written``."""

    codes, scales = codes.copy(), scales.copy()
    blocks = {}
    for t, slot in enumerate(slots):
        if written[t]:
            blocks.setdefault(slot // block, []).append(t)
    for b, tokens in blocks.items():
        offsets = [slots[t] % block for t in tokens]
        others = [o for o in range(block) if o not in offsets]
        for head in range(codes.shape[1]):
            new = rows[tokens, head]
            size = np.abs(new)
            need = least_byte(np.where(np.isfinite(size), size, 0.0).max())
            old = int(scales[b, head])
            byte = need if not others else max(old, need)
            scales[b, head] = byte
            codes[[b * block + o for o in offsets], head] = encoded(np.ldexp(new, 127 - byte))
            if byte > old:
                places = [b * block + o for o in others]
                codes[places, head] = encoded(np.ldexp(VALUES[codes[places, head]], old - byte))
    return codes, scales


def same_codes(got, want):
    """Equal codes; any NaN is as good as another."""

    return np.array_equal(np.where(got & 127 == 127, 127, got), np.where(want & 127 == 127, 127, want))


def turned_rows(rows, cos, sin, neox):
    """float64 rows [tokens, heads, dim] whose first pairs are turned, by cos and sin [tokens, 1, pairs]."""

    half = cos.shape[-1]
    low = np.arange(half) * (1 if neox else 2)
    high = low + (half if neox else 1)
    out = rows.copy()
    out[..., low] = rows[..., low] * cos - rows[..., high] * sin
    out[..., high] = rows[..., high] * cos + rows[..., low] * sin
    return out


def random_pool(slots, heads, dim, block, *, seed, device="cpu", low=110, high=135, empty=()):
    """Codes of every finite value and scales of many sizes; blocks of ``empty`` hold nothing."""

    generator = torch.Generator().manual_seed(seed)
    pool = {}
    for name in ("key", "value"):
        codes = torch.randint(0, 127, (slots, heads, dim), generator=generator, dtype=torch.uint8)
        codes |= torch.randint(0, 2, codes.shape, generator=generator, dtype=torch.uint8) << 7
        scales = torch.randint(low, high, (slots // block, heads), generator=generator, dtype=torch.uint8)
        for b in empty:
            codes[b * block:(b + 1) * block], scales[b] = 0, 0
        pool[f"{name}_buffer"] = codes.view(torch.float8_e4m3fn).to(device)
        pool[f"{name}_scales"] = scales.view(torch.float8_e8m0fnu).to(device)
    return pool
