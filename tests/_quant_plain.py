"""Plain forms of the quantised cache and of the rotary positions: loops over
tokens and heads, float64, whole quotients as fractions.  Used by the host and
GPU tests."""

from __future__ import annotations

from fractions import Fraction

import numpy as np
import torch


def quantise_row(x: torch.Tensor, bits: int):
    """Codes, scale and minimum of one row (1-d, on the host): the exact
    quotients rounded to the nearest, ties to even."""
    top = (1 << bits) - 1
    n = x.numel()
    if not torch.isfinite(x).all():
        return [0] * n, float('nan'), float('nan')
    lo, hi = x.min(), x.max()
    acc = torch.promote_types(x.dtype, torch.float32)
    s = ((hi.to(acc) - lo.to(acc)) * (1 / top)).to(x.dtype)
    if not torch.isfinite(s):
        return [0] * n, float('nan'), float('nan')
    if s == 0:
        return [0] * n, 0.0, float(lo)
    fs, fz = Fraction(float(s)), Fraction(float(lo))
    codes = [min(max(round((Fraction(float(e)) - fz) / fs), 0), top) for e in x]
    return codes, float(s), float(lo)


def unpack(pages: np.ndarray, bits: int) -> np.ndarray:
    """Codes as whole numbers, from bytes."""
    if bits == 8:
        return pages.astype(np.int64)
    out = np.empty((*pages.shape[:-1], 2 * pages.shape[-1]), np.int64)
    out[..., 0::2], out[..., 1::2] = pages % 16, pages // 16
    return out


def values(pages, scales, which, bits):
    """What the codes stand for, float64."""
    s, z = scales[..., 2 * which, None], scales[..., 2 * which + 1, None]
    return unpack(pages, bits) * s + z


def slots(table, starts, offsets, t, p, ps):
    """(token, page, slot) of every token that has a slot."""
    b, m = table.shape
    out = []
    for s in range(b):
        toks = [s] if offsets is None else range(max(int(offsets[s]), 0), min(int(offsets[s + 1]), t))
        for j in toks:
            pos = int(starts[s]) + (0 if offsets is None else j - int(offsets[s]))
            if 0 <= pos < m * ps and 0 <= table[s, pos // ps] < p:
                out.append((j, int(table[s, pos // ps]), pos % ps))
    return out


def rotate(x, positions, freq, interleaved, scale, inverse=False):
    """x [h, t, d] float64 turned by positions [t]; and per element what its
    terms add up to without signs (for error bounds)."""
    out, size = x.copy(), np.abs(x).copy()
    n = len(freq)
    ang = np.asarray(positions, np.float64)[:, None] * np.asarray(freq, np.float64)
    c, s = np.cos(ang) * scale, np.sin(ang) * scale * (-1 if inverse else 1)
    a, b = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if interleaved else (slice(0, n), slice(n, 2 * n))
    out[..., a] = x[..., a] * c - x[..., b] * s
    out[..., b] = x[..., b] * c + x[..., a] * s
    both = (np.abs(x[..., a]) + np.abs(x[..., b])) * abs(scale)
    size[..., a], size[..., b] = both, both
    return out, size
