"""Attention over quantised pages where rows of very different sizes meet, on the
GPU against float64: what is left of the small ones.

Tolerances are derived at each test; u is half a step of the type (eps / 2).
"""

from __future__ import annotations

import math

import _paged_plain as plain
import _quant_plain as qplain
import numpy as np
import pytest
import torch

import nitrix_amd as nx

from test_hip_quantized import DT, E24, _dev, _i32, _n64, _pool, _rand, _setup

pytestmark = pytest.mark.gpu


def _written_pool(dtype, k, v, bits, ps=16):
    """Pages that hold the tokens k, v (h, t, d) in order, as the framework
    writes them, with the table."""
    hk, t, d = k.shape
    p = -(-t // ps)
    pool = _pool(dtype, p, hk, ps, d, v.shape[2], bits)
    table = np.arange(p, dtype=np.int32)[None]
    nx.write_quantized_pages(*pool, k.to(dtype).to(_dev()), v.to(dtype).to(_dev()), _i32(table),
                             _i32([0]), _i32([0, t]), backend='hip')
    return pool, table


def _held(pool, bits):
    sc = _n64(pool[2])
    return [qplain.values(x.cpu().numpy(), sc, w, bits) for w, x in enumerate(pool[:2])]


def _off(out, want):
    """Largest distance of a head's output, relative to its norm."""
    got = _n64(out)
    return (np.linalg.norm(got - want, axis=-1) / np.linalg.norm(want, axis=-1)).max()


@pytest.mark.parametrize('dtype, bits, h, d, ps', [
    ('f16', 4, 4, 128, 16), ('f16', 8, 12, 128, 16), ('f16', 4, 2, 256, 12), ('bf16', 4, 4, 64, 16),
    ('bf16', 8, 2, 256, 16), ('f16', 8, 3, 80, 24),
])
@pytest.mark.parametrize('large', [0, 12])
def test_scores_are_float32_sums(dtype, bits, h, d, ps, large):
    """Scores of some 30, whose last digits count; and with an element of q 2^12
    times the others, where keys are zero.  q is exact and so are the products.  The
    sums lose 2^-24 of themselves, and pass 64 (8 bits: 1024) times q's partial
    sums, sqrt(d) of random sign: sqrt(d / 8 + 8) times that in all, of which eight
    times is allowed for, beside the output's own rounding u.  The large element's
    product is in three sums (q's, what the products' starts from, and its own
    group's), each off by half a last place of it."""
    dt, n, scale = DT[dtype], 400, 3.0
    g = torch.Generator().manual_seed(3)
    k, v = (torch.randn(1, n, d, generator=g) for _ in range(2))
    q = _rand((1, h, d), dt, 2)
    if large:
        k = k.abs()
        k[..., 5], q[..., 5] = 0, 2.0 ** large
    pool, table = _written_pool(dt, k, v, bits, ps)
    out = nx.quantized_paged_attention(q, *pool, _i32(table), _i32([n]), scale=scale, backend='hip')
    hk, hv = _held(pool, bits)
    want, _ = plain.attention(_n64(q), hk, hv, table, [n], scale)
    step = float(pool[2].float().nan_to_num()[..., 0].max()) * (64 if bits == 4 else 1024)
    lost = 8 * math.sqrt(d / 8 + 8) * math.sqrt(d) + (1.5 * 2.0 ** large if large else 0)
    assert _off(out, want) <= torch.finfo(dt).eps / 2 + lost * E24 * step * scale


@pytest.mark.parametrize('dtype', ['bf16', 'f32'])
def test_q_next_to_the_largest_number(dtype):
    """q of 2^126 and 2^127 with keys of 2^-126: scores of ordinary size."""
    dt, n, d = DT[dtype], 40, 8
    g = torch.Generator().manual_seed(3)
    k = (torch.randint(1, 8, (1, n, d), generator=g) - 4.0) * 2.0 ** -125
    v = torch.randn(1, n, d, generator=g)
    pool, table = _written_pool(dt, k, v, 8)
    q = (torch.randint(0, 2, (1, 2, d), generator=g) * 2.0 - 1) * 2.0 ** 126
    q[0, 1] *= 1.5
    q = q.to(dt).to(_dev())
    out = nx.quantized_paged_attention(q, *pool, _i32(table), _i32([n]), scale=0.125, backend='hip')
    hk, hv = _held(pool, 8)
    want, _ = plain.attention(_n64(q), hk, hv, table, [n], 0.125)
    # (scores below 2^4, off by 16 2^-24 of their terms; values below 4)
    u = torch.finfo(dt).eps / 2
    assert (np.abs(_n64(out) - want) <= u * np.abs(want) + 4 * 2.0 ** -15).all()
