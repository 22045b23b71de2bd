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


@pytest.mark.parametrize('dtype', ['bf16', 'f32'])
@pytest.mark.parametrize('size', [1e20, 3e28])
def test_constant_rows_beside_one_of_a_tiny_scale(dtype, size):
    """199 rows of one value (scale 0) and one that is 1e40 times smaller: the sum of
    the constant rows is no weight times a power that the tiny scale asks for.  The
    output is the values' mean but for the scores' roundings, which leave the
    weights' sum what they are: 200 steps of 2^-24 each way and the type's."""
    t, d = 200, 64
    v = torch.full((1, t, d), size)
    v[0, 77] = torch.linspace(0, 1e-19, d)
    k = torch.randn(1, t, d, generator=torch.Generator().manual_seed(1))
    pool, table = _written_pool(DT[dtype], k, v, 4)
    q = _rand((1, 2, d), DT[dtype], 2)
    out = nx.quantized_paged_attention(q, *pool, _i32(table), _i32([t]), backend='hip')
    hk, hv = _held(pool, 4)
    want, rows = plain.attention(_n64(q), hk, hv, table, [t], 0.125)
    # (the tiny row's weight is off by its score's roundings, 2^-14 or less of it)
    u = torch.finfo(DT[dtype]).eps / 2
    assert (np.abs(_n64(out) - want) <= np.abs(want) * (u + 400 * E24 + 2.0 ** -14 / 4)).all()


def _float32_pool(lens, hk, d, bits, sizes):
    """As rows of random values times ``sizes`` (lengths' sum) give."""
    pool, table = _setup(torch.float32, lens, hk, d, d, 16, bits)
    x = torch.randn(*pool[2].shape[:3], 2, d, generator=torch.Generator().manual_seed(8))
    x[..., 1, :] *= sizes
    top = (1 << bits) - 1
    lo, hi = x.amin(-1), x.amax(-1)
    pool[2][..., 0::2] = ((hi - lo) / top).to(pool[2])
    pool[2][..., 1::2] = lo.to(pool[2])
    codes = ((x - lo[..., None]) / (hi - lo)[..., None] * top).round().to(torch.uint8)
    for i in range(2):
        c = codes[..., i, :]
        pool[i].copy_(c if bits == 8 else c[..., ::2] | c[..., 1::2] << 4)
    return pool, table


def _float32_off(pool, table, q, lens, bits):
    out = nx.quantized_paged_attention(q, *pool, _i32(table), _i32(lens), backend='hip')
    k, v = _held(pool, bits)
    want, _ = plain.attention(_n64(q), k, v, table, lens, 1 / math.sqrt(q.shape[2]))
    return max(_off(out[i], want[i]) for i in range(len(lens)))


@pytest.mark.parametrize('bits, d', [(4, 64), (8, 64), (8, 128), (4, 256), (8, 32)])
@pytest.mark.parametrize('ratio', [32, 1024, 2.0 ** 20])
def test_float32_beside_large_values_of_no_weight(bits, d, ratio):
    """A few value rows ``ratio`` times larger than the rest, early in the sequence, at
    scores that leave them no weight: the others keep their digits.  The bound is that
    of ``test_float32_keeps_its_digits``: (12 d / 128) 2^-22 + 2^-20 + 2^-21 of the
    norm, for the scores', the exponentials' and the sums' roundings."""
    lens, hk = [500, 1300], 2
    held, table = _setup(torch.float32, lens, hk, d, d, 16, bits)
    sizes = torch.ones(held[2].shape[0], hk, 16, 1)
    big = [(int(row[0]), s) for row in table for s in (1, 2, 7)]
    for e, s in big:
        sizes[e, :, s] = ratio
    pool, table = _float32_pool(lens, hk, d, bits, sizes)
    for e, s in big:  # keys of one value: q is positive, so that their scores are -100 or less
        pool[2][e, :, s, 0], pool[2][e, :, s, 1] = 0, -16
    q = _rand((2, 2 * hk, d), torch.float32, 5).abs()
    assert float(16 * q.sum(-1).min() / math.sqrt(d)) > 50
    off = _float32_off(pool, table, q, lens, bits)
    assert off <= (12 * d / 128) * 2.0 ** -22 + 2.0 ** -20 + 2.0 ** -21, off


@pytest.mark.parametrize('bits, d', [(4, 64), (8, 128)])
@pytest.mark.parametrize('own', [1.0, 2.0 ** -10])
def test_float32_tail_of_one_large_score(bits, d, own):
    """One token of most of the weight and 20000 that share 2^-6 of it, all of one
    value: their sum keeps its digits though each is 2^-20 of the largest; also where
    the token's own row is 2^-10 as large, so that the tail is what the output is made
    of."""
    n, hk = 20000, 1
    held, table = _setup(torch.float32, [n], hk, d, d, 16, bits)
    sizes = torch.ones(held[2].shape[0], hk, 16, 1)
    first = (int(table[0, 0]), 3)
    sizes[first[0], :, first[1]] = own
    pool, table = _float32_pool([n], hk, d, bits, sizes)
    # (keys of one value each: scores of 0 and of ln(2^20))
    pool[2][..., :2] = torch.where(torch.isnan(pool[2][..., :2]), math.nan, 0)
    q = _rand((1, 2, d), torch.float32, 5).abs()
    q *= math.sqrt(d) / q.sum(-1, keepdim=True)
    pool[2][first[0], :, first[1], 1] = 20 * math.log(2)
    # every token of the tail has the value of the first
    row, one = (int(table[0, 0]), 0, 0), (first[0], 0, first[1])
    tail = ~torch.isnan(pool[2][..., 0])
    tail[one] = False
    pool[1][tail] = pool[1][row].clone()
    pool[2][..., 2:][tail] = pool[2][row][2:].clone()
    off = _float32_off(pool, table, q, [n], bits)
    # (the sums of 20000 equal weights go one way: 157 steps of a wave and the join's)
    assert off <= (12 * d / 128) * 2.0 ** -22 + 2.0 ** -20 + 2.0 ** -21 + 180 * E24, off


@pytest.mark.parametrize('dtype, bits, h, d', [
    ('bf16', 4, 4, 64), ('f16', 4, 4, 128), ('bf16', 8, 12, 128), ('f16', 8, 2, 256),
    ('bf16', 4, 2, 40),
])
@pytest.mark.parametrize('ratio', [2.0 ** 6, 2.0 ** 12])
def test_16_bits_beside_large_values_of_no_weight(dtype, bits, h, d, ratio):
    """As in float32: rows 2^12 times larger (2^24 in bfloat16) at no weight.  Per element
    the output is off by u of itself and, of the values' sizes w |v|, by the scores'
    roundings (q within 2^-22 of its largest element: the codes' sum times that, d + 8
    steps of 2^-24 of a score's terms) and 2^-21 for the weights."""
    ratio = ratio ** 2 if dtype == 'bf16' else ratio
    dt, n = DT[dtype], 700
    g = torch.Generator().manual_seed(3)
    k, v = (torch.randn(1, n, d, generator=g) for _ in range(2))
    for j in (0, 3, 200):
        k[0, j] = -16
        v[0, j] *= ratio
    pool, table = _written_pool(dt, k, v, bits)
    q = _rand((1, h, d), dt, 2).abs()
    out = nx.quantized_paged_attention(q, *pool, _i32(table), _i32([n]), backend='hip')
    hk, hv = _held(pool, bits)
    want, rows = plain.attention(_n64(q), hk, hv, table, [n], 1 / math.sqrt(d))
    kf, vf = (x[:, 0].reshape(-1, d)[:n] for x in (hk, hv))
    sc = _n64(pool[2])[:, 0].reshape(-1, 4)[:n]
    qn = _n64(q)[0]
    u = torch.finfo(dt).eps / 2
    tiny = 4 * (2.0 ** -24 if dt == torch.float16 else float(torch.finfo(dt).tiny))
    for i in range(h):
        w = rows[0, i][0]
        size = np.abs(kf) + 2 * np.abs(sc[:, 1:2])
        es = ((d + 8) * E24 * (size @ np.abs(qn[i])) + 2.0 ** -22 * np.abs(qn[i]).max() *
              size.sum(-1)) / math.sqrt(d)
        rel = es + (w @ es) + 2.0 ** -21
        tol = (w * rel) @ (np.abs(vf) + 2 * np.abs(sc[:, 3:])) + u * np.abs(want[0, i])
        assert (np.abs(_n64(out)[0, i] - want[0, i]) <= tol + tiny).all(), (
            i, (np.abs(_n64(out)[0, i] - want[0, i]) / (tol + tiny)).max())


@pytest.mark.parametrize('dtype, bits, h', [
    ('bf16', 4, 4), ('f16', 4, 4), ('f32', 4, 4), ('bf16', 8, 12), ('f16', 8, 1), ('f32', 8, 12),
])
def test_rows_of_every_size(dtype, bits, h):
    """Value rows times powers of two over most of the type's range, at scores of some
    3, so that a few rows make the output.  Per element: the weights within 2^-19 (a
    score's and its exponential's roundings) of what they are, of the values' sizes w
    |v|, the sums 2^-20 of the largest w s' times the codes, and u of the output."""
    dt, n, d = DT[dtype], 500, 64
    g = torch.Generator().manual_seed(7)
    k, v = (torch.randn(1, n, d, generator=g) for _ in range(2))
    span = 9 if dtype == 'f16' else 80
    v *= 2.0 ** torch.randint(-span, span + 1, (1, n, 1), generator=g)
    pool, table = _written_pool(dt, k, v, bits)
    q = _rand((1, h, d), dt, 2)
    out = nx.quantized_paged_attention(q, *pool, _i32(table), _i32([n]), backend='hip')
    hk, hv = _held(pool, bits)
    want, rows = plain.attention(_n64(q), hk, hv, table, [n], 0.125)
    vf, sc = hv[:, 0].reshape(-1, d)[:n], _n64(pool[2])[:, 0].reshape(-1, 4)[:n]
    u = torch.finfo(dt).eps / 2
    for i in range(h):
        w = rows[0, i][0]
        tol = 2.0 ** -19 * (w @ (np.abs(vf) + 2 * np.abs(sc[:, 3:]))) + u * np.abs(want[0, i])
        tol += 2.0 ** -20 * (w * sc[:, 2]).max() * (15 if bits == 4 else 255) + 2.0 ** -24 * (span == 9)
        assert (np.abs(_n64(out)[0, i] - want[0, i]) <= tol).all(), (
            i, (np.abs(_n64(out)[0, i] - want[0, i]) / tol).max())


@pytest.mark.parametrize('dtype', ['bf16', 'f16', 'f32'])
@pytest.mark.parametrize('step', [0.75, 40.0, -40.0])
def test_scores_that_climb(dtype, step):
    """Scores that grow (fall) by ``step`` a token, over hundreds of powers of two, with
    constant rows (scale 0) among ordinary ones: the last (first) tokens alone are left.
    Scores are one product, exact but for 2^-22 of itself."""
    dt, n, d = DT[dtype], 300, 64
    g = torch.Generator().manual_seed(7)
    v = torch.randn(1, n, d, generator=g)
    v[0, ::3] = 2.5
    v[0, n - 8:n - 2] = -1.5
    k = (torch.arange(n) * step / 8)[None, :, None].expand(1, n, d)
    pool, table = _written_pool(dt, k, v, 4)
    q = torch.full((1, 3, d), 1.0, dtype=dt, device=_dev())
    out = nx.quantized_paged_attention(q, *pool, _i32(table), _i32([n]), backend='hip')
    hk, hv = _held(pool, 4)
    want, _ = plain.attention(_n64(q), hk, hv, table, [n], 0.125)
    # (weights of tokens with the largest scores, off by those scores' 2^-22)
    off = 2.0 ** -22 * n * abs(step) * 2 + 2.0 ** -19
    assert np.abs(_n64(out) - want).max() <= (off + torch.finfo(dt).eps / 2) * 4


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


@pytest.mark.parametrize('dtype, bits, h', [('bf16', 4, 1), ('f16', 4, 1), ('bf16', 8, 1), ('f16', 8, 1),
                                            ('bf16', 4, 12)])
def test_long_even_rows_nearly_cancel(dtype, bits, h):
    """65536 tokens of equal weight, whose values are random: the output is 1/256 of
    them, and a block takes a whole row, 512 steps a wave (96 sequences of the same
    pages).  Of the codes' sum each step may lose 2^-24 of itself; these are random
    but for half of one, a few 2^-24 sqrt(512) in all: 2^-17 of the values' size, 2^-9 of
    the output's, beside its own rounding u."""
    dt, n, hk, d, ps = DT[dtype], 65536, 8, 64, 128
    g = torch.Generator().manual_seed(3)
    x = torch.randn(2, hk, n, d, generator=g)
    pool, table = _written_pool(dt, x[0], x[1], bits, ps)
    rows = 96
    q = torch.zeros(rows, hk * h, d, dtype=dt, device=_dev())
    t = _i32(np.repeat(table, rows, 0))
    out = nx.quantized_paged_attention(q, *pool, t, _i32([n] * rows), backend='hip')
    assert torch.equal(out[0], out[rows - 1])
    top = (1 << bits) - 1
    sc = pool[2].double()
    c = pool[1] if bits == 8 else torch.stack((pool[1] & 15, pool[1] >> 4), -1).flatten(-2)
    held = c.double() * sc[..., 2, None] + sc[..., 3, None]
    want = held.transpose(0, 1).reshape(hk, n, d).mean(1).cpu().numpy().repeat(h, 0)
    u = torch.finfo(dt).eps / 2
    off = _off(out[0], want)
    print(f'[case] off {off:.2e} at {top} codes', flush=True)
    assert off <= u + 2.0 ** -9, off


@pytest.mark.parametrize('dtype, bits', [('bf16', 4), ('f16', 4), ('bf16', 8), ('f16', 8)])
def test_weights_are_pairs(dtype, bits):
    """Two tokens of nearly equal weights and opposite values, of which a hundredth is
    left: weights are held within 2^-22, the sums lose 2^-24 a few times, and the output
    is off by 2^-20 of the values' sizes beside u of itself."""
    dt, d = DT[dtype], 64
    v = torch.randn(1, 2, d, generator=torch.Generator().manual_seed(7))
    v[0, 1] = -v[0, 0]
    k = torch.tensor([0.0, 0.02])[None, :, None].expand(1, 2, d)
    pool, table = _written_pool(dt, k, v, bits)
    q = torch.full((1, 2, d), 0.125, dtype=dt, device=_dev())
    out = nx.quantized_paged_attention(q, *pool, _i32(table), _i32([2]), backend='hip')
    hk, hv = _held(pool, bits)
    want, _ = plain.attention(_n64(q), hk, hv, table, [2], 0.125)
    tol = 2.0 ** -20 * 2 * np.abs(hv).max() + torch.finfo(dt).eps / 2 * np.abs(want)
    assert (np.abs(_n64(out) - want) <= tol).all()


def test_a_page_past_2_31_bytes():
    """One page of more than 2^23 slots of 256 bytes: the last tokens' rows start past
    2^31 bytes of it.  Their keys alone have a score (200), so that they alone count."""
    ps, d, dv, tail = (1 << 23) + 4096, 256, 16, 40
    k = torch.zeros(2, 1, ps, d, dtype=torch.uint8, device=_dev())
    v = torch.zeros(2, 1, ps, dv, dtype=torch.uint8, device=_dev())
    sc = torch.zeros(2, 1, ps, 4, dtype=torch.bfloat16, device=_dev())
    new = [_rand((1, tail, n), torch.bfloat16, s) for n, s in ((d, 1), (dv, 2))]
    n = ps - 3
    table, start, off = _i32([[1]]), _i32([n - tail]), _i32([0, tail])
    nx.write_quantized_pages(k, v, sc, *new, table, start, off, backend='hip')
    sc[1, 0, n - tail:n, 1] += 200 / 16
    q = torch.ones(1, 2, d, dtype=torch.bfloat16, device=_dev())
    out = nx.quantized_paged_attention(q, k, v, sc, table, _i32([n]), backend='hip')
    near = [x[1:, :, n - tail:n].cpu() for x in (k, v, sc)]
    hk, hv = _held(near, 8)
    want, _ = plain.attention(_n64(q), hk, hv, np.array([[0]]), [tail], 1 / 16)
    # (scores of 200, 264 steps of 2^-24 of them)
    assert np.abs(_n64(out) - want).max() <= 4 * (2.0 ** -8 + 264 * 200 * E24)
    got = nx.read_quantized_pages(k, v, sc, table, start, off, tail, bits=8, backend='hip')
    assert np.abs(_n64(got[1])[0] - hv[0, 0]).max() <= 2.0 ** -8 * 4
