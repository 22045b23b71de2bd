"""The quantised cache on the GPU against plain loops (``_quant_plain.py``).

Codes, scales and moved pages have to be equal.  A value read back is one
rounding to its type (u = eps(T) / 2) of a float32 multiply-add (2^-24).

Attention's tolerance is a bound per element, wider than the roundings the kernel
makes (``test_hip_quantized_range.py`` holds it to those):

* q, 16-bit types: 2^-17 of its row's largest element, which the codes' sum of a
  score is off by (the kernel's q is exact down to 2^-29 of it).
* P s': 2^-12 of itself in bf16 (the kernel's two fp16 numbers: 2^-22), 2^-23 in fp16
  and 2^-25 in float32.  The product with ones that takes off what stands in for zero
  sees the same numbers, so the error meets the codes themselves alone.  Small ones:
  2^-27 of the largest weight times the largest scale (the kernel: 2^-34 of the largest
  P s').
* float32 sums, 2^-24 a step: a wave adds up 32 tokens a step, so n / 32 + 24 of
  them (with the join's) over codes with what stands in for zero, up to 1024, and
  the same taken off; scores d + 8 steps.  (For float32 operands, whose codes count
  from their middle, that allows more than there is; ``test_float32_keeps_its_digits``
  holds them to less.)
* the output's rounding, u.
"""

from __future__ import annotations

import math

import _paged_plain as plain
import _quant_plain as qplain
import numpy as np
import pytest
import torch

import nitrix_amd as nx

pytestmark = pytest.mark.gpu

DT = {'bf16': torch.bfloat16, 'f16': torch.float16, 'f32': torch.float32}
E24 = 2.0 ** -24


def _dev():
    return torch.device('cuda:0')


def _i32(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device=_dev())


def _n64(x):
    return x.detach().double().cpu().numpy()


def _rand(shape, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(*shape, generator=g).to(dtype).to(_dev())


def _check(out, q, pool, bits, table, lengths, scale):
    """``out`` against the plain form, on host copies of the operands."""
    dt = q.dtype
    u = torch.finfo(dt).eps / 2
    p_err = {torch.bfloat16: 2.0 ** -12, torch.float16: 2.0 ** -23, torch.float32: 2.0 ** -25}[dt]
    q_err = 0.0 if dt == torch.float32 else 2.0 ** -17
    d = q.shape[2]
    sc = _n64(pool[2])
    codes = [qplain.unpack(x.cpu().numpy(), bits) for x in pool[:2]]
    k, v = (c * sc[..., 2 * w, None] + sc[..., 2 * w + 1, None] for w, c in enumerate(codes))
    # What sums of a key's score and of a value's column go through, without signs:
    # codes, what stands in for zero twice, and the minimum.
    off = (32 if dt == torch.float32 and bits == 4 else 0,
           2048 if bits == 8 or dt == torch.bfloat16 else 128)
    kc, vc = (np.abs(sc[..., 2 * w, None]) * c for w, c in enumerate(codes))
    kab, vab = (
        np.abs(sc[..., 2 * w, None]) * (c + off[w]) + np.abs(sc[..., 2 * w + 1, None])
        for w, c in enumerate(codes)
    )
    qn = _n64(q)
    want, rows = plain.attention(qn, k, v, table, lengths, scale)
    got = _n64(out)
    p, hk, ps, _ = k.shape
    g = q.shape[1] // hk
    tol = np.zeros_like(want)
    for i in range(len(lengths)):
        n = min(max(int(lengths[i]), 0), table.shape[1] * ps)
        at = [(int(table[i, j // ps]), j % ps) for j in range(n)]
        at = [(e, s) for e, s in at if 0 <= e < p]
        if not at:
            continue
        e, s = np.array(at).T
        for h in range(q.shape[1]):
            w, logit, _, _ = rows[i, h]
            es = (d + 8) * E24 * abs(scale) * (kab[e, h // g, s] @ np.abs(qn[i, h]))
            es += q_err * abs(scale) * kc[e, h // g, s].sum(-1) * np.abs(qn[i, h]).max()
            es += 4 * E24 * np.abs(logit)
            rp = es + es.max() + (n + 16) * E24 + 8 * E24 * np.abs(logit).max() + 32 * E24
            codes_v, all_v = vc[e, h // g, s], vab[e, h // g, s]
            tol[i, h] = (w * (rp + 8 * E24)) @ (codes_v + np.abs(sc[e, h // g, s, 3])[:, None])
            tol[i, h] += (w * p_err) @ codes_v
            tol[i, h] += 2.0 ** -27 * w.max() * sc[e, h // g, s, 2].max() * codes[1].max() * len(e)
            tol[i, h] += (n / 32 + 24) * E24 * (w @ all_v)
            tol[i, h] += (u + 8 * E24) * np.abs(want[i, h])
    tiny = 4 * (2.0 ** -24 if dt == torch.float16 else float(torch.finfo(dt).tiny))
    bad = ~(np.abs(got - want) <= tol + tiny)
    assert not bad.any(), (
        f'{bad.sum()} off at {np.argwhere(bad)[:5].tolist()}, worst '
        f'{np.nanmax(np.abs(got - want) / (tol + tiny)):.2f} bounds, nan {np.isnan(got).sum()}')


def _pool(dtype, p, hk, ps, d, dv, bits, seed=0, layout='heads'):
    """Random codes with scales as rows of about -3 .. 3 give."""
    g = torch.Generator().manual_seed(seed)
    k, v = (torch.randint(0, 256, (p, hk, ps, n * bits // 8), generator=g, dtype=torch.uint8)
            for n in (d, dv))
    top = (1 << bits) - 1
    sc = torch.empty(p, hk, ps, 4)
    sc[..., 0::2] = (4 + 3 * torch.rand(p, hk, ps, 2, generator=g)) / top
    sc[..., 1::2] = -2 - 2 * torch.rand(p, hk, ps, 2, generator=g)
    out = [x.to(_dev()) for x in (k, v, sc.to(dtype))]
    if layout == 'heads':
        return out
    wide = []  # pages of a larger allocation, heads before pages
    for x in out:
        y = torch.zeros(hk, p, 2, *x.shape[2:], dtype=x.dtype, device=_dev())
        y[:, :, 1] = x.transpose(0, 1)
        y = y[:, :, 1].transpose(0, 1)
        wide.append(y if y.data_ptr() % 16 == 0 else x)
    return wide


def _table(lens, ps, seed=0, spare=3):
    rng = np.random.default_rng(seed)
    counts = [-(-max(n, 0) // ps) for n in lens]
    p, m = sum(counts) + spare, max(max(counts), 1) + 1
    ids = rng.permutation(p)
    table = np.full((len(lens), m), -1, np.int32)
    at = 0
    used = np.zeros((p, ps), bool)
    for i, c in enumerate(counts):
        table[i, :c] = ids[at:at + c]
        for j in range(c):
            used[ids[at + j], :min(ps, lens[i] - j * ps)] = True
        at += c
    return table, p, used


def _setup(dtype, lens, hk, d, dv, ps, bits, layout='heads', seed=0):
    """Pool and table for ``lens`` tokens, unused slots' scales NaN and codes all
    ones."""
    table, p, used = _table(lens, ps, seed)
    pool = _pool(dtype, p, hk, ps, d, dv, bits, seed, layout)
    idle = torch.from_numpy(~used).to(_dev())
    pool[2].transpose(1, 2)[idle] = math.nan
    for x in pool[:2]:
        x.transpose(1, 2)[idle] = 255
    return pool, table


EDGES = [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 127, 128, 129, 200, 256, 257, 513, 0, 1100]

CASES = [
    # dtype, bits, h, hk, d, dv, ps, layout
    ('bf16', 4, 8, 2, 128, 128, 16, 'heads'),
    ('f16', 4, 8, 2, 128, 128, 64, 'wide'),
    ('f32', 4, 6, 2, 128, 128, 16, 'heads'),
    ('bf16', 4, 4, 4, 64, 64, 16, 'wide'),
    ('f16', 4, 17, 1, 64, 32, 32, 'heads'),
    ('f32', 4, 3, 3, 64, 64, 48, 'heads'),
    ('bf16', 4, 2, 1, 256, 256, 16, 'heads'),
    ('f16', 4, 5, 1, 256, 128, 16, 'heads'),
    ('f32', 4, 2, 1, 256, 256, 32, 'heads'),
    ('bf16', 4, 40, 1, 32, 32, 128, 'wide'),
    ('bf16', 4, 6, 2, 96, 8, 16, 'heads'),
    # more than eight heads a key head: whole products
    ('bf16', 4, 16, 1, 128, 128, 16, 'heads'),
    ('f32', 4, 12, 1, 128, 128, 16, 'heads'),
    ('bf16', 8, 32, 2, 128, 128, 32, 'heads'),
    ('f16', 8, 9, 1, 256, 256, 16, 'heads'),
    ('f32', 8, 10, 1, 64, 64, 16, 'heads'),
    ('f16', 4, 20, 1, 128, 96, 16, 'wide'),
    ('bf16', 8, 8, 2, 128, 128, 16, 'heads'),
    ('f16', 8, 6, 3, 64, 128, 32, 'wide'),
    ('f32', 8, 4, 2, 128, 128, 16, 'heads'),
    ('f32', 8, 2, 1, 256, 256, 16, 'heads'),
    ('bf16', 8, 4, 1, 256, 192, 64, 'heads'),
    ('bf16', 8, 4, 2, 64, 64, 16, 'heads'),
    # rows that end inside a lane's codes, pages that are no multiple of a half
    ('bf16', 4, 6, 2, 80, 80, 16, 'heads'),
    ('f16', 4, 14, 2, 200, 8, 48, 'heads'),
    ('f32', 4, 2, 1, 8, 40, 16, 'heads'),
    ('bf16', 4, 8, 2, 128, 128, 1, 'heads'),
    ('bf16', 4, 8, 2, 64, 64, 8, 'wide'),
    ('f16', 4, 6, 1, 256, 40, 24, 'heads'),
    ('f32', 4, 4, 2, 128, 128, 7, 'heads'),
    ('bf16', 8, 8, 2, 80, 80, 24, 'heads'),
    ('f16', 8, 4, 2, 128, 72, 10, 'heads'),
    ('f32', 8, 4, 2, 64, 64, 5, 'wide'),
    ('f32', 8, 2, 1, 248, 256, 5, 'heads'),
]


@pytest.mark.parametrize('case', CASES, ids=lambda c: '_'.join(map(str, c)))
def test_attention(case):
    dt, bits, h, hk, d, dv, ps, layout = case
    print(f'[case] {case}', flush=True)
    pool, table = _setup(DT[dt], EDGES, hk, d, dv, ps, bits, layout)
    q = _rand((len(EDGES), h, d), DT[dt], 9)
    out = nx.quantized_paged_attention(q, *pool, _i32(table), _i32(EDGES), backend='hip')
    torch.cuda.synchronize()
    _check(out, q, pool, bits, table, EDGES, 1 / math.sqrt(d))
    assert (out[0] == 0).all()
    again = nx.quantized_paged_attention(q, *pool, _i32(table), _i32(EDGES), backend='hip')
    assert torch.equal(out, again)


@pytest.mark.parametrize('bits', [4, 8])
@pytest.mark.parametrize('ps', [16, 12])
def test_short_tables(ps, bits):
    """Rows that a block takes whole."""
    lens = [0, 1, 16, 40, 77, 128, 129, 150]
    pool, table = _setup(torch.bfloat16, lens, 2, 128, 128, ps, bits)
    q = _rand((8, 8, 128), torch.bfloat16, 3)
    out = nx.quantized_paged_attention(q, *pool, _i32(table), _i32(lens), backend='hip')
    _check(out, q, pool, bits, table, lens, 1 / math.sqrt(128))


@pytest.mark.parametrize('bits', [4, 8])
@pytest.mark.parametrize('ps', [16, 12])
def test_bad_pages_and_lengths(ps, bits):
    """Entries that name no page hold no tokens, lengths are clamped."""
    lens = [100, 300, 64, 40, 90, 17]
    table, p, _ = _table(lens, ps)
    pool = _pool(torch.float16, p, 2, ps, 64, 64, bits)
    table[0, 2] = -1
    table[1, 0], table[1, 5] = p, 2 ** 31 - 1
    table[2, :] = -2 ** 31
    table[5, 1] = p + 7
    lengths = [100, 2 ** 31 - 1, 64, -5, 90, 17]
    table[1][table[1] == -1] = 0
    q = _rand((6, 4, 64), torch.float16, 3)
    out = nx.quantized_paged_attention(q, *pool, _i32(table), _i32(lengths), backend='hip')
    _check(out, q, pool, bits, table, lengths, 0.125)
    assert (out[2] == 0).all() and (out[3] == 0).all()


def test_scales_and_large_logits():
    lens = [5, 400, 130]
    pool, table = _setup(torch.bfloat16, lens, 1, 64, 64, 16, 4)
    q = _rand((3, 4, 64), torch.bfloat16, 4) * 8
    for scale in (0.0, 1.0):
        out = nx.quantized_paged_attention(q, *pool, _i32(table), _i32(lens), scale=scale,
                                           backend='hip')
        _check(out, q, pool, 4, table, lens, scale)
    out = nx.quantized_paged_attention(q, *pool, _i32(table), _i32(lens), scale=-0.5, backend='hip')
    _check(out, -q, pool, 4, table, lens, 0.5)


@pytest.mark.parametrize('bits', [4, 8])
def test_a_value_that_is_nan_stays_in_its_sequence(bits):
    lens = [40, 300, 200]
    pool, table = _setup(torch.bfloat16, lens, 1, 64, 64, 16, bits)
    pool[2][int(table[1, 3]), 0, 5, 2] = math.nan
    pool[2][int(table[2, 1]), 0, 9, 0] = math.inf
    q = _rand((3, 2, 64), torch.bfloat16, 4)
    out = nx.quantized_paged_attention(q, *pool, _i32(table), _i32(lens), backend='hip')
    assert torch.isfinite(out[0].float()).all() and torch.isnan(out[1].float()).all()
    assert torch.isnan(out[2].float()).all()


def test_large_and_small_rows():
    """Scales over the whole range of bf16: P s' leaves no range."""
    lens = [200]
    pool, table = _setup(torch.bfloat16, lens, 1, 64, 64, 16, 4)
    # (keys as they are, values a power of two larger or smaller)
    for power in (100, -100, 0):
        sc = pool[2].clone()
        sc[..., 2:] *= 2.0 ** power
        q = _rand((1, 2, 64), torch.bfloat16, 4)
        out = nx.quantized_paged_attention(q, pool[0], pool[1], sc, _i32(table), _i32(lens),
                                           backend='hip')
        _check(out, q, (pool[0], pool[1], sc), 4, table, lens, 0.125)


@pytest.mark.parametrize('dtype, value', [('bf16', 1e30), ('f16', 3e4), ('f32', -1e25), ('bf16', 0.0)])
def test_rows_of_one_value(dtype, value):
    """Constant values have a scale of zero, whatever they are; half of the second
    sequence's, of the first's all."""
    lens = [300, 200]
    pool, table = _setup(DT[dtype], lens, 1, 64, 64, 16, 4)
    for j in list(table[0, :19]) + list(table[1, :6]):
        pool[2][int(j), ..., 2] = 0
        pool[2][int(j), ..., 3] = value
    q = _rand((2, 3, 64), DT[dtype], 4)
    out = nx.quantized_paged_attention(q, *pool, _i32(table), _i32(lens), backend='hip')
    z = pool[2][int(table[0, 0]), 0, 0, 3].item()
    # (the sum of weights times the value over the sum of weights, 300 steps each)
    assert (out[0].double() - z).abs().max() <= abs(z) * (600 * E24 + torch.finfo(DT[dtype]).eps / 2)
    _check(out, q, pool, 4, table, lens, 0.125)


@pytest.mark.parametrize('dtype, bits', [('bf16', 4), ('f32', 8)])
def test_one_long_sequence(dtype, bits):
    """Every block a piece of the same rows."""
    lens = [40001]
    pool, table = _setup(DT[dtype], lens, 2, 64, 64, 16, bits)
    q = _rand((1, 6, 64), DT[dtype], 5)
    out = nx.quantized_paged_attention(q, *pool, _i32(table), _i32(lens), backend='hip')
    _check(out, q, pool, bits, table, lens, 0.125)


@pytest.mark.parametrize('bits, lens, hk, d', [
    (4, [700, 90, 333], 4, 64), (8, [8192, 5000], 2, 128), (4, [60000], 1, 64), (8, [2371, 197], 2, 256),
    (4, [484, 1100], 3, 32),
])
def test_float32_keeps_its_digits(bits, lens, hk, d):
    """Values of random sign nearly cancel in a long row, and an error that does not
    (one of the codes' middle, of a single weight) stands out.  Each weight may be off
    by its score's and its exponent's roundings: 3 d / 32 products' sums, half a step
    of a score below 8 each, half a step of an exponent below 32, and 8 steps of 2^-24
    for the exponential, the products behind it and the sums' share: (12 d / 128) 2^-22
    + 2^-20 + 2^-21, at most 4.5 2^-20 (d = 256; below 128 3 2^-20).  These are as
    random as the values, so that the whole output is off by no more than that share
    of its norm."""
    pool, table = _setup(torch.float32, lens, hk, d, d, 16, bits)
    x = torch.randn(*pool[2].shape[:3], 2, 2, d, generator=torch.Generator().manual_seed(8))
    top = (1 << bits) - 1
    lo, hi = x[..., 0, :, :].amin(-1), x[..., 0, :, :].amax(-1)
    pool[2][..., 0::2] = ((hi - lo) / top).to(pool[2])
    pool[2][..., 1::2] = lo.to(pool[2])
    codes = ((x[..., 0, :, :] - lo[..., None]) / (hi - lo)[..., None] * top).round().to(torch.uint8)
    for i in range(2):
        c = codes[..., i, :]
        pool[i].copy_(c if bits == 8 else c[..., ::2] | c[..., 1::2] << 4)
    q = _rand((len(lens), 2 * hk, d), torch.float32, 5)
    out = nx.quantized_paged_attention(q, *pool, _i32(table), _i32(lens), backend='hip')
    sc = _n64(pool[2])
    k, v = (qplain.values(y.cpu().numpy(), sc, i, bits) for i, y in enumerate(pool[:2]))
    want, _ = plain.attention(_n64(q), k, v, table, lens, 1 / math.sqrt(d))
    for i in range(len(lens)):
        for h in range(2 * hk):
            off = np.linalg.norm(_n64(out[i, h]) - want[i, h]) / np.linalg.norm(want[i, h])
            assert off <= (4.5 if d > 128 else 3) * 2.0 ** -20, (lens[i], h, off)


def test_many_sequences():
    rng = np.random.default_rng(2)
    lens = [int(x) for x in rng.integers(0, 90, 700)]
    lens[5] = 1100
    pool, table = _setup(torch.bfloat16, lens, 2, 32, 32, 16, 4)
    q = _rand((700, 4, 32), torch.bfloat16, 6)
    out = nx.quantized_paged_attention(q, *pool, _i32(table), _i32(lens), backend='hip')
    _check(out, q, pool, 4, table, lens, 1 / math.sqrt(32))


@pytest.mark.parametrize('rows, longest', [(130, 1500), (127, 1500), (130, 2500)])
def test_rows_shared_by_blocks_or_a_block_each(rows, longest):
    rng = np.random.default_rng(rows)
    lens = [int(x) for x in rng.integers(0, 60, rows)]
    lens[7], lens[8], lens[rows - 1] = longest, 0, 129
    pool, table = _setup(torch.bfloat16, lens, 2, 64, 64, 16, 4)
    q = _rand((rows, 2, 64), torch.bfloat16, 6)
    out = nx.quantized_paged_attention(q, *pool, _i32(table), _i32(lens), backend='hip')
    _check(out, q, pool, 4, table, lens, 0.125)


def test_operand_layouts():
    lens = [70, 3]
    pool, table = _setup(torch.bfloat16, lens, 2, 64, 64, 16, 4)
    base = _rand((4, 2, 65), torch.bfloat16, 7)
    wide = _i32(np.pad(table, ((0, 0), (0, 3)), constant_values=99))
    for q in (base[:, :, :64].transpose(0, 1), _rand((2, 3, 4, 64), torch.bfloat16, 8)[:, 1]):
        for t in (wide[:, :table.shape[1]], _i32(table.T.copy()).T):
            out = nx.quantized_paged_attention(q, *pool, t, _i32([70, 0, 3, 0])[::2], backend='hip')
            _check(out, q, pool, 4, table, lens, 0.125)


def test_a_pool_past_2_32_bytes():
    p, hk, ps, d = 150000, 4, 128, 128
    k, v = (torch.empty(p, hk, ps, d // 2, dtype=torch.uint8, device=_dev()) for _ in range(2))
    sc = torch.empty(p, hk, ps, 4, dtype=torch.bfloat16, device=_dev())
    assert k.numel() > 1 << 32
    ids = [p - 1, 1, p - 2, p // 2 + 7]
    small = _pool(torch.bfloat16, 4, hk, ps, d, d, 4)
    for x, y in zip((k, v, sc), small):
        x[ids] = y
    table = np.array([[p - 1, 1, p - 2], [p // 2 + 7, -1, -1]], np.int32)
    lens = [300, 100]
    q = _rand((2, 8, d), torch.bfloat16, 1)
    out = nx.quantized_paged_attention(q, k, v, sc, _i32(table), _i32(lens), backend='hip')
    near = np.array([[0, 1, 2], [3, -1, -1]], np.int32)
    _check(out, q, small, 4, near, lens, 1 / math.sqrt(d))
    new = _rand((2, 2 * hk, d), torch.bfloat16, 2).transpose(0, 1)
    for pool, t in (((k, v, sc), table), (small, near)):
        nx.write_quantized_pages(*pool, new[:hk], new[hk:], _i32(t), _i32([300, 100]), backend='hip')
    for x, y in zip((k, v, sc), small):
        assert torch.equal(x[ids], y)
    a, b = (nx.read_quantized_pages(*pool, _i32(t), _i32([300, 100]), backend='hip')
            for pool, t in (((k, v, sc), table), (small, near)))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    nx.copy_pages(k, v, [p - 1], [p - 3], scales=sc, backend='hip')
    assert all(torch.equal(x[p - 3], x[p - 1]) for x in (k, v, sc))


# ---------------------------------------------------------------------------
# Writing and reading back
# ---------------------------------------------------------------------------


def _written(pool, k, v, table, starts, offsets, bits):
    """The pool as plain loops write it (host copies)."""
    want = [x.cpu().clone() for x in pool]
    k, v = k.cpu(), v.cpu()
    for tok, page, slot in qplain.slots(table, starts, offsets, k.shape[1], want[0].shape[0],
                                        want[0].shape[2]):
        for which, x in enumerate((k, v)):
            for h in range(k.shape[0]):
                c, s, z = qplain.quantise_row(x[h, tok], bits)
                c = torch.tensor(c, dtype=torch.uint8)
                row = c if bits == 8 else c[0::2] | c[1::2] << 4
                if math.isfinite(s):
                    want[which][page, h, slot] = row
                want[2][page, h, slot, 2 * which] = s
                want[2][page, h, slot, 2 * which + 1] = z
    return want


def _same(got, want):
    for a, w in zip(got, want):
        torch.testing.assert_close(a.cpu(), w, rtol=0, atol=0, equal_nan=True)


@pytest.mark.parametrize('bits', [4, 8])
@pytest.mark.parametrize('dtype, hk, d, dv, ps, layout', [
    ('bf16', 8, 128, 128, 16, 'heads'), ('f16', 3, 64, 32, 24, 'wide'),
    ('f32', 1, 8, 256, 7, 'heads'), ('bf16', 2, 80, 200, 64, 'wide'),
])
@pytest.mark.parametrize('packed', [True, False])
def test_write_and_read(dtype, hk, d, dv, ps, layout, packed, bits):
    starts = np.array([0, 5, 100, 31, 2, 0, -7, 9], np.int32)
    new = [20, 0, 37, 1, 30, 0, 20, 16] if packed else [1] * 8
    lens = [int(max(a + n, 1)) for a, n in zip(starts, new)]
    table, p, _ = _table(lens, ps)
    pool = _pool(DT[dtype], p, hk, ps, d, dv, bits, layout=layout)
    table[2, 1] = -1
    table[4, 0] = p + 3
    starts[7] = table.shape[1] * ps - 8  # runs out of the table
    off = np.concatenate([[4], 4 + np.cumsum(new)]).astype(np.int32) if packed else None
    t = int(off[-1]) + 9 if packed else 8
    nk = _rand((t, hk, d), DT[dtype], 20).transpose(0, 1)
    nv = _rand((hk, t, dv), DT[dtype], 21)
    want = _written(pool, nk, nv, table, starts, off, bits)
    args = (_i32(table), _i32(starts), None if off is None else _i32(off))
    nx.write_quantized_pages(*pool, nk, nv, *args, backend='hip')
    _same(pool, want)
    k, v = nx.read_quantized_pages(*pool, *args, t, bits=bits, backend='hip')
    u = torch.finfo(DT[dtype]).eps / 2
    sc = _n64(pool[2])
    for which, got in enumerate((k, v)):
        held = qplain.values(want[which].numpy(), sc, which, bits)
        ref, size = np.zeros(tuple(got.shape)), np.zeros(tuple(got.shape))
        for tok, page, slot in qplain.slots(table, starts, off, t, p, ps):
            ref[:, tok] = held[page, :, slot]
            size[:, tok] = np.abs(sc[page, :, slot, 2 * which + 1])[:, None] + np.abs(ref[:, tok])
        assert (np.abs(_n64(got) - ref) <= u * np.abs(ref) * (1 + E24) + 2 * E24 * size).all()


@pytest.mark.parametrize('dtype', ['bf16', 'f16', 'f32'])
@pytest.mark.parametrize('bits', [4, 8])
def test_rows_next_to_a_border(dtype, bits):
    """Ties, constant rows, denormal and huge ranges, NaN and infinity, and
    minima far from the other elements."""
    dt, top = DT[dtype], (1 << bits) - 1
    info = torch.finfo(dt)
    rows = []
    for s in (1.0, 2.0 ** -8, 2.0 ** 9):  # quotients n + 1/2 exactly
        x = torch.arange(32) * 0.5
        x[1] = top
        rows.append((x.clamp(max=top) - 3) * s)
    g = torch.Generator().manual_seed(4)
    for z in (0.0, -7.5, 6.5, -0.4375):  # a minimum far larger than the others' places
        x = torch.rand(32, generator=g) * 2.0 ** -torch.arange(32.0)
        x[0], x[1] = z, z + top
        rows.append(x.clamp(min=z))
    rows.append(torch.full((32,), -1.25))
    rows.append(torch.rand(32, generator=g) * float(info.tiny))
    rows.append(torch.rand(32, generator=g) * float(info.smallest_normal) * 2 ** -5)
    rows.append((torch.rand(32, generator=g) - 0.5) * float(info.max) * 0.9)
    rows.append((torch.rand(32, generator=g) - 0.5).sign() * float(info.max))
    for bad in (math.nan, math.inf, -math.inf):
        x = torch.randn(32, generator=g)
        x[17] = bad
        rows.append(x)
    rows += [torch.randn(32, generator=g) * 2.0 ** e for e in (-20, 0, 3, 10)]
    x = torch.stack(rows).to(dt)[None].to(_dev())
    t = x.shape[1]
    pool = _pool(dt, 3, 1, 16, 32, 32, bits)
    table, starts, off = np.array([[2, 0]], np.int32), np.array([1], np.int32), np.array([0, t], np.int32)
    y = x.flip(-1).contiguous()
    want = _written(pool, x, y, table, starts, off, bits)
    nx.write_quantized_pages(*pool, x, y, _i32(table), _i32(starts), _i32(off), backend='hip')
    finite = torch.isfinite(want[2])
    torch.testing.assert_close(pool[2].cpu()[finite], want[2][finite], rtol=0, atol=0)
    k, v = nx.read_quantized_pages(*pool, _i32(table), _i32(starts), _i32(off), t, bits=bits,
                                   backend='hip')
    for i in range(t):
        c, s, z = qplain.quantise_row(x[0, i].cpu(), bits)
        if not (math.isfinite(s) and math.isfinite(z)):
            assert torch.isnan(k[0, i].float()).all() and torch.isnan(v[0, i].float()).all(), i
            continue
        page, slot = int(table[0, (1 + i) // 16]), (1 + i) % 16
        for which, row in ((0, c), (1, c[::-1])):
            got = qplain.unpack(pool[which][page, 0, slot].cpu().numpy(), bits)
            assert got.tolist() == list(row), (i, which)


def test_writes_equal_the_other_engine_on_many_rows():
    for dtype in DT.values():
        for bits in (4, 8):
            t, hk, d = 3000, 4, 128
            x, y = (_rand((t, hk, d), dtype, s).transpose(0, 1) * 3 for s in (1, 2))
            table = _i32(np.random.default_rng(0).permutation(188)[None])
            pools = [_pool(dtype, 188, hk, 16, d, d, bits) for _ in range(2)]
            for pool, backend in zip(pools, ('hip', 'jax')):
                nx.write_quantized_pages(*pool, x, y, table, _i32([3]), _i32([0, t]),
                                         backend=backend)
            assert all(torch.equal(a, b) for a, b in zip(*pools))


@pytest.mark.parametrize('dtype, bits, d, ps', [('bf16', 4, 8, 5), ('f32', 8, 64, 16), ('f16', 4, 128, 16)])
def test_pages_move_with_their_scales(dtype, bits, d, ps):
    lens = [40, 3 * ps, 7, 0, 0, 2 * ps + 1]
    table, p, _ = _table(lens, ps, spare=9)
    refs = np.bincount(table[table >= 0], minlength=p)
    pools = [_pool(DT[dtype], p, 3, ps, d, 2 * d, bits) for _ in range(2)]
    src, dst = [0, 1, 5, 0, 9], [3, 4, 2, 0, 1]
    out = []
    for pool, backend in zip(pools, ('hip', 'jax')):
        k, v, s = pool
        t, n, r = nx.fork_sequences(k, v, _i32(table), _i32(lens), _i32(refs), _i32(src), _i32(dst),
                                    scales=s, backend=backend)
        t, r = nx.compact_pages(k, v, t, r, scales=s, backend=backend)
        free = [i for i in range(p) if int(r[i]) == 0]
        nx.copy_pages(k, v, [0, 1], free[:2], scales=s, backend=backend)
        out.append((t, n, r))
    assert all(torch.equal(a, b) for a, b in zip(*out))
    # (what a moved page leaves in slots behind the last token is not compared)
    t, n, _ = out[0]
    for i in range(len(lens)):
        for j in range(int(n[i])):
            e, s = int(t[i, j // ps]), j % ps
            for a, b in zip(*pools):
                assert torch.equal(a[e, :, s], b[e, :, s])


# ---------------------------------------------------------------------------
# Together, streams and graphs
# ---------------------------------------------------------------------------


def test_a_decoding_run():
    """Prompts rotated, written and attended as the cache holds them, then tokens
    one by one, against float64 attention over what was read back."""
    dt, hk, h, d, ps = torch.bfloat16, 2, 6, 64, 16
    prompts, steps = [37, 1, 64], 5
    table = _i32(np.random.default_rng(3).permutation(30).reshape(3, 10))
    pool = _pool(dt, 30, hk, ps, d, d, 4)
    freq = nx.rotary_frequencies(d, device=_dev())
    off = _i32(np.concatenate([[0], np.cumsum(prompts)]))
    t = sum(prompts)
    zeros = _i32([0, 0, 0])
    q, k, v = (_rand((t, n, d), dt, s).transpose(0, 1) for s, n in ((1, h), (2, hk), (3, hk)))
    q, k = nx.rotary_embed(q, k, nx.packed_positions(off, t), freq, backend='hip')
    nx.write_quantized_pages(*pool, k, v, table, zeros, off, backend='hip')
    kc, vc = nx.read_quantized_pages(*pool, table, zeros, off, t, backend='hip')
    out = nx.packed_attention(q, kc, vc, off, causal=True, backend='hip')
    want = nx.packed_attention(q.cpu().double(), kc.cpu().double(), vc.cpu().double(), off.cpu(),
                               causal=True)
    # (one rounding of P and one of the output, and what 64 or fewer terms of
    # fp32 sums add)
    assert float((out.cpu().double() - want).abs().max()) <= 3 * 2.0 ** -8 * float(vc.abs().max())
    lengths = _i32(prompts)
    for step in range(steps):
        q, k, v = (_rand((3, n, d), dt, 10 * step + s).transpose(0, 1)
                   for s, n in ((4, h), (5, hk), (6, hk)))
        q, k = nx.rotary_embed(q, k, lengths, freq, backend='hip')
        nx.write_quantized_pages(*pool, k, v, table, lengths, backend='hip')
        lengths = lengths + 1
        q = q.transpose(0, 1)
        out = nx.quantized_paged_attention(q, *pool, table, lengths, backend='hip')
        _check(out, q, pool, 4, table.cpu().numpy(), lengths.tolist(), 1 / math.sqrt(d))


def test_streams_and_graph_replay():
    lens = [300, 45, 0, 1200]
    pool, table = _setup(torch.bfloat16, lens, 2, 64, 64, 16, 4)
    q = _rand((4, 8, 64), torch.bfloat16, 11)
    t, n = _i32(table), _i32(lens)
    freq = nx.rotary_frequencies(64, device=_dev())
    want = nx.quantized_paged_attention(q, *pool, t, n, backend='hip')
    torch.cuda.synchronize()
    st = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for s in st:
        with torch.cuda.stream(s):
            outs.append(nx.quantized_paged_attention(q, *pool, t, n, backend='hip'))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    new = _rand((4, 4, 64), torch.bfloat16, 12)
    graph = torch.cuda.CUDAGraph()

    def step():
        rq, k = nx.rotary_embed(q.transpose(0, 1), new[:, :2].transpose(0, 1), n - 1, freq,
                                backend='hip')
        v = new[:, 2:].transpose(0, 1)
        nx.write_quantized_pages(*pool, k, v, t, n - 1, backend='hip')
        held = nx.read_quantized_pages(*pool, t, n - 1, backend='hip')
        return nx.quantized_paged_attention(rq.transpose(0, 1), *pool, t, n, backend='hip'), held

    with torch.cuda.graph(graph, stream=st[0]):
        out, held = step()
    for ls in ([300, 45, 0, 1200], [17, 16, 0, 1], [256, 2, 0, 1100]):
        n.copy_(_i32(ls))
        new.copy_(_rand((4, 4, 64), torch.bfloat16, sum(ls)))
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone(), held[0].clone(), held[1].clone()
        again, (k, v) = step()
        assert torch.equal(got[0], again) and torch.equal(got[1], k) and torch.equal(got[2], v)


def test_two_graphs_do_not_share_results():
    """Two captured calls replayed on two streams keep their own workspaces."""
    pool, table = _setup(torch.bfloat16, [9000, 5000], 2, 64, 64, 16, 4)
    t = _i32(table)
    calls = []
    for lens, seed in (([9000, 5000], 1), ([4321, 77], 2)):
        q, n = _rand((2, 4, 64), torch.bfloat16, seed), _i32(lens)
        want = nx.quantized_paged_attention(q, *pool, t, n, backend='hip')
        graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            out = nx.quantized_paged_attention(q, *pool, t, n, backend='hip')
        calls.append((graph, stream, out, want, q, n))
    for _ in range(3):
        for graph, stream, out, *_ in calls:
            out.zero_()
        torch.cuda.synchronize()
        for graph, stream, *_ in calls:
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for _, _, out, want, *_ in calls:
            assert torch.equal(out, want)


def test_declined_calls_fall_back_loudly():
    pool, table = _setup(torch.bfloat16, [20], 1, 64, 64, 16, 4)
    pool[2].nan_to_num_()
    q = _rand((1, 2, 64), torch.bfloat16, 1)
    nx.reset_fallback_state()
    with pytest.warns(nx.NitrixBackendFallback):
        out = nx.quantized_paged_attention(q.requires_grad_(True), *pool, _i32(table), _i32([20]))
    assert out.requires_grad
    k12, v12 = (torch.zeros(3, 1, 16, 6, dtype=torch.uint8, device=_dev()) for _ in range(2))
    sc = torch.zeros(3, 1, 16, 4, dtype=torch.bfloat16, device=_dev())
    x = _rand((1, 1, 12), torch.bfloat16, 2)
    with pytest.warns(nx.NitrixBackendFallback):
        nx.write_quantized_pages(k12, v12, sc, x, x, _i32([[2]]), _i32([3]))
    gap = torch.zeros(3, 1, 32, 8, dtype=torch.uint8, device=_dev())[:, :, ::2]
    with pytest.warns(nx.NitrixBackendFallback):
        nx.read_quantized_pages(gap, gap.clone(), sc, _i32([[2]]), _i32([3]))

@pytest.mark.parametrize('bits', [4, 8])
@pytest.mark.parametrize('dtype', ['bf16', 'f16', 'f32'])
def test_rows_up_to_the_largest_number_read_back_finite(dtype, bits):
    """A scale rounded up takes the last code past the type's largest number: it reads
    back as that, within the step and the scale's rounding; infinite scales and
    minima stay what they are."""
    dt, top = DT[dtype], (1 << bits) - 1
    most = float(torch.finfo(dt).max)
    lo = -most if dtype == 'f16' else 0.0
    x = torch.linspace(0, 1, 32, dtype=torch.float64)[None, None] * (most - lo) + lo
    x = x.to(dt).repeat(1, 5, 1).to(_dev())
    pool = _pool(dt, 3, 1, 16, 32, 32, bits)
    table, starts, off = _i32([[1]]), _i32([2]), _i32([0, 5])
    nx.write_quantized_pages(*pool, x, x, table, starts, off, backend='hip')
    sc = pool[2]
    sc[1, 0, 4, 0], sc[1, 0, 5, 1], sc[1, 0, 6, 2] = math.inf, math.inf, math.nan
    k, v = nx.read_quantized_pages(*pool, table, starts, off, 5, bits=bits, backend='hip')
    for y in (k[:, :2], v[:, :4]):
        assert torch.isfinite(y).all() and float(y.max()) == most
        off_by = (y.double() - x[:, :y.shape[1]].double()).abs().max()
        step = (most - lo) / top
        assert off_by <= step / 2 + (most - lo) * torch.finfo(dt).eps
    assert not torch.isfinite(k[0, 2]).any() and (k[0, 3] == math.inf).all()
    assert torch.isnan(v[0, 4]).all()


@pytest.mark.parametrize('b', [1023, 1024, 3000])
def test_many_sequences_written_and_read(b):
    """Offsets that are kept on the chip and ones that are not; empty sequences."""
    rng = np.random.default_rng(b)
    new = rng.integers(0, 4, b)
    off = np.concatenate([[2], 2 + np.cumsum(new)]).astype(np.int32)
    t, hk, d = int(off[-1]) + 3, 1, 16
    starts = rng.integers(0, 30, b).astype(np.int32)
    table = rng.permutation(3 * b).reshape(b, 3).astype(np.int32)
    pools = [_pool(torch.float16, 3 * b, hk, 16, d, d, 8) for _ in range(2)]
    x, y = (_rand((hk, t, d), torch.float16, s) for s in (1, 2))
    args = _i32(table), _i32(starts), _i32(off)
    held = []
    for pool, backend in zip(pools, ('hip', 'jax')):
        nx.write_quantized_pages(*pool, x, y, *args, backend=backend)
        held.append(nx.read_quantized_pages(*pool, *args, t, bits=8, backend=backend))
    assert all(torch.equal(a, b) for a, b in zip(*pools))
    for got, want in zip(*held):
        torch.testing.assert_close(got, want, rtol=2.0 ** -10, atol=2.0 ** -24)
    assert (held[0][0][:, :2] == 0).all() and (held[0][0][:, -3:] == 0).all()
