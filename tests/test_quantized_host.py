"""Host side of the quantised cache: the reference engine against plain loops,
refusals, and the C ABI's checks (CPU only)."""

from __future__ import annotations

import ctypes
import math

import _paged_plain as plain
import _quant_plain as qplain
import numpy as np
import pytest
import torch

import nitrix_amd as nx
from nitrix_amd import _lib

DT = {'bf16': torch.bfloat16, 'f16': torch.float16, 'f32': torch.float32}


def _i32(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32)


def _pool(p, hk, ps, d, dv, bits, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    k, v = (torch.randint(0, 256, (p, hk, ps, n * bits // 8), generator=g, dtype=torch.uint8)
            for n in (d, dv))
    return k, v, (torch.rand(p, hk, ps, 4, generator=g) - 0.3).to(dtype)


def _rows(shape, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(*shape, generator=g).to(dtype)


@pytest.mark.parametrize('bits', [4, 8])
@pytest.mark.parametrize('dtype', ['bf16', 'f16', 'f32'])
def test_write_reference(dtype, bits):
    dt = DT[dtype]
    k0 = _pool(30, 2, 4, 16, 8, bits, dt)
    table = np.random.default_rng(1).permutation(30)[:30].reshape(6, 5).astype(np.int32)
    table[2, 1], table[3, 0] = -1, 30
    starts = np.array([0, 3, 2, 1, -2, 19], np.int32)
    offsets = np.array([2, 5, 5, 9, 12, 16, 19], np.int32)
    k, v = _rows((2, 21, 16), dt, 2), _rows((2, 21, 8), dt, 3)
    k[0, 3] = 1.5  # a constant row
    k[1, 4, 3], v[0, 5, 0] = math.nan, math.inf
    got = [x.clone() for x in k0]
    nx.write_quantized_pages(*got, k, v, _i32(table), _i32(starts), _i32(offsets))
    want = [x.clone() for x in k0]
    for tok, page, slot in qplain.slots(table, starts, offsets, 21, 30, 4):
        for which, x in enumerate((k, v)):
            for h in range(2):
                c, s, z = qplain.quantise_row(x[h, tok], bits)
                c = torch.tensor(c, dtype=torch.uint8)
                want[which][page, h, slot] = c if bits == 8 else c[0::2] | c[1::2] << 4
                want[2][page, h, slot, 2 * which] = s
                want[2][page, h, slot, 2 * which + 1] = z
    for a, w in zip(got, want):
        torch.testing.assert_close(a, w, rtol=0, atol=0, equal_nan=True)


@pytest.mark.parametrize('bits', [4, 8])
def test_read_reference(bits):
    pool = _pool(30, 2, 4, 16, 8, bits, torch.float32)
    table = np.random.default_rng(1).permutation(30)[:18].reshape(3, 6).astype(np.int32)
    table[1, 2] = -7
    starts, offsets = np.array([1, 20, 0], np.int32), np.array([1, 6, 12, 30], np.int32)
    k, v = nx.read_quantized_pages(*pool, _i32(table), _i32(starts), _i32(offsets), 33, bits=bits)
    for which, got in enumerate((k, v)):
        all_values = qplain.values(pool[which].numpy(), pool[2].double().numpy(), which, bits)
        want = np.zeros(tuple(got.shape))
        for tok, page, slot in qplain.slots(table, starts, offsets, 33, 30, 4):
            want[:, tok] = all_values[page, :, slot]
        np.testing.assert_allclose(got.numpy(), want, rtol=2 ** -22, atol=2 ** -22)
    one = nx.read_quantized_pages(*pool, _i32(table), _i32([1, 3, 2]), bits=bits)
    assert one[0].shape == (2, 3, 16) and one[1].shape == (2, 3, 8)


@pytest.mark.parametrize('bits', [4, 8])
@pytest.mark.parametrize('ps', [1, 5, 16])
def test_attention_reference(ps, bits):
    rng = np.random.default_rng(ps)
    p, m, b = 40, 6, 7
    pool = _pool(p, 2, ps, 16, 8, bits, torch.float64)
    table, lengths, _ = plain.cache(rng, b, m, p, ps)
    lengths[0], lengths[1], lengths[2] = -3, m * ps + 9, 0
    table[3, 0] = p + 5
    used = np.zeros((p, ps), bool)
    for i in range(b):
        for j in range(min(max(lengths[i], 0), m * ps)):
            if 0 <= table[i, j // ps] < p:
                used[table[i, j // ps], j % ps] = True
    pool[2].transpose(1, 2)[torch.from_numpy(~used)] = math.nan
    q = torch.from_numpy(rng.standard_normal((b, 6, 16)))
    k, v = (qplain.values(pool[w].numpy(), pool[2].numpy(), w, bits) for w in (0, 1))
    want, _ = plain.attention(q.numpy(), k, v, table, lengths, 0.05)
    got = nx.quantized_paged_attention(q, *pool, _i32(table), _i32(lengths), scale=0.05)
    np.testing.assert_allclose(got.numpy(), want, atol=1e-12)
    assert (want[0] == 0).all() and (want[2] == 0).all()


def test_attention_reference_is_differentiable():
    pool = _pool(5, 1, 2, 8, 8, 4, torch.float64)
    scales = pool[2].requires_grad_(True)
    q = torch.randn(2, 2, 8, dtype=torch.float64, requires_grad=True)
    table, lengths = _i32([[0, 3], [4, -1]]), _i32([3, 1])
    assert torch.autograd.gradcheck(
        lambda a, s: nx.quantized_paged_attention(a, pool[0], pool[1], s, table, lengths),
        (q, scales))


def test_a_round_trip_is_off_by_at_most_half_a_step():
    # What rounding s to its type (relative eps / 2) moves the largest code by
    # is at most top * eps / 2 steps, clamped codes included.
    for dtype in (torch.float32, torch.bfloat16):
        for bits in (4, 8):
            pool = _pool(2, 1, 8, 32, 32, bits, dtype)
            x, y = _rows((1, 8, 32), dtype, 5), _rows((1, 8, 32), dtype, 6)
            table, starts, offsets = _i32([[1]]), _i32([0]), _i32([0, 8])
            nx.write_quantized_pages(*pool, x, y, table, starts, offsets)
            k, v = nx.read_quantized_pages(*pool, table, starts, offsets, 8, bits=bits)
            eps = torch.finfo(dtype).eps / 2
            for which, (a, b) in enumerate(((x, k), (y, v))):
                step = pool[2][1, 0, :, 2 * which].double()[:, None]
                bound = step * (0.5 + ((1 << bits) - 1) * eps) + eps * a[0].double().abs().amax() * 2
                assert ((a[0].double() - b[0].double()).abs() <= bound).all()


@pytest.mark.parametrize('bits', [4, 8])
def test_pages_move_with_their_scales(bits):
    pool = _pool(12, 2, 4, 8, 16, bits, torch.float16)
    before = [x.clone() for x in pool]
    nx.copy_pages(pool[0], pool[1], [3, 4], [7, 9], scales=pool[2])
    for x, w in zip(pool, before):
        assert torch.equal(x[[7, 9]], w[[3, 4]])
    table, lengths = _i32([[7, 9, -1], [-1, -1, -1]]), _i32([6, 0])
    refs = _i32([0] * 7 + [1, 0, 1, 0, 0])
    table, lengths, refs = nx.fork_sequences(pool[0], pool[1], table, lengths, refs, _i32([0]),
                                             _i32([1]), scales=pool[2])
    assert table.tolist() == [[7, 9, -1], [7, 0, -1]] and lengths.tolist() == [6, 6]
    for x in pool:
        assert torch.equal(x[0, :, :2], x[9, :, :2])
    table, refs = nx.compact_pages(pool[0], pool[1], table, refs, scales=pool[2])
    assert table.tolist() == [[1, 2, -1], [1, 0, -1]] and refs.tolist()[:3] == [1, 2, 1]
    for x, w in zip(pool, before):
        assert torch.equal(x[1], w[3]) and torch.equal(x[2], w[4])


def test_refusals():
    k, v, s = _pool(4, 2, 4, 16, 16, 4, torch.float32)
    t, n = _i32([[0, 1]]), _i32([5])
    q = torch.zeros(1, 4, 16)
    att = nx.quantized_paged_attention
    for args in (
        (q, k.float(), v, s, t, n), (q, k, v, s.int(), t, n), (q, k, v, s[..., :3], t, n),
        (q, k, v[:3], s, t, n), (q, k[0], v, s, t, n), (q[0], k, v, s, t, n),
        (q[..., :12], k, v, s, t, n), (q[:, :3], k, v, s, t, n), (q, k, v, s, t.long(), n),
        (q, k, v, s, t, n.long()), (q, k, v, s, _i32([[0], [1]]), n), (q, k, v, s, t[:, :0], n),
        (q, k[:0], v[:0], s[:0], t, n),
    ):
        with pytest.raises(ValueError, match='quantized_paged_attention'):
            att(*args)
    x = torch.zeros(2, 3, 16)
    o, st = _i32([0, 3]), _i32([0])
    write = nx.write_quantized_pages
    for args in (
        (k, v, s, x[0], x, t, st, o), (k, v, s, x, x[:, :2], t, st, o),
        (k, v, s, x[:1], x, t, st, o), (k, v, s, x[..., :8], x, t, st, o),
        (k, v, s, x[..., :6], x, t, st, o), (k, v, s, x, x, t, st), (k, v, s, x, x, t, st.long(), o),
        (k, v, s, x, x, t, st, o.long()), (k, v, s, x, x, t, st, _i32([0])),
        (k, v, s[:, :, :1].expand(-1, -1, 4, -1), x, x, t, st, o),
        (k[:1].expand(4, -1, -1, -1), v, s, x, x, t, st, o),
        (k, v, s, x.clone().requires_grad_(True), x, t, st, o),
    ):
        with pytest.raises(ValueError, match='write_quantized_pages'):
            write(*args)
    read = nx.read_quantized_pages
    for args, kw in (
        ((k, v, s, t, st, o), {}), ((k, v, s, t, st, o, -1), {}), ((k, v, s, t, st, None, 2), {}),
        ((k, v, s, t, st, o, 3), {'bits': 2}), ((k, v, s, t.float(), st, o, 3), {}),
    ):
        with pytest.raises(ValueError, match='read_quantized_pages'):
            read(*args, **kw)
    with pytest.raises(ValueError, match='copy_pages'):
        nx.copy_pages(k, v, [0], [1], scales=s[:2])
    with pytest.raises(ValueError, match='fork_sequences'):
        nx.fork_sequences(k, v.float(), t, n, _i32([1] * 4), st, st, scales=s)


def test_nothing_to_do():
    pool = _pool(4, 2, 4, 16, 24, 4, torch.float32)
    before = [x.clone() for x in pool]
    t = _i32([[0, 1]])
    nx.write_quantized_pages(*pool, torch.zeros(2, 0, 16), torch.zeros(2, 0, 24), t, _i32([0]),
                             _i32([0, 0]))
    assert all(torch.equal(a, b) for a, b in zip(pool, before))
    k, v = nx.read_quantized_pages(*pool, t, _i32([0]), _i32([0, 0]), 0)
    assert k.shape == (2, 0, 16) and v.shape == (2, 0, 24)
    out = nx.quantized_paged_attention(torch.zeros(0, 4, 16), *pool, t[:0], _i32([]))
    assert out.shape == (0, 4, 24)

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
    x = x.to(dt).repeat(1, 5, 1)
    pool = _pool(3, 1, 16, 32, 32, bits, dt)
    table, starts, off = _i32([[1]]), _i32([2]), _i32([0, 5])
    nx.write_quantized_pages(*pool, x, x, table, starts, off)
    sc = pool[2]
    sc[1, 0, 4, 0], sc[1, 0, 5, 1], sc[1, 0, 6, 2] = math.inf, math.inf, math.nan
    k, v = nx.read_quantized_pages(*pool, table, starts, off, 5, bits=bits)
    for y in (k[:, :2], v[:, :4]):
        assert torch.isfinite(y).all() and float(y.max()) == most
        off_by = (y.double() - x[:, :y.shape[1]].double()).abs().max()
        step = (most - lo) / top
        assert off_by <= step / 2 + (most - lo) * torch.finfo(dt).eps
    assert not torch.isfinite(k[0, 2]).any() and (k[0, 3] == math.inf).all()
    assert torch.isnan(v[0, 4]).all()


# ---------------------------------------------------------------------------
# C ABI
# ---------------------------------------------------------------------------


def _desc(P=8, Hk=2, PS=16, D=64, Dv=64, dtype=_lib.NXA_BF16, bits=4):
    d = _lib.NxaQuantPoolDesc()
    d.P, d.Hk, d.PS, d.D, d.Dv, d.io_dtype, d.bits = P, Hk, PS, D, Dv, dtype, bits
    kb, vb = D * bits // 8, Dv * bits // 8
    d.k_str[:] = (Hk * PS * kb, PS * kb)
    d.v_str[:] = (Hk * PS * vb, PS * vb)
    d.s_str[:] = (Hk * PS * 4, PS * 4)
    return d


def _rc(fn, *args):
    return fn(*args), _lib.lib().nxa_last_error().decode()


def test_pool_check_codes():
    check = _lib.lib().nxa_quant_pool_check
    assert check(ctypes.byref(_desc())) == 0
    assert check(ctypes.byref(_desc(bits=8, D=256, Dv=8, dtype=_lib.NXA_F32))) == 0
    assert check(None) == _lib.NXA_E_ARG
    for bad, code in (
        (_desc(dtype=9), _lib.NXA_E_DTYPE), (_desc(bits=3), _lib.NXA_E_UNSUPPORTED),
        (_desc(P=0), _lib.NXA_E_SHAPE), (_desc(PS=(1 << 30) + 16), _lib.NXA_E_SHAPE),
        (_desc(Hk=(1 << 24) + 1), _lib.NXA_E_SHAPE),
        (_desc(D=260), _lib.NXA_E_UNSUPPORTED), (_desc(Dv=12), _lib.NXA_E_UNSUPPORTED),
    ):
        assert check(ctypes.byref(bad)) == code
    for field in ('k_str', 'v_str', 's_str'):
        for x in (-4, 6):
            d = _desc()
            getattr(d, field)[1] = x
            assert check(ctypes.byref(d)) == _lib.NXA_E_LAYOUT


def test_entry_points_check_before_any_launch():
    lib = _lib.lib()
    d = ctypes.byref(_desc())
    ok, odd = 1 << 20, (1 << 20) + 8
    s2 = _lib.I64x2(64, 128)

    def write(k_pages=ok, scales=ok, k=ok, T=4, table=ok, starts=ok, offsets=ok, B=2, M=3, ks=s2):
        return lib.nxa_quant_write(d, k_pages, ok, scales, k, ks, ok, s2, T, table, M, starts,
                                   offsets, B, M, None)

    for kw, code in (
        ({'k_pages': None}, _lib.NXA_E_ARG), ({'scales': odd}, _lib.NXA_E_LAYOUT),
        ({'k': odd}, _lib.NXA_E_LAYOUT), ({'T': 0}, _lib.NXA_E_SHAPE),
        ({'T': 1 << 26}, _lib.NXA_E_SHAPE), ({'table': None}, _lib.NXA_E_ARG),
        ({'starts': None}, _lib.NXA_E_ARG), ({'offsets': None}, _lib.NXA_E_SHAPE),
        ({'B': 0}, _lib.NXA_E_SHAPE), ({'ks': _lib.I64x2(4, 128)}, _lib.NXA_E_LAYOUT),
        ({'ks': None}, _lib.NXA_E_ARG),
    ):
        assert write(**kw) == code, kw

    need = lib.nxa_quant_paged_workspace_bytes(d, 4, 3000, 8)
    assert need > 0 and lib.nxa_quant_paged_workspace_bytes(d, 4, 3, 8) == 0
    assert lib.nxa_quant_paged_workspace_bytes(d, 4, 3000, 7) == 0

    def attend(H=8, M=3000, q=ok, ws=ok, size=need, lengths=ok):
        return lib.nxa_quant_paged_fwd(d, ok, ok, ok, q, s2, ok, M, lengths, 4, M, H, 1.0, ok, s2,
                                       ws, size, None)

    for kw, code in (
        ({'H': 7}, _lib.NXA_E_SHAPE), ({'M': 1 << 27}, _lib.NXA_E_SHAPE),
        ({'q': odd}, _lib.NXA_E_LAYOUT), ({'ws': None}, _lib.NXA_E_WORKSPACE),
        ({'size': need - 1}, _lib.NXA_E_WORKSPACE), ({'lengths': None}, _lib.NXA_E_ARG),
    ):
        assert attend(**kw) == code, kw

    one = (ctypes.c_int32 * 1)(8)
    assert lib.nxa_quant_copy(d, ok, ok, ok, one, one, 1, None) == _lib.NXA_E_ARG
    assert lib.nxa_quant_copy(d, ok, ok, odd, one, one, 1, None) == _lib.NXA_E_LAYOUT
    assert lib.nxa_quant_fork(d, ok, ok, None, 1, 1, ok, ok, ok, ok, ok, 1, ok + 64, ok + 64,
                              ok + 64, ok, 1 << 20, None) == _lib.NXA_E_ARG
    assert lib.nxa_quant_compact(d, ok, ok, ok, 4, ok, ok, ok, ok + 64, ok, 1 << 20,
                                 None) == _lib.NXA_E_ARG
