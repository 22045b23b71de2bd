"""Host side of the paged cache: the reference engine against plain loops,
refusals, and the C ABI's checks (CPU only)."""

from __future__ import annotations

import contextlib
import ctypes

import _paged_plain as plain
import numpy as np
import pytest
import torch

import nitrix_amd as nx
from nitrix_amd import _lib


def _i32(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32)


def _pools(rng, p, hk, ps, d, dv):
    return rng.standard_normal((p, hk, ps, d)), rng.standard_normal((p, hk, ps, dv))


@pytest.mark.parametrize('ps', [1, 5, 16])
@pytest.mark.parametrize('h, hk', [(6, 2), (3, 3), (20, 1)])
def test_attention_reference(ps, h, hk):
    rng = np.random.default_rng(ps)
    p, m, b = 40, 6, 7
    k, v = _pools(rng, p, hk, ps, 8, 4)
    table, lengths, _ = plain.cache(rng, b, m, p, ps)
    lengths[0], lengths[1], lengths[2] = -3, m * ps + 9, 0
    table[3, 0] = p + 5
    unused = np.ones((p, ps), bool)
    for i in range(b):
        for j in range(min(max(lengths[i], 0), m * ps)):
            if 0 <= table[i, j // ps] < p:
                unused[table[i, j // ps], j % ps] = False
    for x in (k, v):
        x.transpose(0, 2, 1, 3)[unused] = np.nan
    q = rng.standard_normal((b, h, 8))
    want, _ = plain.attention(q, k, v, table, lengths, 0.3)
    got = nx.paged_attention(*map(torch.from_numpy, (q, k, v)), _i32(table), _i32(lengths), scale=0.3)
    np.testing.assert_allclose(got.numpy(), want, atol=1e-13)
    assert (want[0] == 0).all() and (want[2] == 0).all()


def test_attention_reference_is_differentiable():
    rng = np.random.default_rng(0)
    k, v = (torch.from_numpy(x).requires_grad_(True) for x in _pools(rng, 5, 1, 2, 4, 4))
    q = torch.randn(2, 2, 4, dtype=torch.float64, requires_grad=True)
    table, lengths = _i32([[0, 3], [4, -1]]), _i32([3, 1])
    assert torch.autograd.gradcheck(
        lambda *a: nx.paged_attention(*a, table, lengths), (q, k, v))


@pytest.mark.parametrize('packed', [False, True])
def test_write_reference(packed):
    rng = np.random.default_rng(1)
    p, hk, ps, m, b = 30, 2, 4, 5, 6
    k0, v0 = _pools(rng, p, hk, ps, 8, 4)
    table = rng.permutation(p)[:b * m].reshape(b, m).astype(np.int32)
    table[2, 1] = -1
    table[3, 0] = p
    starts = np.array([0, 3, 2, 1, -2, 19], np.int32)
    offsets = np.array([2, 5, 5, 9, 12, 16, 19], np.int32) if packed else None
    t = 21 if packed else b
    k, v = rng.standard_normal((hk, t, 8)), rng.standard_normal((hk, t, 4))
    want = k0.copy(), v0.copy()
    plain.write(*want, k, v, table, starts, offsets)
    got = torch.from_numpy(k0.copy()), torch.from_numpy(v0.copy())
    nx.write_pages(*got, torch.from_numpy(k), torch.from_numpy(v), _i32(table), _i32(starts),
                   _i32(offsets) if packed else None)
    for a, w in zip(got, want):
        np.testing.assert_array_equal(a.numpy(), w)


@pytest.mark.parametrize('seed', range(4))
def test_page_management_reference(seed):
    rng = np.random.default_rng(seed)
    b, m, p, ps = 9, 5, 30, 3
    state = plain.cache(rng, b, m, p, ps)
    k, v = _pools(rng, p, 2, ps, 4, 4)
    tk, tv = torch.from_numpy(k.copy()), torch.from_numpy(v.copy())
    ts = [_i32(x) for x in state]

    def same(got, want):
        for a, w in zip(got, want):
            np.testing.assert_array_equal(a.numpy(), w)
            assert a.dtype == torch.int32

    rows = [1, 1, 4, -2, b]
    want = plain.free(*state, rows)
    got = nx.free_sequences(*ts, _i32(rows))
    same(got, want)
    src, dst = [0, 2, 5, 2, 6, 9, 7], [1, 4, 4, 1, 6, 2, -1]
    want = plain.fork(k, v, *want, src, dst)
    got = nx.fork_sequences(tk, tv, *got, _i32(src), _i32(dst))
    same(got, want)
    np.testing.assert_array_equal(tk.numpy(), k)
    counts = rng.integers(-1, 9, b)
    want = plain.extend(*want, counts, ps)
    got = nx.extend_sequences(*got, _i32(counts), ps)
    same(got, want)
    counts[:] = 100  # more than there is
    want = plain.extend(*want, counts, ps)
    got = nx.extend_sequences(*got, _i32(counts), ps)
    same(got, want)
    want = plain.free(*want, [0, 3, 8])
    got = nx.free_sequences(*got, _i32([0, 3, 8]))
    want2 = plain.compact(k, v, want[0], want[2])
    got2 = nx.compact_pages(tk, tv, got[0], got[2])
    same(got2, want2)
    np.testing.assert_array_equal(tk.numpy(), k)
    np.testing.assert_array_equal(tv.numpy(), v)


def test_copy_reference():
    k, v = torch.arange(12.).reshape(6, 1, 2, 1), -torch.arange(12.).reshape(6, 1, 2, 1)
    want = k.clone()
    want[[4, 0]] = want[[1, 2]]
    nx.copy_pages(k, v, [1, 2], [4, 0])
    assert torch.equal(k, want) and torch.equal(v, -want)
    nx.copy_pages(k, v, [], [])


@pytest.mark.parametrize('src, dst, match', [
    ([1], [1], 'both a source and a target'),
    ([1, 2], [3, 3], 'target of two'),
    ([1, 2], [2, 4], 'both a source and a target'),
    ([6], [1], 'outside'),
    ([1], [-1], 'outside'),
    ([1, 2], [3], 'sources'),
    ([1.5], [2], 'page numbers'),
    ([[1]], [2], 'page numbers'),
])
def test_copy_refusals(src, dst, match):
    k = torch.zeros(6, 1, 2, 4)
    with pytest.raises(ValueError, match=match):
        nx.copy_pages(k, k.clone(), src, dst)


def _args(**kw):
    a = dict(q=torch.zeros(3, 4, 8), k_pages=torch.zeros(5, 2, 4, 8), v_pages=torch.zeros(5, 2, 4, 8),
             page_table=_i32(np.zeros((3, 2))), lengths=_i32([1, 2, 3]))
    a.update(kw)
    return a


@pytest.mark.parametrize('kw, match', [
    (dict(k_pages=torch.zeros(5, 2, 8)), 'pages must be'),
    (dict(v_pages=torch.zeros(4, 2, 4, 8)), 'same, non-empty'),
    (dict(k_pages=torch.zeros(0, 2, 4, 8), v_pages=torch.zeros(0, 2, 4, 8)), 'non-empty'),
    (dict(v_pages=torch.zeros(5, 2, 4, 8).half()), 'share device and dtype'),
    (dict(q=torch.zeros(3, 4, 16)), 'd=8'),
    (dict(q=torch.zeros(3, 3, 8)), 'multiple'),
    (dict(q=torch.zeros(3, 0, 8)), 'multiple'),
    (dict(page_table=torch.zeros(3, 2, dtype=torch.long)), 'int32'),
    (dict(page_table=_i32(np.zeros((2, 2)))), 'int32 of shape'),
    (dict(page_table=_i32(np.zeros((3, 0)))), 'no columns'),
    (dict(lengths=_i32([1, 2])), 'lengths'),
    (dict(lengths=torch.zeros(3, dtype=torch.int32, device='meta')), 'lengths is on'),
    (dict(q=torch.zeros(3, 4, 8, device='meta')), 'q is on'),
])
def test_attention_refusals(kw, match):
    with pytest.raises(ValueError, match=match):
        nx.paged_attention(**_args(**kw))


def test_no_sequences():
    out = nx.paged_attention(**_args(q=torch.zeros(0, 4, 8), page_table=_i32(np.zeros((0, 2))),
                                     lengths=_i32([])))
    assert out.shape == (0, 4, 8)


@pytest.mark.parametrize('kw, match', [
    (dict(k=torch.zeros(1, 3, 8)), 'k and v must be'),
    (dict(v=torch.zeros(2, 3, 4)), 'k and v must be'),
    (dict(k=torch.zeros(2, 4, 8), v=torch.zeros(2, 4, 8)), 'one token a sequence'),
    (dict(starts=_i32([0, 1])), 'starts'),
    (dict(offsets=_i32([0, 1, 2])), 'offsets'),
    (dict(page_table=_i32(np.zeros((3, 0)))), 'must not be empty'),
    (dict(k=torch.zeros(2, 3, 8, requires_grad=True)), 'not differentiable'),
    (dict(k_pages=torch.zeros(1, 2, 4, 8).expand(5, 2, 4, 8)), 'share memory'),
])
def test_write_refusals(kw, match):
    a = dict(k_pages=torch.zeros(5, 2, 4, 8), v_pages=torch.zeros(5, 2, 4, 8),
             k=torch.zeros(2, 3, 8), v=torch.zeros(2, 3, 8), page_table=_i32(np.zeros((3, 2))),
             starts=_i32([0, 1, 2]))
    a.update(kw)
    with pytest.raises(ValueError, match=match):
        nx.write_pages(**a)


def test_management_refusals():
    t, n, c = _i32(np.zeros((3, 2))), _i32([0, 0, 0]), _i32(np.zeros(5))
    k = torch.zeros(5, 1, 4, 8)
    with pytest.raises(ValueError, match='rows must be int32'):
        nx.free_sequences(t, n, c, torch.tensor([1]))
    with pytest.raises(ValueError, match='refs must count'):
        nx.free_sequences(t, n, _i32([]), _i32([0]))
    with pytest.raises(ValueError, match='page_size'):
        nx.extend_sequences(t, n, c, n, 0)
    with pytest.raises(ValueError, match='2\\^31'):
        nx.extend_sequences(t, n, c, n, 1 << 30)
    with pytest.raises(ValueError, match='counts'):
        nx.extend_sequences(t, n, c, c, 4)
    with pytest.raises(ValueError, match='refs'):
        nx.fork_sequences(k, k.clone(), t, n, n, _i32([0]), _i32([1]))
    with pytest.raises(ValueError, match='dst'):
        nx.fork_sequences(k, k.clone(), t, n, c, _i32([0]), _i32([1, 2]))
    with pytest.raises(ValueError, match='refs'):
        nx.compact_pages(k, k.clone(), t, n)
    with pytest.raises(ValueError, match='not differentiable'):
        nx.compact_pages(k.clone().requires_grad_(True), k.clone(), t, c)
    with pytest.raises(nx.NitrixBackendError):
        nx.compact_pages(k, k.clone(), t, c, backend='hip')


def _pool(**kw):
    d = _lib.NxaPoolDesc()
    for n, x in {**dict(P=10, Hk=2, PS=16, D=64, Dv=64, io_dtype=_lib.NXA_BF16), **kw}.items():
        if not n.endswith('_str'):
            setattr(d, n, x)
    for n in ('k_str', 'v_str'):
        getattr(d, n)[:] = kw.get(n, (2048, 1024, 64))
    return d


@pytest.mark.parametrize('kw, code', [
    ({}, _lib.NXA_OK),
    (dict(P=0), _lib.NXA_E_SHAPE),
    (dict(PS=0), _lib.NXA_E_SHAPE),
    (dict(P=(1 << 30) + 1), _lib.NXA_E_SHAPE),
    (dict(PS=(1 << 30) + 1), _lib.NXA_E_SHAPE),
    (dict(Dv=0), _lib.NXA_E_SHAPE),
    (dict(D=12), _lib.NXA_E_UNSUPPORTED),
    (dict(D=512), _lib.NXA_E_UNSUPPORTED),
    (dict(io_dtype=7), _lib.NXA_E_DTYPE),
    (dict(k_str=(2048, 1024, 60)), _lib.NXA_E_LAYOUT),
    (dict(v_str=(-8, 1024, 64)), _lib.NXA_E_LAYOUT),
    (dict(v_str=(8, 8, 1 << 26)), _lib.NXA_E_LAYOUT),
])
def test_c_pool_check(kw, code):
    assert _lib.lib().nxa_pool_check(ctypes.byref(_pool(**kw))) == code


def test_c_entries_refuse_before_any_launch():
    lib, P, s = _lib.lib(), 1 << 12, _lib.I64x2(128, 64)
    d = ctypes.byref(_pool())
    need = lib.nxa_paged_workspace_bytes(d, 4, 100, 6)
    assert need > 0 and lib.nxa_paged_workspace_bytes(d, 4, 100, 5) == 0

    def att(B=4, M=100, H=6, ws=P, n=need, table=P, q=P, pool=d, rs=8):
        return lib.nxa_paged_fwd(pool, P, P, q, s, table, rs, P, B, M, H, 0.1, P, s, ws, n, None)
    assert att(H=5) == _lib.NXA_E_SHAPE
    assert att(B=0) == _lib.NXA_E_SHAPE
    assert att(B=1 << 20, M=1 << 20) == _lib.NXA_E_SHAPE
    assert att(ws=None) == _lib.NXA_E_WORKSPACE
    assert att(n=need - 1) == _lib.NXA_E_WORKSPACE
    assert att(table=None) == _lib.NXA_E_ARG
    assert att(q=P + 2) == _lib.NXA_E_LAYOUT
    assert att(rs=-1) == _lib.NXA_E_LAYOUT
    assert att(pool=None) == _lib.NXA_E_ARG
    w = lib.nxa_pages_write
    assert w(d, P, P, P, s, P, s, 5, P, 8, P, None, 4, 8, None) == _lib.NXA_E_SHAPE
    assert w(d, P, P, P, s, P, s, 0, P, 8, P, P, 4, 8, None) == _lib.NXA_E_SHAPE
    assert w(d, P, P, P, s, P, s, 4, P, 8, None, None, 4, 8, None) == _lib.NXA_E_ARG
    ints = (ctypes.c_int32 * 2)(1, 10)
    assert lib.nxa_pages_copy(d, P, P, ints, ints, 2, None) == _lib.NXA_E_ARG
    assert lib.nxa_pages_copy(d, P, P, None, None, 1, None) == _lib.NXA_E_ARG
    assert lib.nxa_pages_free(2, 2, 4, P, P, P, P, 1, P, 2 * P, 3 * P, None) == _lib.NXA_E_ARG
    assert lib.nxa_pages_free(2, 2, 4, P, P, P, None, 1, 2 * P, 2 * P, 2 * P, None) == _lib.NXA_E_ARG
    assert lib.nxa_pages_extend(2, 2, 4, 8, P, P, P, P, 2 * P, 2 * P, 2 * P, P, 15,
                                None) == _lib.NXA_E_WORKSPACE
    assert lib.nxa_pages_extend(2, 1 << 20, 4, 1 << 11, P, P, P, P, 2 * P, 2 * P, 2 * P, P, 16,
                                None) == _lib.NXA_E_SHAPE
    assert lib.nxa_pages_free(2, 2, (1 << 30) + 1, P, P, P, P, 1, 2 * P, 2 * P, 2 * P,
                              None) == _lib.NXA_E_SHAPE
    assert lib.nxa_pages_fork(d, P, P, 2, 2, P, P, P, P, P, 1, 2 * P, 2 * P, 2 * P, None, 0,
                              None) == _lib.NXA_E_WORKSPACE
    assert lib.nxa_pages_compact(d, P, P, 4, P, P, 2 * P, 2 * P, P, 8, None) == _lib.NXA_E_WORKSPACE
    assert lib.nxa_pages_compact(d, P, P, 4, P, P, P, 2 * P, P, 1 << 20, None) == _lib.NXA_E_ARG


def test_forward_mode_is_left_to_the_reference_engine_or_refused():
    """A tensor with a tangent need not have requires_grad."""
    from torch.autograd import forward_ad

    from nitrix_amd.paged import HipNotTileable, _paged_hip

    a = _args()
    a['k_pages'], a['v_pages'] = torch.randn(5, 2, 4, 8), torch.randn(5, 2, 4, 8)
    t, n, c = _i32(np.zeros((3, 2))), _i32([3, 4, 5]), _i32([1, 0, 1, 1, 0])
    with forward_ad.dual_level():
        for name in ('q', 'k_pages', 'v_pages'):
            x = a[name]
            dual = {**a, name: forward_ad.make_dual(x, torch.randn_like(x))}
            assert forward_ad.unpack_dual(nx.paged_attention(**dual)).tangent is not None
            with pytest.raises(HipNotTileable, match='forward-mode'):
                _paged_hip(*dual.values(), 1.0)
        k = forward_ad.make_dual(torch.randn(2, 3, 8), torch.randn(2, 3, 8))
        pool = forward_ad.make_dual(a['k_pages'].clone(), torch.randn(5, 2, 4, 8))
        v = torch.zeros(2, 3, 8)
        for call in (lambda: nx.write_pages(a['k_pages'], a['v_pages'], k, v, t, n),
                     lambda: nx.write_pages(pool, a['v_pages'], v, v, t, n),
                     lambda: nx.fork_sequences(pool, a['v_pages'], t, n, c, _i32([0]), _i32([1])),
                     lambda: nx.compact_pages(pool, a['v_pages'], t, c),
                     lambda: nx.copy_pages(pool, a['v_pages'], [0], [1])):
            with pytest.raises(ValueError, match='forward-mode'):
                call()


def test_extents_past_a_grid_are_declined(monkeypatch):
    """A launch holds less than 2^32 threads; attention's rows past 2^24 are
    shared by its blocks instead of one each."""
    lib, P, s = _lib.lib(), 1 << 12, _lib.I64x2(128, 64)
    d = _pool()
    small = lib.nxa_paged_workspace_bytes(ctypes.byref(d), (1 << 23) - 1, 1, 2)
    assert small == 0 and lib.nxa_paged_workspace_bytes(ctypes.byref(d), 1 << 23, 1, 2) > 0
    w = lib.nxa_pages_write
    assert w(ctypes.byref(d), P, P, P, s, P, s, 1 << 26, P, 8, P, P, 4, 8, None) == _lib.NXA_E_SHAPE
    n = 1 << 24
    assert lib.nxa_pages_free(2, 2, 4, P, P, P, P, n, 2 * P, 2 * P, 2 * P, None) == _lib.NXA_E_SHAPE
    assert lib.nxa_pages_fork(ctypes.byref(d), P, P, 2, 2, P, P, P, P, P, n, 2 * P, 2 * P, 2 * P, P,
                              1 << 40, None) == _lib.NXA_E_SHAPE
    ints = (ctypes.c_int32 * 400)(*range(400))
    many = _pool(Hk=41944, P=400, k_str=(0, 1024, 64), v_str=(0, 1024, 64))
    assert lib.nxa_pages_copy(ctypes.byref(many), P, P, ints, ints, 400, None) == _lib.NXA_E_SHAPE

    from nitrix_amd import paged

    def declined():
        _lib.check(lib.nxa_pool_check(ctypes.byref(_pool(P=0))))

    monkeypatch.setattr(paged, 'resolve_backend', lambda *a: 'hip')
    monkeypatch.setattr(paged, '_on', lambda dev: contextlib.nullcontext())
    nx.reset_fallback_state()
    with pytest.warns(nx.NitrixBackendFallback, match='must be positive'):
        assert paged._dispatch('f', 'auto', None, declined, lambda: 7, (), None) == 7


def test_fork_of_a_row_whose_last_tokens_are_in_no_page():
    """Nothing to copy: the new row ends with its whole pages instead of a page
    of whatever a free one holds, and no page is handed out for it."""
    table = _i32([[0, 1, -1, -1], [2, 9, -1, -1], [3, 4, -1, -1], [-1] * 4, [-1] * 4, [-1] * 4])
    lengths, refs = _i32([10, 6, 7, 0, 0, 0]), _i32([1, 1, 1, 1, 1, 0, 0, 0])
    k = torch.arange(8.).reshape(8, 1, 1, 1).expand(8, 1, 4, 4).contiguous()
    t, n, c = nx.fork_sequences(k, -k, table, lengths, refs, _i32([0, 1, 2]), _i32([3, 4, 5]))
    assert t[3:].tolist() == [[0, 1, -1, -1], [2, -1, -1, -1], [3, 5, -1, -1]]
    assert n.tolist() == [10, 6, 7, 8, 4, 7] and c.tolist() == [2, 2, 2, 2, 1, 1, 0, 0]
    assert (k[5, :, :3] == 4).all() and (k[6:] > 5).all()
