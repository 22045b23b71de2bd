"""Host side of packed attention: refusals, layouts, the reference engine
against a plain float64 implementation, the C ABI's checks (CPU only)."""

from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest
import torch

import nitrix_amd as nx
from nitrix_amd import _lib
from nitrix_amd.packed import (
    HipNotTileable,
    _check_tileable,
    _empty_like,
    _kernel_layout,
    packed_attention,
    reference_packed_attention,
)


def plain(q, k, v, ends, scale, causal):
    """float64, one (sequence, head) at a time."""
    q, k, v = (x.astype(np.float64) for x in (q, k, v))
    g = q.shape[0] // k.shape[0]
    out = np.zeros(q.shape[:2] + v.shape[2:])
    for a, b in zip(ends[:-1], ends[1:]):
        for h in range(q.shape[0]):
            if b <= a:
                continue
            s = scale * q[h, a:b] @ k[h // g, a:b].T
            if causal:
                s = np.where(np.tri(b - a, dtype=bool), s, -np.inf)
            p = np.exp(s - s.max(-1, keepdims=True))
            out[h, a:b] = p / p.sum(-1, keepdims=True) @ v[h // g, a:b]
    return out


def _inputs(h, hk, t, d, dv=None, seed=0):
    rng = np.random.default_rng(seed)
    return (rng.standard_normal((h, t, d)), rng.standard_normal((hk, t, d)),
            rng.standard_normal((hk, t, dv or d)))


@pytest.mark.parametrize('causal', [False, True])
@pytest.mark.parametrize('ends', [[0, 9], [0, 0, 4, 4, 9], [2, 3, 7], [0, 1], [5, 5]])
def test_reference_engine_matches_the_plain_form(ends, causal):
    q, k, v = _inputs(6, 2, 9, 8, 4)
    args = [torch.from_numpy(x) for x in (q, k, v)]
    got = reference_packed_attention(*args, torch.tensor(ends, dtype=torch.int32), causal=causal)
    want = plain(q, k, v, ends, 1 / math.sqrt(8), causal)
    # float64 throughout: a few units of the last place of values of order one
    np.testing.assert_allclose(got.numpy(), want, atol=1e-13)


def test_reference_engine_gradients_by_differences():
    q, k, v = (torch.from_numpy(x).requires_grad_(True) for x in _inputs(4, 2, 7, 4))
    off = torch.tensor([1, 3, 3, 6], dtype=torch.int32)
    assert torch.autograd.gradcheck(
        lambda *a: reference_packed_attention(*a, off, causal=True), (q, k, v))


def test_reference_engine_rows_of_no_sequence():
    q, k, v = (torch.from_numpy(x) for x in _inputs(2, 1, 6, 4))
    for x in (q, k, v):
        x[:, :1] = math.nan
        x[:, 5:] = math.inf
    ts = [x.requires_grad_(True) for x in (q, k, v)]
    out = packed_attention(*ts, torch.tensor([1, 3, 5], dtype=torch.int32))
    assert (out[:, [0, 5]] == 0).all() and torch.isfinite(out).all()
    grads = torch.autograd.grad(out.sum(), ts)
    for g in grads:
        assert (g[:, [0, 5]] == 0).all() and torch.isfinite(g).all()


def test_reference_engine_no_sequence_has_zero_gradients():
    ts = [torch.from_numpy(x).requires_grad_(True) for x in _inputs(2, 1, 3, 4)]
    out = packed_attention(*ts, torch.tensor([2, 2], dtype=torch.int32))
    assert (out == 0).all()
    for g in torch.autograd.grad(out.sum(), ts):
        assert (g == 0).all()


def test_empty_row_of_tokens():
    q, k, v = (torch.zeros(2, 0, 8) for _ in range(3))
    assert packed_attention(q, k, v, torch.tensor([0, 0], dtype=torch.int32)).shape == (2, 0, 8)


@pytest.mark.parametrize('change, match', [
    (dict(q=torch.zeros(1, 4, 9, 8)), 'ndim'),
    (dict(k=torch.zeros(2, 9, 16)), 'head-dim'),
    (dict(v=torch.zeros(2, 8, 8)), 'same tokens'),
    (dict(q=torch.zeros(5, 9, 8)), 'multiple'),
    (dict(v=torch.zeros(1, 9, 8)), 'multiple'),
    (dict(k=torch.zeros(0, 9, 8), v=torch.zeros(0, 9, 8)), 'multiple'),
    (dict(offsets=torch.tensor([0, 9])), 'int32'),
    (dict(offsets=torch.tensor([0], dtype=torch.int32)), 'at least one'),
    (dict(offsets=torch.zeros(2, 2, dtype=torch.int32)), 'int32'),
    (dict(offsets=torch.zeros(2, dtype=torch.int32, device='meta')), 'one device'),
])
def test_refusals(change, match):
    a = dict(q=torch.zeros(4, 9, 8), k=torch.zeros(2, 9, 8), v=torch.zeros(2, 9, 8),
             offsets=torch.tensor([0, 9], dtype=torch.int32))
    a.update(change)
    with pytest.raises(ValueError, match=match):
        packed_attention(**a)


def test_explicit_hip_off_the_device_raises():
    z = torch.zeros(2, 3, 8)
    with pytest.raises(nx.NitrixBackendError):
        packed_attention(z, z, z, torch.tensor([0, 3], dtype=torch.int32), backend='hip')


def test_declined_types_and_head_dims():
    for dt, d, dv in ((torch.float64, 8, 8), (torch.bfloat16, 12, 8), (torch.float32, 8, 6),
                      (torch.bfloat16, 264, 8)):
        with pytest.raises(HipNotTileable):
            _check_tileable(torch.zeros(2, 3, d, dtype=dt), torch.zeros(2, 3, d, dtype=dt),
                            torch.zeros(2, 3, dv, dtype=dt))
    with pytest.raises(HipNotTileable):
        _check_tileable(torch.zeros(2, 3, 8), torch.zeros(2, 3, 8).half(), torch.zeros(2, 3, 8))


def test_layouts_read_in_place_and_copied():
    x = torch.zeros(10, 4, 8, dtype=torch.bfloat16).transpose(0, 1)
    assert _kernel_layout(x) is x
    assert _empty_like(x, 16).transpose(0, 1).is_contiguous()
    fused = torch.zeros(10, 3, 4, 8, dtype=torch.bfloat16)[:, 1].transpose(0, 1)
    assert _kernel_layout(fused) is fused
    odd = torch.zeros(4, 10, 9, dtype=torch.bfloat16)[:, :, :8]
    assert _kernel_layout(odd).is_contiguous()
    flip = torch.zeros(4, 8, 10, dtype=torch.bfloat16).transpose(1, 2)
    assert _kernel_layout(flip).is_contiguous()
    assert _empty_like(torch.zeros(4, 10, 8), 8).is_contiguous()


def _desc(**kw):
    d = _lib.NxaPackedDesc()
    base = dict(T=100, nseq=3, H=8, Hk=2, D=64, Dv=64, io_dtype=_lib.NXA_BF16, causal=1, scale=0.1)
    for n, x in {**base, **kw}.items():
        if not n.endswith('_str'):
            setattr(d, n, x)
    for n in ('q_str', 'k_str', 'v_str', 'o_str'):
        getattr(d, n)[:] = kw.get(n, (6400, 64))
    return d


@pytest.mark.parametrize('kw, code', [
    ({}, _lib.NXA_OK),
    (dict(T=0), _lib.NXA_E_SHAPE),
    (dict(nseq=0), _lib.NXA_E_SHAPE),
    (dict(Hk=3), _lib.NXA_E_SHAPE),
    (dict(Hk=0), _lib.NXA_E_SHAPE),
    (dict(T=1 << 30, H=64, Hk=2), _lib.NXA_E_SHAPE),
    (dict(D=0), _lib.NXA_E_SHAPE),
    (dict(D=264), _lib.NXA_E_UNSUPPORTED),
    (dict(Dv=12), _lib.NXA_E_UNSUPPORTED),
    (dict(io_dtype=9), _lib.NXA_E_DTYPE),
    (dict(q_str=(6400, 60)), _lib.NXA_E_LAYOUT),
    (dict(k_str=(-8, 64)), _lib.NXA_E_LAYOUT),
    (dict(v_str=(8, 1 << 26)), _lib.NXA_E_LAYOUT),
])
def test_c_check(kw, code):
    assert _lib.lib().nxa_packed_check(ctypes.byref(_desc(**kw))) == code


def test_c_entries_refuse_before_any_launch():
    lib = _lib.lib()
    d = _desc()
    P, s = 1 << 12, _lib.I64x2(6400, 64)
    assert lib.nxa_packed_fwd(ctypes.byref(d), P, P, P, None, P, None, None, None) == _lib.NXA_E_ARG
    assert lib.nxa_packed_fwd(ctypes.byref(d), P + 8, P, P, P, P, None, None, None) == _lib.NXA_E_LAYOUT
    assert lib.nxa_packed_fwd(None, P, P, P, P, P, None, None, None) == _lib.NXA_E_ARG
    assert lib.nxa_packed_fwd(ctypes.byref(d), P, P, P, P, P, P + 4, None, None) == _lib.NXA_E_LAYOUT
    need = lib.nxa_packed_workspace_bytes(ctypes.byref(d))
    assert need >= 2 * 8 * 100 * 4
    assert lib.nxa_packed_workspace_bytes(ctypes.byref(_desc(T=0))) == 0

    def bwd(ws, n, lse=P, st=s):
        return lib.nxa_packed_bwd(ctypes.byref(d), P, P, P, P, P, None, lse, P, s, P, st, P, s, P, s,
                                  ws, n, None)
    assert bwd(None, need) == _lib.NXA_E_WORKSPACE
    assert bwd(P, need - 1) == _lib.NXA_E_WORKSPACE
    assert bwd(P + 16, need) == _lib.NXA_E_WORKSPACE
    assert bwd(P, need, lse=None) == _lib.NXA_E_ARG
    assert bwd(P, need, st=_lib.I64x2(6400, 63)) == _lib.NXA_E_LAYOUT


def _readable(x):
    epc = 16 // x.element_size()
    return (x.data_ptr() % 16 == 0 and x.stride(2) == 1 and x.stride(0) % epc == 0
            and x.stride(1) % epc == 0)


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
def test_contiguous_views_the_kernels_cannot_read_are_copied(dtype):
    """Slices of a flat buffer off a 16-byte boundary, and axes of size one
    whose stride is no multiple of 16 bytes, count as contiguous."""
    flat = torch.randn(1 + 4 * 10 * 8).to(dtype)
    views = [flat[1:].view(4, 10, 8), flat[1:1 + 80].view(1, 10, 8), flat[1:1 + 32].view(4, 1, 8),
             torch.as_strided(flat, (1, 10, 8), (83, 8, 1)),
             torch.as_strided(flat, (4, 1, 8), (8, 9, 1)),
             torch.as_strided(flat, (1, 1, 8), (3, 1 << 27, 1))]
    for x in views:
        assert x.is_contiguous() and not _readable(x)
        y = _kernel_layout(x)
        assert _readable(y) and torch.equal(x, y)


def test_forward_mode_is_left_to_the_reference_engine():
    """A tensor with a tangent need not have requires_grad: the fused engine
    declines it, the reference engine's tangent is that of differences."""
    from torch.autograd import forward_ad

    from nitrix_amd.packed import packed_attention_hip

    off = torch.tensor([0, 4, 7], dtype=torch.int32)
    ins = [torch.from_numpy(x) for x in _inputs(4, 2, 7, 8, seed=3)]
    for i in range(3):
        t = torch.from_numpy(np.random.default_rng(i).standard_normal(ins[i].shape))
        with forward_ad.dual_level():
            dual = [forward_ad.make_dual(x, t) if n == i else x for n, x in enumerate(ins)]
            out, tangent = forward_ad.unpack_dual(packed_attention(*dual, off, causal=True))
            with pytest.raises(HipNotTileable, match='forward-mode'):
                packed_attention_hip(*(x.float() for x in dual), off, scale=1.0)
        ahead, behind = (packed_attention(*(x + s * t if n == i else x for n, x in enumerate(ins)),
                                          off, causal=True) for s in (2.0 ** -14, -2.0 ** -14))
        # (float64: rounding 2^-53 / 2^-14 of values of order one, and 2^-28 of
        # a third derivative of some hundred)
        torch.testing.assert_close(tangent, (ahead - behind) * 2.0 ** 13, atol=1e-5, rtol=0)


def test_no_part_of_a_group_is_without_a_head():
    """Blocks that share a group's query heads take ceil(G / parts) each: the
    workspace has as many planes of dk and dv as that takes."""
    lib, seen = _lib.lib(), set()
    for g in range(1, 41):
        for t in [65536 // n + 1 for n in range(1, 41)] + [512, 100000, 130000]:
            for nseq in (1, 200):
                d = _desc(T=t, nseq=nseq, H=g, Hk=1, D=8, Dv=8)
                rows = -(-g * t * 4 // 256) * 256
                more = lib.nxa_packed_workspace_bytes(ctypes.byref(d)) - 2 * rows
                parts, odd = divmod(more, 4 * t * 16)
                assert odd == 0 and parts != 1 and parts <= g
                parts = max(parts, 1)
                per = -(-g // parts)
                assert (parts - 1) * per < g, (g, t, nseq, parts)
                seen.add((g, parts))
    assert {(7, 4), (16, 1), (16, 4), (16, 6), (16, 8), (16, 16), (5, 3)} <= seen


@pytest.mark.parametrize('kw, fwd, bwd', [
    # 128 rows and 256 threads a block, 512 in dK / dV
    (dict(H=64, Hk=64, T=64, nseq=(1 << 18) - 1), True, False),
    (dict(H=64, Hk=64, T=64, nseq=1 << 18), False, False),
    (dict(H=64, Hk=64, T=64, nseq=(1 << 17) - 1), True, True),
    (dict(H=64, Hk=64, T=64, nseq=1 << 17), True, False),
    (dict(H=2, Hk=2, T=(1 << 30) - 128 * 18, nseq=1), True, False),
    (dict(H=2, Hk=2, T=(1 << 29) - 128 * 18, nseq=1), True, True),
    # 8 waves: 256 rows and 512 threads
    (dict(H=2, Hk=2, T=(1 << 30) - 256 * 18, nseq=1, D=128), True, False),
    (dict(H=2, Hk=2, T=1 << 30, nseq=1, D=128), False, False),
    # float32: -delta of 16 rows a block of 256
    (dict(H=2, Hk=2, T=(1 << 27) - 16, nseq=1, io_dtype=_lib.NXA_F32), True, True),
    (dict(H=2, Hk=2, T=1 << 27, nseq=1, io_dtype=_lib.NXA_F32), True, False),
    # ... and 32-row blocks where they are few
    (dict(H=1, Hk=1, T=1000, nseq=(1 << 24) - 64, io_dtype=_lib.NXA_F32), True, True),
    (dict(H=1, Hk=1, T=1000, nseq=(1 << 24) - 62, io_dtype=_lib.NXA_F32), False, False),
])
def test_extents_past_a_grid_are_declined(kw, fwd, bwd):
    """A launch holds less than 2^32 threads."""
    lib, d = _lib.lib(), _desc(**kw)
    assert lib.nxa_packed_check(ctypes.byref(d)) == (_lib.NXA_OK if fwd else _lib.NXA_E_SHAPE)
    assert (lib.nxa_packed_workspace_bytes(ctypes.byref(d)) > 0) == bwd
    P, s = 1 << 12, _lib.I64x2(6400, 64)
    if not fwd:
        assert lib.nxa_packed_fwd(ctypes.byref(d), P, P, P, P, P, None, None,
                                  None) == _lib.NXA_E_SHAPE
    if not bwd:
        assert lib.nxa_packed_bwd(ctypes.byref(d), P, P, P, P, P, None, P, P, s, P, s, P, s, P, s,
                                  P, 1 << 40, None) == _lib.NXA_E_SHAPE


def test_extents_the_library_declines_fall_back(monkeypatch):
    from nitrix_amd import packed

    def declined(*args, **kw):
        _lib.check(_lib.lib().nxa_packed_check(ctypes.byref(_desc(T=0))))

    monkeypatch.setattr(packed, 'resolve_backend', lambda *a: 'hip')
    monkeypatch.setattr(packed, 'packed_attention_hip', declined)
    q, k, v = (torch.from_numpy(x) for x in _inputs(4, 2, 7, 8))
    off = torch.tensor([0, 7], dtype=torch.int32)
    nx.reset_fallback_state()
    with pytest.warns(nx.NitrixBackendFallback, match='must be positive'):
        out = packed_attention(q, k, v, off)
    assert torch.equal(out, reference_packed_attention(q, k, v, off))
