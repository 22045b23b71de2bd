"""Packed attention on the GPU at sizes on both sides of every rule that picks
a kernel: how many query heads a dK / dV block streams, 4 or 8 waves at head
dim 128, blocks of 128 or of 32 rows in float32, sequences ranked or searched
for.  Against the formulas in float64 on the device, with the bounds of
``test_hip_packed.py``; and stores beside the outputs, watched by guard bytes.
"""

from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest
import torch
from test_hip_packed import DT, E24, _ends, _off, _tokens, _train

from nitrix_amd import _lib, packed
from nitrix_amd.packed import packed_attention

pytestmark = pytest.mark.gpu


def _dev():
    return torch.device('cuda:0')


def _bounds(q, k, v, do, scale, causal, u, dt):
    """``test_hip_packed._bounds`` for several key-value heads at once, on the
    device: q, do [x, g, n, d], k, v [x, n, d] in float64."""
    n, d = k.shape[1:]
    dv_ = v.shape[2]
    f32 = dt == torch.float32
    sub = 2.0 ** -25 if dt == torch.float16 else 0.0
    subx = 0.0 if f32 else 2.0 ** -25
    kt, vt = (x.transpose(1, 2).contiguous()[:, None] for x in (k, v))
    kb, vb = k[:, None], v[:, None]
    s = scale * (q @ kt)
    es = (d + 8) * E24 * scale * (q.abs() @ kt.abs()) + 4 * E24 * s.abs()
    if causal:
        keep = torch.ones(n, n, dtype=torch.bool, device=q.device).tril()
        s = torch.where(keep, s, -math.inf)
        es = torch.where(keep, es, 0.0)
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - m)
    del s
    p /= p.sum(-1, keepdim=True)
    rp = es + es.amax(-1, keepdim=True) + (n + 16) * E24 + 8 * E24 * m.abs() + 16 * E24
    del es
    o = p @ vb
    to = (p * (rp + u + n * E24) + sub) @ vb.abs() + (u + 4 * E24) * o.abs()
    if do is None:
        return (o,), (to,)
    ado = do.abs()
    dp = do @ vt
    delta = (o * do).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    edp = (dv_ + 8) * E24 * (ado @ vt.abs())
    tod = to - u * (1 - 2 * u) * o.abs()
    edl = ((tod * ado).sum(-1, keepdim=True) + (dv_ + 8) * E24 * (o.abs() * ado).sum(-1, keepdim=True)
           + (0 if f32 else 2.0 ** -16) * delta.abs())
    tds = ds.abs() * (rp + (0 if f32 else 2.0 ** -11) + u) + p * (edp + edl) * (1 + rp)
    tds += sub + subx * ((dp - delta).abs() + edp + edl)
    rows = q.shape[1] * n
    dq = scale * (ds @ kb)
    tq = scale * ((tds + n * E24 * ds.abs()) @ kb.abs()) + (u + 4 * E24) * dq.abs()

    def over_heads(x, y):  # sum over the group's heads and rows
        return (x.transpose(2, 3).contiguous() @ y).sum(1)

    dk = scale * over_heads(ds, q)
    tk = scale * over_heads(tds + rows * E24 * ds.abs(), q.abs()) + (u + 4 * E24) * dk.abs()
    dv = over_heads(p, do)
    tv = over_heads(p * (rp + u + rows * E24) + sub, ado) + (u + 4 * E24) * dv.abs()
    return (o, dq, dk, dv), (to, tq, tk, tv)


def _check(q, k, v, ends, got, scale, causal, do=None, heads=None):
    """Every row of every sequence (of key-value heads ``heads``)."""
    dt = q.dtype
    u = 0.0 if dt == torch.float32 else torch.finfo(dt).eps / 2
    tiny = 4 * float(torch.finfo(dt).tiny if dt != torch.float16 else 2.0 ** -24)
    t, hk = q.shape[1], k.shape[0]
    g = q.shape[0] // hk
    heads = range(hk) if heads is None else heads
    for name, x in zip(('o', 'dq', 'dk', 'dv'), got):
        assert (x[:, :ends[0]] == 0).all() and (x[:, ends[-1]:] == 0).all(), f'{name}: rows of none'
    wide = lambda x: x.detach().reshape(hk, g, t, -1)  # noqa: E731
    for a, b in zip(ends[:-1], ends[1:]):
        if b == a:
            continue
        # (a few gigabytes a piece)
        per = max(1, (1 << 28) // (g * (b - a) ** 2))
        for h0 in range(0, len(heads), per):
            hs = list(heads)[h0:h0 + per]
            cut = lambda x: x.detach()[hs, a:b].double()  # noqa: E731
            cutq = lambda x: wide(x)[hs, :, a:b].double()  # noqa: E731
            want, tol = _bounds(cutq(q), cut(k), cut(v), None if do is None else cutq(do), scale,
                                causal, u, dt)
            parts = [cutq(got[0])]
            if do is not None:
                parts += [cutq(got[1]), cut(got[2]), cut(got[3])]
            for name, x, w, e in zip(('o', 'dq', 'dk', 'dv'), parts, want, tol):
                off = ~((x - w).abs() <= e + tiny)
                assert not off.any(), (
                    f'{name} rows {a}..{b} heads {hs}: {int(off.sum())} off, worst '
                    f'{float(((x - w).abs() / (e + tiny)).nan_to_num().max()):.2f} bounds, nan '
                    f'{int(x.isnan().sum())}')


def _lens(total, n, seed):
    """n lengths of very different size that add up to ``total``, some of them
    0 and 1."""
    rng = np.random.default_rng(seed)
    w = rng.lognormal(0.0, 1.0, n)
    if n > 8:
        w[rng.permutation(n)[:2]] = 0.0
    x = (w / w.sum() * total).astype(int)
    if n > 8:
        x[np.flatnonzero(x == 0)[0]] = 1
    x[x.argmax()] += total - x.sum()
    return x.tolist()


def _parts(h, hk, t, nseq):
    """Blocks that share a group's heads, from the workspace's size."""
    d = _lib.NxaPackedDesc()
    d.T, d.nseq, d.H, d.Hk, d.D, d.Dv, d.io_dtype = t, nseq, h, hk, 8, 8, _lib.NXA_BF16
    more = _lib.lib().nxa_packed_workspace_bytes(ctypes.byref(d)) - 2 * (-(-h * t * 4 // 256) * 256)
    return max(1, more // (4 * hk * t * 16))


def _run(dt, h, hk, d, dv, lens, lead, pad, causal, heads=None, seed=1):
    ends = _ends(lens, lead)
    t = ends[-1] + pad
    q, k, v = _tokens(t, h, hk, d, dv, DT[dt], seed)
    do = _tokens(t, h, h, dv, dv, DT[dt], seed + 1)[0]
    got = _train(q, k, v, _off(ends), do, causal=causal)
    torch.cuda.synchronize()
    _check(q, k, v, ends, got, 1 / math.sqrt(d), causal, do, heads)
    with torch.no_grad():
        assert torch.equal(packed_attention(q, k, v, _off(ends), causal=causal, backend='hip'), got[0])


# dtype, h, hk, d, dv, tokens, sequences, lead, pad, causal, parts
GROUPS = [
    ('bf16', 16, 8, 128, 128, 8240, 60, 2, 7, True, 1),
    ('bf16', 16, 8, 128, 128, 8240, 60, 0, 0, False, 1),
    ('f16', 24, 8, 64, 64, 8300, 70, 0, 3, True, 1),
    ('f16', 16, 8, 96, 80, 8240, 60, 0, 0, False, 1),
    ('bf16', 16, 8, 256, 192, 8240, 60, 0, 5, True, 1),
    ('f16', 16, 8, 200, 256, 8240, 60, 3, 0, False, 1),
    ('bf16', 7, 1, 128, 128, 14000, 100, 0, 9, True, 4),   # 2, 2, 2 and 1 heads
    ('f16', 7, 1, 64, 128, 14000, 100, 5, 0, False, 4),
    ('bf16', 10, 2, 64, 64, 12000, 90, 0, 0, True, 3),     # 2, 2 and 1 heads
    ('f16', 16, 1, 128, 64, 9000, 80, 0, 4, True, 8),
    ('bf16', 5, 1, 256, 256, 22000, 100, 1, 1, True, 3),
    ('f16', 7, 1, 256, 64, 14000, 100, 0, 0, False, 4),
    # sequences of 1024 and more on average: twice the parts
    ('bf16', 8, 4, 128, 128, 16400, 5, 0, 6, True, 2),
    ('f16', 8, 8, 64, 64, 16400, 5, 0, 0, True, 1),
    # more than 256 sequences: searched for, not ranked
    ('bf16', 16, 8, 64, 64, 9000, 300, 4, 11, False, 1),
    ('f16', 6, 2, 128, 128, 20000, 400, 0, 0, True, 2),
    # float32 at head dims 64, 128 and 256, one or more heads a block
    ('f32', 16, 8, 64, 64, 8300, 100, 2, 3, True, 1),
    ('f32', 16, 8, 64, 32, 8300, 100, 0, 0, False, 1),
    ('f32', 7, 1, 64, 64, 14000, 100, 0, 0, True, 4),
    ('f32', 16, 8, 128, 100, 8300, 60, 0, 1, True, 1),
    ('f32', 7, 1, 96, 128, 14000, 100, 0, 0, False, 4),
    ('f32', 16, 8, 256, 256, 8300, 60, 0, 0, True, 1),
    ('f32', 5, 1, 192, 256, 22000, 100, 3, 0, False, 3),
]


@pytest.mark.parametrize('case', GROUPS, ids=lambda c: '_'.join(map(str, c[:7] + c[9:])))
def test_heads_that_share_keys(case):
    """dK / dV blocks that stream one head (as many parts as heads), several,
    or unequal numbers of them."""
    dt, h, hk, d, dv, total, n, lead, pad, causal, parts = case
    print(f'[case] {case}', flush=True)
    assert _parts(h, hk, total + lead + pad, n) == parts
    heads = range(hk) if hk <= 2 else (0, hk // 2, hk - 1)
    _run(dt, h, hk, d, dv, _lens(total, n, h + n), lead, pad, causal, heads)


# dtype, h, hk, d, dv, lens, pad, causal, waves of a forward block at head dim 128
WAVES = [
    ('bf16', 16, 4, 128, 128, [4100], 0, True, 8),
    ('f16', 8, 4, 128, 128, [9000, 0, 130], 5, True, 8),
    ('f16', 32, 8, 96, 128, [2100], 0, False, 8),
    ('bf16', 32, 8, 128, 80, [2900, 1, 1500], 3, False, 8),
    ('bf16', 32, 8, 128, 128, [2100, 700], 0, True, 4),
    ('f16', 32, 8, 128, 72, [1300, 1200], 0, False, 4),
    ('bf16', 8, 2, 128, 128, [4100], 0, True, 4),          # few blocks
    ('f16', 8, 2, 128, 128, [2100], 0, False, 4),
]


@pytest.mark.parametrize('case', WAVES, ids=lambda c: '_'.join(map(str, c[:5] + c[7:])))
def test_four_and_eight_waves(case):
    dt, h, hk, d, dv, lens, pad, causal, waves = case
    print(f'[case] {case}', flush=True)
    t = sum(lens) + pad
    few = h * (t // 256 + 1) < 256 or t // len(lens) < (3000 if causal else 1400)
    assert (4 if few else 8) == waves
    _run(dt, h, hk, d, dv, lens, 0, pad, causal, (0, hk - 1))


# h, hk, lens, causal, blocks of 32 rows in the forward, dQ, dK / dV
SPLITS = [
    (8, 8, [400] * 10, True, (False, True, True)),
    (8, 8, [400] * 10, False, (False, True, False)),
    (8, 8, [200] * 20, False, (False, True, True)),
    (8, 2, [415] * 20, True, (False, False, False)),
    (8, 2, [8000, 0, 300], False, (False, True, False)),
    (16, 8, [83] * 100, True, (False, False, False)),
    (16, 8, [8000, 300], True, (False, False, False)),
    (6, 6, [250] * 20, False, (True, True, True)),
    (2, 2, [3000, 77], True, (True, True, True)),
]


@pytest.mark.parametrize('case', SPLITS, ids=lambda c: f'{c[0]}_{c[1]}_{len(c[2])}_{sum(c[2])}_{c[3]}')
def test_float32_blocks(case):
    """Head dim 64: blocks of 128 rows, or of 32 whose waves split the tiles."""
    h, hk, lens, causal, split = case
    print(f'[case] {case}', flush=True)
    t, n = sum(lens), len(lens)
    q128, k128 = h * t // 128, hk * _parts(h, hk, t, n) * t // 128
    assert split == (q128 < 240, q128 <= 512 or (q128 <= 1024 and t // n >= 2048),
                     k128 <= 128 or (k128 <= 256 and (causal or t // n < 320)))
    _run('f32', h, hk, 64, 64, lens, 0, 0, causal, (0, hk - 1))


# --- stores beside the outputs ------------------------------------------------


class _Guarded:
    """A tensor inside a larger buffer of sentinel bytes."""

    EDGE, BYTE = 1 << 16, 0xA5

    def __init__(self, shape, dtype):
        n = math.prod(shape) * torch.empty((), dtype=dtype).element_size()
        self.buf = torch.full((2 * self.EDGE + -(-n // 256) * 256,), self.BYTE, dtype=torch.uint8,
                              device=_dev())
        self.n = n
        self.x = self.buf[self.EDGE:self.EDGE + n].view(dtype).view(shape)

    def untouched_around(self):
        e = self.EDGE
        return bool((self.buf[:e] == self.BYTE).all() and (self.buf[e + self.n:] == self.BYTE).all())


@pytest.mark.parametrize('dtype, h, hk, d', [('bf16', 4, 2, 64), ('f16', 7, 1, 128),
                                             ('bf16', 2, 1, 256), ('f32', 4, 2, 64), ('f32', 2, 1, 128)])
@pytest.mark.parametrize('t, many', [(200, False), (14000, False), (4000, True)])
def test_offsets_out_of_order_store_nothing_beside_the_outputs(dtype, h, hk, d, t, many):
    """Offsets the documentation excludes leave rows undefined, but no store
    leaves the tensors: the bytes around every output and the workspace."""
    print(f'[case] {dtype} {h} {hk} {d} {t} {many}', flush=True)
    dt, lib = DT[dtype], _lib.lib()
    q, k, v = (x.contiguous() for x in _tokens(t, h, hk, d, d, dt, 16))
    do = torch.randn_like(q)
    if many:  # searched for
        lists = [np.random.default_rng(s).integers(-9, t + 9, 301).tolist() for s in range(3)]
    else:
        lists = [[-5, t // 2, 4 * t], [0, t * 3 // 4, t // 4, t], [t, 0],
                 [2 ** 31 - 1, -2 ** 31], [7, 7], [t // 2, t, 0, t // 2]]
    for ends in lists:
        off = _off(ends)
        o, o_lo, dq = (_Guarded((h, t, d), dt) for _ in range(3))
        dk, dv = (_Guarded((hk, t, d), dt) for _ in range(2))
        lse = _Guarded((h, t), torch.float32)
        # (rows of no sequence keep these)
        o.x.zero_(), o_lo.x.zero_(), lse.x.zero_()
        desc = packed._desc(q, k, v, o.x, off, 0.1, True)
        ws = _Guarded((lib.nxa_packed_workspace_bytes(ctypes.byref(desc)),), torch.uint8)
        lo = None if dt == torch.float32 else o_lo.x.data_ptr()
        st = [_lib.I64x2(*x.stride()[:2]) for x in (do, dq.x, dk.x, dv.x)]
        args = (ctypes.byref(desc), q.data_ptr(), k.data_ptr(), v.data_ptr(), off.data_ptr(),
                o.x.data_ptr(), lo, lse.x.data_ptr())
        stream = torch.cuda.current_stream().cuda_stream
        _lib.check(lib.nxa_packed_fwd(*args, stream))
        _lib.check(lib.nxa_packed_bwd(
            *args, do.data_ptr(), st[0], dq.x.data_ptr(), st[1], dk.x.data_ptr(), st[2],
            dv.x.data_ptr(), st[3], ws.x.data_ptr(), ws.x.numel(), stream))
        torch.cuda.synchronize()
        for name, x in dict(o=o, o_lo=o_lo, lse=lse, dq=dq, dk=dk, dv=dv, ws=ws).items():
            assert x.untouched_around(), (name, ends[:8])


def test_float16_probabilities_past_two_saturate():
    """Scores past 2^23, whose log-sum-exp in float32 leaves P of 2 and more
    where 1/2 is right: as an operand of dS such a P counts as 2 and does not
    wrap.  dV of one query shows the P that the kernel sees."""
    n, d, scale = 256, 64, 8.0
    g = torch.Generator().manual_seed(5)
    q = (256 * (1 + torch.arange(n) / 256.0))[:, None, None].expand(n, 2, d)
    k = torch.full((n, 2, d), 256.0)
    v0 = torch.randn(n, 1, d, generator=g)
    v = torch.cat((v0, -v0), 1)  # the output and delta are zero
    do = torch.zeros(n, 2, d)
    do[:, 1] = torch.randn(n, d, generator=g)
    q, k, v, do = (x.reshape(1, 2 * n, d).to(torch.float16).to(_dev()) for x in (q, k, v, do))
    got = _train(q, k, v, _off(range(0, 2 * n + 1, 2)), do, scale=scale)
    o, _, dk, dv = (x.double().reshape(n, 2, d) for x in got)
    q, v, do = (x.double().reshape(n, 2, d) for x in (q, v, do))
    assert (o == 0).all()
    top = do[:, 1:].abs().argmax(-1, keepdim=True)
    p = dv.gather(2, top.expand(n, 2, 1)) / do[:, 1:].gather(2, top)  # [n, 2, 1]
    assert int((p > 2.01).sum()) > 10 and int((p < 1.9).sum()) > 10
    ds = p.clamp(max=2) * (v * do[:, 1:]).sum(-1, keepdim=True)
    want = scale * ds * q[:, 1:]
    # roundings of 2^-11: P as dV's operand and dV, P's exchange, dS, dK; dP in
    # float32 of 64 terms; 2^-12 for the largest P below 2
    tol = 6 * 2.0 ** -11 * want.abs() + scale * q[:, 1:] * p * 2.0 ** -16
    near = (dk - want).abs() <= tol
    # a dK past fp16's largest number, 65504, is infinite, as it is to round
    # (|want| up to 8 * 512 * 2 * |v . do|, some 2e5); 2^-8: tol next to there
    edge = 65504 * (1 - 2.0 ** -8)
    past = (want.abs() >= edge) & (dk.abs() >= edge) & (dk.sign() == want.sign())
    assert (near | past).all() and int(near.sum()) > dk.numel() // 2
