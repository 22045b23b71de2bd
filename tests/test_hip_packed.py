"""Packed attention on the GPU against a plain float64 implementation.

Every tolerance is a bound computed element by element beside the expected
value, from the roundings the kernels make: u = eps(T) / 2 for each rounding
to the I/O type (the probabilities and dS as matrix operands, the outputs;
zero times anything for float32, whose operands are not rounded), 2^-11 for
the fp16 copy of P inside dK / dV (bf16; fp16 has a finer one), 2^-16 for delta as a pair of bf16 terms,
2^-24 a step for float32 sums.  fp16 numbers below 2^-14 are 2^-24 apart, so
there half a step is 2^-25 however small the value: an absolute term for the
fp16 copy of P (both 16-bit types) and for P and dS as fp16 operands.
``_bounds`` spells them out.
"""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

import nitrix_amd as nx
from nitrix_amd.packed import packed_attention, packed_attention_hip

pytestmark = pytest.mark.gpu

E24 = 2.0 ** -24


def _dev():
    return torch.device('cuda:0')


def _bounds(q, k, v, do, scale, causal, u, dt):
    """One sequence of one key-value head: q, do [g, n, d], k, v [n, d], all
    float64.  Expected (o, dq, dk, dv) and the bound of each."""
    n, d = k.shape
    dv_ = v.shape[1]
    f32 = dt == torch.float32
    sub = 2.0 ** -25 if dt == torch.float16 else 0.0  # half a step of a small fp16 operand
    subx = 0.0 if f32 else 2.0 ** -25                  # of the fp16 copy of P
    s = scale * np.einsum('gid,jd->gij', q, k)
    # a float32 dot of d products, scaled and shifted in base 2
    es = (d + 8) * E24 * scale * np.einsum('gid,jd->gij', np.abs(q), np.abs(k)) + 4 * E24 * np.abs(s)
    if causal:
        keep = np.tri(n, dtype=bool)
        s = np.where(keep, s, -np.inf)
        es = np.where(keep, es, 0.0)
    m = s.max(-1, keepdims=True)
    p = np.exp(s - m)
    p /= p.sum(-1, keepdims=True)
    # relative error of a probability: its own logit, the normaliser's, the
    # maximum's and lse's rounding, the sum, the hardware exponential (2 ulp)
    rp = es + es.max(-1, keepdims=True) + (n + 16) * E24 + 8 * E24 * np.abs(m) + 16 * E24
    o = np.einsum('gij,jd->gid', p, v)
    av = np.abs(v)
    # (P is kept relative to a row's maximum, its sum is at least 1)
    to = np.einsum('gij,jd->gid', p * (rp + u + n * E24) + sub, av) + u * np.abs(o) + 4 * E24 * np.abs(o)
    if do is None:
        return (o,), (to,)
    ado = np.abs(do)
    dp = np.einsum('gid,jd->gij', do, v)
    delta = (o * do).sum(-1, keepdims=True)
    ds = p * (dp - delta)
    edp = (dv_ + 8) * E24 * np.einsum('gid,jd->gij', ado, av)
    # (delta is taken from o with its rounding kept apart: u^2 of it is left)
    tod = to - u * (1 - 2 * u) * np.abs(o)
    edl = ((tod * ado).sum(-1, keepdims=True) + (dv_ + 8) * E24 * (np.abs(o) * ado).sum(-1, keepdims=True)
           + (0 if f32 else 2.0 ** -16) * np.abs(delta))
    tds = np.abs(ds) * (rp + (0 if f32 else 2.0 ** -11) + u) + p * (edp + edl) * (1 + rp)
    tds = tds + sub + subx * (np.abs(dp - delta) + edp + edl)
    rows = q.shape[0] * n
    dq = scale * np.einsum('gij,jd->gid', ds, k)
    tq = scale * np.einsum('gij,jd->gid', tds + n * E24 * np.abs(ds), np.abs(k)) + (u + 4 * E24) * np.abs(dq)
    dk = scale * np.einsum('gij,gid->jd', ds, q)
    tk = scale * np.einsum('gij,gid->jd', tds + rows * E24 * np.abs(ds), np.abs(q)) + (u + 4 * E24) * np.abs(dk)
    dv = np.einsum('gij,gid->jd', p, do)
    tv = np.einsum('gij,gid->jd', p * (rp + u + rows * E24) + sub, ado) + (u + 4 * E24) * np.abs(dv)
    return (o, dq, dk, dv), (to, tq, tk, tv)


def _check(q, k, v, ends, got, scale, causal, do=None):
    """``got``: o, or (o, dq, dk, dv), torch tensors."""
    dt = q.dtype
    f32 = dt == torch.float32
    u = 0.0 if f32 else torch.finfo(dt).eps / 2
    tiny = 4 * float(torch.finfo(dt).tiny if dt != torch.float16 else 2.0 ** -24)
    n64 = lambda x: x.detach().double().cpu().numpy()  # noqa: E731
    names = ('o', 'dq', 'dk', 'dv')
    got = [n64(x) for x in got]
    q, k, v = n64(q), n64(k), n64(v)
    do = None if do is None else n64(do)
    g = q.shape[0] // k.shape[0]
    for name, x in zip(names, got):
        out = np.ones(x.shape[1], bool)
        out[max(0, min(ends[0], x.shape[1])):max(ends)] = False
        assert (x[:, out] == 0).all(), f'{name}: rows of no sequence'
    for a, b in zip(ends[:-1], ends[1:]):
        if b <= a:
            continue
        for hk in range(k.shape[0]):
            hs = slice(hk * g, (hk + 1) * g)
            want, tol = _bounds(q[hs, a:b], k[hk, a:b], v[hk, a:b],
                                None if do is None else do[hs, a:b], scale, causal, u, dt)
            parts = [got[0][hs, a:b]]
            if do is not None:
                parts += [got[1][hs, a:b], got[2][hk, a:b], got[3][hk, a:b]]
            for name, x, w, t in zip(names, parts, want, tol):
                bad = ~(np.abs(x - w) <= t + tiny)
                assert not bad.any(), (
                    f'{name} rows {a}..{b} head {hk}: {bad.sum()} off, worst '
                    f'{np.nanmax(np.abs(x - w) / (t + tiny)):.2f} bounds, nan {np.isnan(x).sum()}')


def _ends(lens, lead=0):
    return [lead] + [int(x) for x in lead + np.cumsum(lens)]


def _tokens(t, h, hk, d, dv, dtype, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)

    def rnd(*s):
        return (torch.randn(*s, generator=g) * scale).to(dtype).to(_dev()).transpose(0, 1)

    return rnd(t, h, d), rnd(t, hk, d), rnd(t, hk, dv)


def _off(ends):
    return torch.tensor(ends, dtype=torch.int32, device=_dev())


def _train(q, k, v, off, do, **kw):
    ts = [x.detach().requires_grad_(True) for x in (q, k, v)]
    out = packed_attention(*ts, off, backend='hip', **kw)
    return (out, *torch.autograd.grad(out, ts, do))


EDGES = [0, 1, 2, 31, 32, 33, 0, 63, 64, 65, 127, 128, 129, 255, 256, 257, 300, 0]

CASES = [
    # dtype, h, hk, d, dv, lens, lead, pad, causal
    ('bf16', 4, 2, 64, 64, EDGES, 0, 0, True),
    ('bf16', 4, 2, 64, 64, EDGES, 0, 0, False),
    ('bf16', 8, 2, 128, 128, EDGES, 3, 5, True),
    ('f16', 3, 1, 128, 128, EDGES, 0, 70, False),
    ('f16', 2, 2, 256, 256, [257, 1, 130], 1, 1, True),
    ('bf16', 7, 1, 256, 64, [100, 0, 200], 0, 0, False),
    ('bf16', 6, 2, 80, 40, [5, 300, 77], 0, 0, True),
    ('bf16', 16, 1, 32, 96, [1, 1, 1, 190], 0, 2, True),
    ('bf16', 1, 1, 8, 8, [1], 0, 0, True),
    ('f32', 4, 2, 64, 64, EDGES, 2, 9, True),
    ('f32', 3, 3, 32, 64, EDGES, 0, 0, False),
    ('f32', 4, 1, 128, 100, [129, 300, 0, 1], 0, 0, True),
    ('f32', 2, 1, 256, 256, [130, 33], 0, 1, True),
    ('f32', 2, 1, 192, 4, [64, 65], 0, 0, False),
]
DT = {'bf16': torch.bfloat16, 'f16': torch.float16, 'f32': torch.float32}


@pytest.mark.parametrize('case', CASES, ids=lambda c: '_'.join(map(str, c[:5] + c[8:])))
def test_forward_and_backward(case):
    dt, h, hk, d, dv, lens, lead, pad, causal = case
    ends = _ends(lens, lead)
    t = ends[-1] + pad
    print(f'[case] {case}', flush=True)
    q, k, v = _tokens(t, h, hk, d, dv, DT[dt], 1)
    do = _tokens(t, h, h, dv, dv, DT[dt], 2)[0]
    scale = 1 / math.sqrt(d)
    got = _train(q, k, v, _off(ends), do, causal=causal)
    torch.cuda.synchronize()
    _check(q, k, v, ends, got, scale, causal, do)
    with torch.no_grad():
        o = packed_attention(q, k, v, _off(ends), causal=causal, backend='hip')
    assert torch.equal(o, got[0])
    assert got[0].stride() == (dv, h * dv, 1) or h == 1


@pytest.mark.parametrize('dtype', ['bf16', 'f32'])
@pytest.mark.parametrize('scale', [0.0, -0.3, 2.0])
def test_scales(dtype, scale):
    ends = _ends([70, 1, 200])
    q, k, v = _tokens(ends[-1], 4, 2, 64, 64, DT[dtype], 3)
    do = _tokens(ends[-1], 4, 4, 64, 64, DT[dtype], 4)[0]
    got = _train(q, k, v, _off(ends), do, causal=True, scale=scale)
    if scale >= 0:
        _check(q, k, v, ends, got, scale, True, do)
    else:  # the bound's sums take |scale|: swap the sign into q
        _check(-q, k, v, ends, (got[0], -got[1], got[2], got[3]), -scale, True, do)


@pytest.mark.parametrize('dtype', ['bf16', 'f32'])
def test_rows_of_no_sequence_may_hold_anything(dtype):
    ends = _ends([40, 90], 17)
    t = ends[-1] + 33
    q, k, v = _tokens(t, 4, 2, 64, 64, DT[dtype], 5)
    do = _tokens(t, 4, 4, 64, 64, DT[dtype], 6)[0]
    for i, x in enumerate((q, k, v, do)):
        x[:, :17] = (math.nan, math.inf)[i % 2]
        x[:, ends[-1]:] = (math.inf, math.nan)[i % 2]
    got = _train(q, k, v, _off(ends), do, causal=False)
    assert all(torch.isfinite(x).all() for x in got)
    _check(q, k, v, ends, got, 0.125, False, do)


def test_a_nan_stays_in_its_sequence():
    ends = _ends([64, 64, 64])
    q, k, v = _tokens(192, 2, 1, 64, 64, torch.bfloat16, 7)
    v[:, 70] = math.nan
    o = packed_attention(q, k, v, _off(ends), causal=True, backend='hip')
    # (the sequence's earlier rows weigh it with zero, and 0 * NaN is NaN, as
    # in the reference engine's product)
    assert torch.isfinite(o[:, :64]).all() and torch.isfinite(o[:, 128:]).all()
    assert torch.isnan(o[:, 70:128]).all()


def test_large_logits():
    ends = _ends([130, 3])
    q, k, v = _tokens(133, 2, 1, 64, 64, torch.bfloat16, 8, scale=12.0)
    o = packed_attention(q, k, v, _off(ends), causal=True, backend='hip')
    _check(q, k, v, ends, (o,), 0.125, True)


@pytest.mark.parametrize('layout', ['heads', 'fused', 'odd', 'shared_heads'])
@pytest.mark.parametrize('dtype', ['bf16', 'f32'])
def test_layouts(layout, dtype):
    ends = _ends([65, 20, 130])
    t, h, hk, d = ends[-1], 4, 4, 64
    q, k, v = _tokens(t, h, hk, d, d, DT[dtype], 9)
    do = _tokens(t, h, h, d, d, DT[dtype], 10)[0]
    if layout == 'heads':
        q, k, v, do = (x.contiguous() for x in (q, k, v, do))
    elif layout == 'fused':
        x = torch.stack([y.transpose(0, 1) for y in (q, k, v)], 1).contiguous()
        q, k, v = (x[:, i].transpose(0, 1) for i in range(3))
    elif layout == 'odd':
        q = torch.nn.functional.pad(q, (0, 1))[..., :d]
        do = torch.nn.functional.pad(do, (1, 0))[..., 1:]
    else:  # one key-value head broadcast by a zero stride
        k, v = k[:1].expand(hk, t, d), v[:1].expand(hk, t, d)
    got = _train(q, k, v, _off(ends), do, causal=True)
    _check(q, k, v, ends, got, 0.125, True, do)


def test_sum_cotangent():
    """A cotangent of zero strides."""
    ends = _ends([50, 60])
    q, k, v = _tokens(110, 2, 1, 32, 32, torch.bfloat16, 11)
    ts = [x.detach().requires_grad_(True) for x in (q, k, v)]
    out = packed_attention(*ts, _off(ends), backend='hip')
    grads = torch.autograd.grad(out.sum(), ts)
    _check(q, k, v, ends, (out, *grads), 1 / math.sqrt(32), False, torch.ones_like(out))


def test_one_gradient_only():
    ends = _ends([50, 60])
    q, k, v = _tokens(110, 2, 1, 32, 32, torch.bfloat16, 12)
    do = torch.randn_like(q)
    full = _train(q, k, v, _off(ends), do)
    kk = k.detach().requires_grad_(True)
    out = packed_attention(q, kk, v, _off(ends), backend='hip')
    out.backward(do)
    assert torch.equal(kk.grad, full[2])


def test_gradients_by_differences():
    ends = _ends([37, 3, 70])
    ts = [x.detach().requires_grad_(True) for x in _tokens(110, 4, 2, 32, 16, torch.float32, 13)]
    w = torch.randn(4, 110, 16, device=_dev())

    def loss(*a):
        return (packed_attention(*a, _off(ends), causal=True, backend='hip').double() * w).sum()

    grads = torch.autograd.grad(loss(*ts), ts)
    for i in range(3):
        r = torch.randn_like(ts[i])
        r /= r.norm()
        step = 2.0 ** -6
        lo, hi = ([x.detach() + (j * step * r if n == i else 0) for n, x in enumerate(ts)]
                  for j in (-1, 1))
        num = ((loss(*hi) - loss(*lo)) / (2 * step)).item()
        ana = (grads[i].double() * r).sum().item()
        # The difference quotient: two float32 losses of 7040 terms, each off
        # by at most 2^-20 of its value (2^-20 * 7040 * |w||o| ~ 7e-3 summed
        # without cancellation, / 2 step -> 0.2 worst case, a hundredth of it
        # for independent signs), and step^2 / 6 of a third derivative of
        # order |w| ~ 40.
        assert abs(num - ana) <= 2e-3 + 40 * step ** 2 / 6


@pytest.mark.parametrize('dtype', ['bf16', 'f16', 'f32'])
def test_single_tokens_have_no_score_gradients(dtype):
    """A softmax over one key does not depend on q and k: dP = delta, and what
    their roundings leave of dQ and dK is far below a rounding of o."""
    n, d = 300, 128
    q, k, v = _tokens(n, 2, 2, d, d, DT[dtype], 17)
    do = _tokens(n, 2, 2, d, d, DT[dtype], 18)[0]
    got = _train(q, k, v, _off(range(n + 1)), do, causal=True)
    _check(q, k, v, list(range(n + 1)), got, 1 / math.sqrt(d), True, do)
    for g in got[1:3]:
        # delta as two bf16 terms: 2^-16 of |o||do| ~ 11, times |k| / sqrt(d)
        assert g.abs().max() < 2.0 ** -16 * 60 * 4.5 / math.sqrt(d) * 2


def test_many_tiny_sequences():
    rng = np.random.default_rng(0)
    lens = rng.integers(0, 4, 3000)
    ends = _ends(lens)
    q, k, v = _tokens(ends[-1], 2, 1, 16, 16, torch.bfloat16, 14)
    do = _tokens(ends[-1], 2, 2, 16, 16, torch.bfloat16, 15)[0]
    got = _train(q, k, v, _off(ends), do, causal=True)
    _check(q, k, v, ends, got, 0.25, True, do)


def test_offsets_out_of_order_or_range_stay_in_bounds():
    """Values the documentation excludes: whatever they give, it is finite
    and the tensors next to the operands are untouched."""
    q, k, v = _tokens(200, 2, 1, 64, 64, torch.bfloat16, 16)
    do = torch.randn_like(q)
    for ends in ([-5, 100, 900], [0, 150, 50, 200], [200, 0], [2 ** 31 - 1, -2 ** 31], [7, 7]):
        got = _train(q, k, v, _off(ends), do, causal=True)
        torch.cuda.synchronize()
        assert all(x.shape[1] == 200 for x in got)
    ends = [-5, 100, 900]  # clamped to 0, 100, 200
    got = _train(q, k, v, _off(ends), do, causal=True)
    _check(q, k, v, [0, 100, 200], got, 0.125, True, do)


def test_many_offsets_out_of_order_stay_in_bounds():
    """As above for more sequences than are ranked, whose tiles are searched
    for: offsets that jump send the search to a sequence behind its slot."""
    t = 4000
    q, k, v = _tokens(t, 2, 1, 64, 64, torch.bfloat16, 60)
    do = torch.randn_like(q)
    for seed in range(3):
        ends = np.random.default_rng(seed).integers(0, t, 301).tolist()
        got = _train(q, k, v, _off(ends), do, causal=True)
        torch.cuda.synchronize()
        assert all(x.shape[1] == t for x in got)
    ends = sorted(ends)  # as many in order
    _check(q, k, v, ends, _train(q, k, v, _off(ends), do, causal=True), 0.125, True, do)


def test_repeated_calls_agree_and_streams_do_not_mix():
    ends = _ends([300, 200, 11])
    sets = [(_tokens(511, 4, 2, 64, 64, torch.bfloat16, 20 + i)) for i in range(2)]
    do = [torch.randn_like(s[0]) for s in sets]
    want = [_train(*s, _off(ends), d, causal=True) for s, d in zip(sets, do)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = []
    off = _off(ends)
    torch.cuda.synchronize()
    for st, s, d in zip(streams, sets, do):
        with torch.cuda.stream(st):
            got.append(_train(*s, off, d, causal=True))
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        for x, y in zip(a, b):
            assert torch.equal(x, y)


def test_graph_replay_with_other_offsets():
    ends = _ends([100, 28, 172])
    q, k, v = _tokens(300, 4, 2, 64, 64, torch.bfloat16, 30)
    off = _off(ends)
    st = torch.cuda.Stream()
    with torch.no_grad():
        with torch.cuda.stream(st):
            packed_attention(q, k, v, off, causal=True, backend='hip')
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            out = packed_attention(q, k, v, off, causal=True, backend='hip')
        for e in (ends, [0, 1, 1, 300], [10, 150, 160, 290], ends):
            off.copy_(_off(e))
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, packed_attention(q, k, v, _off(e), causal=True, backend='hip'))


@pytest.mark.parametrize('dtype, h, hk, t', [('bf16', 8, 1, 700), ('f16', 4, 2, 300),
                                             ('f32', 2, 1, 300)])
def test_captured_training_step(dtype, h, hk, t):
    """Forward and backward captured together, replayed with other inputs and
    offsets and eager calls in between: the bytes of an eager step."""
    dt = {'bf16': torch.bfloat16, 'f16': torch.float16, 'f32': torch.float32}[dtype]
    q, k, v = _tokens(t, h, hk, 64, 64, dt, 70)
    do = torch.randn_like(q)
    off = _off([0, t // 3, t])
    ins = [x.requires_grad_(True) for x in (q, k, v)]

    def step():
        out = packed_attention(*ins, off, causal=True, backend='hip')
        return (out, *torch.autograd.grad(out, ins, do))

    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        out = step()
    for i, ends in enumerate(([0, t // 3, t], [0, 1, t], [5, t - 80, t - 7])):
        off.copy_(_off(ends))
        with torch.no_grad():
            for x, y in zip(ins, _tokens(t, h, hk, 64, 64, dt, 80 + i)):
                x.copy_(y)
        graph.replay()
        torch.cuda.synchronize()
        got = [x.detach().clone() for x in out]
        want = _train(q, k, v, _off(ends), do, causal=True)
        for x, y in zip(got, want):
            assert torch.equal(x, y)


def test_rows_past_2_31_elements():
    """A row stride that puts late tokens beyond 2^31 elements (and 2^32
    bytes) of the operands' base."""
    t, stride = 33100, 65600
    buf = torch.empty(t * stride, dtype=torch.bfloat16, device=_dev()).view(t, stride)
    x = torch.randn(t, 3 * 64, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
    buf[:, :192] = x.to(_dev())
    q, k, v = (buf[:, 64 * i:64 * i + 64].unsqueeze(0) for i in range(3))
    assert q.data_ptr() == buf.data_ptr()
    ends = [0, 100, t - 200, t]
    do = torch.randn(1, t, 64, device=_dev(), dtype=torch.bfloat16)
    got = _train(q, k, v, _off(ends), do, causal=True)
    tail = slice(t - 200, t)
    _check(q[:, tail], k[:, tail], v[:, tail], [0, 200], [g[:, tail] for g in got], 0.125, True,
           do[:, tail])


def test_declined_calls_fall_back_loudly():
    q, k, v = _tokens(20, 2, 1, 12, 12, torch.bfloat16, 40)
    nx.reset_fallback_state()
    with pytest.warns(nx.NitrixBackendFallback):
        packed_attention(q, k, v, _off([0, 20]))
    with pytest.raises(nx.HipNotTileable):
        packed_attention_hip(q, k, v, _off([0, 20]), scale=1.0)


def test_in_place_change_between_the_passes_raises():
    q, k, v = (x.detach().requires_grad_(True) for x in _tokens(20, 2, 1, 16, 16, torch.bfloat16, 41))
    off = _off([0, 20])
    out = packed_attention(q, k, v, off, backend='hip')
    off += 1
    with pytest.raises(RuntimeError, match='modified by an inplace'):
        out.sum().backward()


def _off_by_one(x):
    """The same numbers, contiguous, one element past a 16-byte boundary."""
    flat = torch.empty(x.numel() + 1, dtype=x.dtype, device=x.device)
    y = flat[1:].view(x.shape)
    y.copy_(x)
    assert y.is_contiguous() and y.data_ptr() % 16
    return y


@pytest.mark.parametrize('dtype', ['bf16', 'f32'])
@pytest.mark.parametrize('t, h, hk', [(85, 4, 2), (1, 2, 1), (40, 1, 1)])
def test_contiguous_operands_off_a_boundary(dtype, t, h, hk):
    """Slices of flat buffers, the cotangent's among them."""
    ends = _ends([t - t // 3, t // 3])
    q, k, v = _tokens(t, h, hk, 64, 64, DT[dtype], 90)
    do = _tokens(t, h, h, 64, 64, DT[dtype], 91)[0]
    want = _train(q, k, v, _off(ends), do, causal=True)
    ins = [_off_by_one(x) for x in (q, k, v)]
    got = _train(*ins, _off(ends), _off_by_one(do), causal=True)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    with torch.no_grad():
        assert torch.equal(packed_attention(*ins, _off(ends), causal=True, backend='hip'), want[0])


def test_forward_mode_falls_back_loudly():
    from torch.autograd import forward_ad

    q, k, v = _tokens(60, 4, 2, 32, 32, torch.float32, 92)
    off = _off([0, 25, 60])
    with forward_ad.dual_level():
        ins = [forward_ad.make_dual(x, torch.randn_like(x)) for x in (q, k, v)]
        nx.reset_fallback_state()
        with pytest.warns(nx.NitrixBackendFallback, match='forward-mode'):
            got = forward_ad.unpack_dual(packed_attention(*ins, off, causal=True))
        want = forward_ad.unpack_dual(packed_attention(*ins, off, causal=True, backend='jax'))
        for a, b in zip(got, want):
            assert a is not None and torch.equal(a, b)
    # a cotangent with a tangent: the backward has no derivative
    ts = [x.detach().requires_grad_(True) for x in (q, k, v)]
    out = packed_attention(*ts, off, backend='hip')
    with forward_ad.dual_level(), pytest.raises(RuntimeError, match='not itself differentiable'):
        torch.autograd.grad(out, ts, forward_ad.make_dual(torch.ones_like(out), torch.ones_like(out)))


def test_more_sequences_than_a_grid_holds_fall_back():
    """64 heads of 2^18 sequences: 2^32 threads forward; of 2^17: backward."""
    q, k, v = _tokens(40, 64, 64, 8, 8, torch.float32, 93)
    off = torch.full(((1 << 18) + 1,), 40, dtype=torch.int32, device=_dev())
    off[0], off[1] = 0, 25
    nx.reset_fallback_state()
    with pytest.warns(nx.NitrixBackendFallback, match='grid'):
        out = packed_attention(q, k, v, off, causal=True)
    _check(q, k, v, [0, 25, 40], (out,), 1 / math.sqrt(8), True)
    fewer = off[:(1 << 17) + 1]
    b = [x.to(torch.bfloat16) for x in (q, k, v)]
    _check(*b, [0, 25, 40], (packed_attention(*b, fewer, causal=True, backend='hip'),),
           1 / math.sqrt(8), True)
    nx.reset_fallback_state()
    with pytest.warns(nx.NitrixBackendFallback, match='grid'):
        packed_attention(b[0].requires_grad_(True), b[1], b[2], fewer, causal=True)
