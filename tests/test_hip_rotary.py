"""Rotary positions on the GPU against float64 (``_quant_plain.rotate``).

The tolerance: the angle's fraction of a turn, its sine and cosine and the two
products, each off by 2^-24 or little more of what the two terms are without their
signs (2^-20 of it bounds the sum of them), and one rounding to the type.
"""

from __future__ import annotations

from fractions import Fraction

import _quant_plain as qplain
import numpy as np
import pytest
import torch

import nitrix_amd as nx

pytestmark = pytest.mark.gpu

DT = {'bf16': torch.bfloat16, 'f16': torch.float16, 'f32': torch.float32}


def _dev():
    return torch.device('cuda:0')


def _rand(shape, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(*shape, generator=g).to(dtype).to(_dev())


def _n64(x):
    return x.detach().double().cpu().numpy()


def _check(got, x, pos, freq, interleaved, scale, inverse=False):
    """One (h, t, d) result against the plain form."""
    u = torch.finfo(x.dtype).eps / 2
    want, size = qplain.rotate(_n64(x), pos, freq.cpu().numpy(), interleaved, scale, inverse)
    tol = u * np.abs(want) + 2.0 ** -20 * size * (np.arange(x.shape[-1]) < 2 * len(freq))
    tiny = 2.0 ** -25 if x.dtype == torch.float16 else float(torch.finfo(x.dtype).tiny)
    assert got.shape == x.shape and got.dtype == x.dtype
    bad = ~(np.abs(_n64(got) - want) <= tol + tiny)
    assert not bad.any(), f'{bad.sum()} off at {np.argwhere(bad)[:5].tolist()}'
    r = 2 * len(freq)
    assert torch.equal(got[..., r:], x[..., r:])


CASES = [
    # dtype, h, hk, t, d, r, interleaved
    ('bf16', 32, 8, 70, 128, 128, False),
    ('bf16', 32, 8, 70, 128, 128, True),
    ('f16', 8, 2, 1, 64, 64, False),
    ('f16', 8, 2, 33, 64, 32, True),
    ('f32', 6, 6, 21, 64, 40, False),
    ('f32', 6, 1, 5, 256, 256, True),
    ('bf16', 3, 3, 130, 256, 256, False),
    ('bf16', 4, 1, 9, 96, 48, False),
    # turned and copied elements, or both halves, in one chunk; odd head dims
    ('bf16', 5, 1, 7, 80, 20, False),
    ('f16', 2, 2, 6, 64, 4, True),
    ('f32', 3, 1, 11, 7, 6, False),
    ('bf16', 1, 1, 3, 2, 2, True),
    ('f16', 2, 1, 5, 255, 254, False),
    # many tokens: a block takes four
    ('bf16', 3, 1, 1031, 128, 64, False),
    ('f16', 4, 4, 514, 64, 64, True),
    ('f32', 1, 1, 2001, 32, 20, False),
    ('bf16', 30, 10, 517, 128, 128, False),
    ('f32', 16, 16, 515, 96, 96, True),
    ('bf16', 40, 13, 513, 100, 100, False),
]


@pytest.mark.parametrize('case', CASES, ids=lambda c: '_'.join(map(str, c)))
def test_forward_and_backward(case):
    dt, h, hk, t, d, r, inter = case
    print(f'[case] {case}', flush=True)
    rng = np.random.default_rng(t)
    pos = rng.integers(-50, 200000, t)
    pos[0] = 0
    freq = nx.rotary_frequencies(r, device=_dev())
    # tokens before heads, as a projection leaves them, and heads before tokens
    q = _rand((t, h, d), DT[dt], 1).transpose(0, 1).requires_grad_(True)
    k = _rand((hk, t, d), DT[dt], 2).requires_grad_(True)
    p = torch.tensor(pos, dtype=torch.int32, device=_dev())
    out = nx.rotary_embed(q, k, p, freq, interleaved=inter, scale=1.25, backend='hip')
    for x, y in zip((q, k), out):
        _check(y, x, pos, freq, inter, 1.25)
    grads = _rand((h, t, d), DT[dt], 3), _rand((t, hk, d), DT[dt], 4).transpose(0, 1)
    back = torch.autograd.grad(out, (q, k), grads)
    for x, y in zip(grads, back):
        # (turned back; the elements behind r pass)
        _check(y, x, pos, freq, inter, 1.25, inverse=True)
    p64 = nx.rotary_embed(q, k, p.long(), freq, interleaved=inter, scale=1.25, backend='hip')
    assert all(torch.equal(a, b) for a, b in zip(out, p64))


def test_gradients_by_differences():
    """Against differences of the fused forward itself (float32, linear: a step
    of any size will do, so 2^-10 of rounding is left of a step of 8)."""
    q = _rand((2, 3, 8), torch.float32, 1).requires_grad_(True)
    pos, freq = torch.arange(3, device=_dev()) * 1000, nx.rotary_frequencies(6, device=_dev())
    w = _rand((2, 3, 8), torch.float32, 2)
    out, _ = nx.rotary_embed(q, None, pos, freq, backend='hip')
    (grad,) = torch.autograd.grad((out * w).sum(), q)
    with torch.no_grad():
        for i in range(q.numel()):
            e = torch.zeros_like(q).view(-1)
            e[i] = 8.0
            e = e.view_as(q)
            a, b = (nx.rotary_embed(q + s * e, None, pos, freq, backend='hip')[0] for s in (1, -1))
            want = float(((a - b) * w).double().sum()) / 16
            assert abs(want - float(grad.view(-1)[i])) < 2.0 ** -16


def test_backward_of_one_output_and_twice():
    q = _rand((2, 5, 16), torch.float32, 1).requires_grad_(True)
    k = _rand((1, 5, 16), torch.float32, 2).requires_grad_(True)
    pos, freq = torch.arange(5, device=_dev()), nx.rotary_frequencies(16, device=_dev())
    a, b = nx.rotary_embed(q, k, pos, freq, scale=2.0, backend='hip')
    (only,) = torch.autograd.grad(b.sum(), k, retain_graph=True)
    both = torch.autograd.grad((a.sum(), b.sum()), (q, k), create_graph=True)
    assert torch.equal(only, both[1])
    assert torch.autograd.grad(b.sum(), q, retain_graph=True, allow_unused=True)[0] is None
    # the gradient of the gradient turns forward again
    c = _rand((2, 5, 16), torch.float32, 3).requires_grad_(True)
    (g,) = torch.autograd.grad(a, q, c, create_graph=True)
    w = _rand((2, 5, 16), torch.float32, 4)
    (gg,) = torch.autograd.grad(g, c, w)
    want, _ = nx.rotary_embed(w, None, pos, freq, scale=2.0, backend='hip')
    assert torch.equal(gg, want)


def test_shared_and_broadcast_inputs():
    """A key head expanded over heads, and one row for every token."""
    base = _rand((1, 6, 64), torch.bfloat16, 1).requires_grad_(True)
    k = base.expand(4, 6, 64)
    row = _rand((2, 1, 64), torch.bfloat16, 2).expand(2, 6, 64)
    pos = torch.arange(6, device=_dev())
    freq = nx.rotary_frequencies(64, device=_dev())
    q2, k2 = nx.rotary_embed(row, k, pos, freq, backend='hip')
    _check(q2, row, pos.cpu().numpy(), freq, False, 1.0)
    _check(k2, k, pos.cpu().numpy(), freq, False, 1.0)
    w = _rand((4, 6, 64), torch.bfloat16, 3)
    (g,) = torch.autograd.grad(k2, base, w)
    each, _ = nx.rotary_embed(w, None, -pos, freq, backend='hip')
    torch.testing.assert_close(g, each.sum(0, keepdim=True), rtol=2.0 ** -7, atol=2.0 ** -6)


@pytest.mark.parametrize('lead', [(), (2,), (2, 3)])
def test_leading_axes_and_layouts(lead):
    h, t, d = 4, 9, 64
    freq = nx.rotary_frequencies(d, device=_dev())
    fused = _rand((*lead, t, 3 * h, d + 1), torch.bfloat16, 1)  # odd strides
    for x in (fused[..., :h, :d].transpose(-3, -2), fused[..., :h, 1:].transpose(-3, -2),
              _rand((*lead, h, d, t), torch.bfloat16, 2).transpose(-1, -2)):
        pos = torch.arange(t, device=_dev(), dtype=torch.int32) * 7
        for p in (pos, (pos + torch.arange(2, device=_dev(), dtype=torch.int32).view(
                2, *[1] * len(lead))).expand(*lead, t) if lead else pos):
            got, none = nx.rotary_embed(x, None, p, freq, backend='hip')
            assert none is None and got.shape == x.shape
            rows, ps = got.reshape(-1, h, t, d), p.expand(*lead, t).reshape(-1, t)
            for i, y in enumerate(x.reshape(-1, h, t, d)):
                _check(rows[i], y, ps[i].cpu().numpy(), freq, False, 1.0)


def test_far_positions():
    """The fraction of a turn is kept at positions past 2^31."""
    pos = torch.tensor([2 ** 20 + 1, 2 ** 31 - 1, 2 ** 40 + 12345, -2 ** 33 - 7], device=_dev())
    x = _rand((2, 4, 64), torch.float32, 1)
    freq = nx.rotary_frequencies(64, device=_dev())
    got, _ = nx.rotary_embed(x, None, pos, freq, backend='hip')
    # (p w in float64 is off by 2^-53 of itself: 2^-13 rad at 2^40, here and there)
    want, size = qplain.rotate(_n64(x), pos.cpu().numpy(), freq.cpu().numpy(), False, 1.0)
    off = 2.0 ** -20 + 2.0 ** -51 * np.abs(pos.cpu().numpy().astype(np.float64))
    assert (np.abs(_n64(got) - want) <= off[None, :, None] * size).all()


def test_float32_frequencies_and_nan_elsewhere():
    x = _rand((2, 4, 64), torch.bfloat16, 1)
    pos = torch.arange(4, device=_dev())
    f32 = nx.rotary_frequencies(64, device=_dev()).float()
    a, _ = nx.rotary_embed(x, None, pos, f32, backend='hip')
    b, _ = nx.rotary_embed(x, None, pos, f32.double(), backend='hip')
    assert torch.equal(a, b)
    x[1, 2, 5] = float('nan')
    c, _ = nx.rotary_embed(x, None, pos, f32, backend='hip')
    bad = torch.isnan(c)
    assert bad[1, 2, 5] and bad[1, 2, 37] and int(bad.sum()) == 2


def test_streams_and_graph_replay():
    q, k = _rand((4, 40, 128), torch.bfloat16, 1), _rand((2, 40, 128), torch.bfloat16, 2)
    q.requires_grad_(True), k.requires_grad_(True)
    dq, dk = torch.ones_like(q), torch.ones_like(k)
    off = torch.tensor([0, 13, 40], dtype=torch.int32, device=_dev())
    start = torch.tensor([5, 100], dtype=torch.int32, device=_dev())
    freq = nx.rotary_frequencies(128, device=_dev())

    def step():
        pos = nx.packed_positions(off, 40, start)
        out = nx.rotary_embed(q, k, pos, freq, backend='hip')
        return (*out, *torch.autograd.grad(out, (q, k), (dq, dk)))

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        held = step()
    for i in range(3):
        with torch.no_grad():
            q.copy_(_rand((4, 40, 128), torch.bfloat16, 10 + i))
            dk.copy_(_rand((2, 40, 128), torch.bfloat16, 20 + i))
            off[1] = 7 + i
            start.add_(1000)
        graph.replay()
        torch.cuda.synchronize()
        got = [x.detach().clone() for x in held]
        assert all(torch.equal(a, b) for a, b in zip(got, step()))
        torch.cuda.synchronize()


def test_with_packed_attention():
    """Queries and keys turned on the way into a training step of packed
    attention, against float64 end to end."""
    h, hk, d = 4, 2, 64
    off = torch.tensor([0, 30, 31, 77], dtype=torch.int32, device=_dev())
    t = 80
    x = [_rand((n, t, d), torch.float32, s).requires_grad_(True)
         for s, n in ((1, h), (2, hk), (3, hk))]
    w = _rand((h, t, d), torch.float32, 4)
    grads = []
    for dev, dt, backend in ((_dev(), torch.float32, 'hip'), ('cpu', torch.float64, 'jax')):
        q, k, v = (y.detach().to(dev, dt).requires_grad_(True) for y in x)
        o = off.to(dev)
        freq = nx.rotary_frequencies(d, device=dev)
        a, b = nx.rotary_embed(q, k, nx.packed_positions(o, t), freq, backend=backend)
        out = nx.packed_attention(a, b, v, o, causal=True, backend=backend)
        grads.append((out, *torch.autograd.grad(out, (q, k, v), w.to(dev, dt))))
    for a, b in zip(*grads):
        # (float32 sums of up to 64 and 46 terms of size 1, and of gradients over
        # two heads: 2^-24 a term and factor, a thousand of them)
        assert float((a.cpu().double() - b).abs().max()) < 2.0 ** -14


def test_declined_calls_fall_back_loudly():
    pos = torch.arange(3, device=_dev())
    wide = _rand((1, 3, 264), torch.bfloat16, 1)
    freq = nx.rotary_frequencies(264, device=_dev())
    nx.reset_fallback_state()
    with pytest.warns(nx.NitrixBackendFallback):
        nx.rotary_embed(wide, None, pos, freq)
    x64 = wide[..., :64].double().requires_grad_(True)
    with pytest.warns(nx.NitrixBackendFallback):
        y, _ = nx.rotary_embed(x64, None, pos, freq[:32])
    assert y.requires_grad and y.dtype == torch.float64
    empty = nx.rotary_embed(wide[:, :0], None, pos[:0], freq)[0]
    assert empty.shape == (1, 0, 264)


def test_only_what_is_trained_has_a_gradient():
    """As in the other engine: the output of an input without a gradient has none,
    and may go into a cache."""
    h, t, d = 2, 5, 16
    freq, pos = nx.rotary_frequencies(d, device=_dev()), torch.arange(t, device=_dev())
    for which in range(2):
        x = [_rand((h, t, d), torch.float32, s) for s in (1, 2)]
        x[which].requires_grad_(True)
        for backend in ('hip', 'jax'):
            out = nx.rotary_embed(*x, pos, freq, backend=backend)
            assert [y.requires_grad for y in out] == [which == 0, which == 1]
            out[which].sum().backward()
    pages = [torch.zeros(1, h, 16, d, device=_dev()) for _ in range(2)]
    i32 = dict(dtype=torch.int32, device=_dev())
    q, k = (_rand((h, t, d), torch.float32, s) for s in (1, 2))
    _, turned = nx.rotary_embed(q.requires_grad_(True), k, pos, freq, backend='hip')
    nx.write_pages(*pages, turned, k, torch.zeros(1, 1, **i32), torch.zeros(1, **i32),
                   torch.tensor([0, t], **i32), backend='hip')
    assert torch.equal(pages[0][0, :, :t], turned)


@pytest.mark.parametrize('inter', [False, True])
def test_far_positions_to_the_last_digit(inter):
    """Against turns in whole fractions.  In float32 a half turn is off by 2^-25 of
    itself (2^-23.3 rad), sine and cosine by 2^-23, the products and their sum by 2^-24
    each: 2^-21 of the terms' size covers them, wherever a token stands."""
    pi = Fraction('3.14159265358979323846264338327950288419716939937510582097494459')
    pos = [10 ** 9, 2 ** 31 - 1, 2 ** 40 + 12345, -2 ** 45 - 7, 2 ** 52 + 1]
    freq = nx.rotary_frequencies(64, device=_dev())
    x = _rand((2, len(pos), 64), torch.float32, 1)
    got, _ = nx.rotary_embed(x, None, torch.tensor(pos, device=_dev()), freq, interleaved=inter,
                             backend='hip')
    turns = [[float(p * Fraction(w) / (2 * pi) % 1) for w in freq.tolist()] for p in pos]
    # (as angles of position 1, a token at a time)
    for i, t in enumerate(turns):
        want, size = qplain.rotate(_n64(x)[:, i:i + 1], [1], 2 * np.pi * np.array(t), inter, 1.0)
        assert (np.abs(_n64(got)[:, i:i + 1] - want) <= 2.0 ** -21 * size).all(), pos[i]
