"""Host side of the rotary positions: the reference engine, frequencies,
refusals, and the C ABI's checks (CPU only)."""

from __future__ import annotations

import ctypes
import math

import _quant_plain as qplain
import numpy as np
import pytest
import torch

import nitrix_amd as nx
from nitrix_amd import _lib


def _rand(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed), dtype=torch.float64)


@pytest.mark.parametrize('interleaved', [False, True])
@pytest.mark.parametrize('d, r', [(8, 8), (10, 6), (7, 2)])
def test_reference(d, r, interleaved):
    freq = nx.rotary_frequencies(r, base=100.0)
    pos = [0, 5, -3, 10 ** 9, 17]
    q, k = _rand(3, 5, d), _rand(2, 5, d, seed=1)
    got = nx.rotary_embed(q, k, torch.tensor(pos), freq, interleaved=interleaved, scale=1.5)
    for x, y in zip((q, k), got):
        want, _ = qplain.rotate(x.numpy(), pos, freq.numpy(), interleaved, 1.5)
        np.testing.assert_allclose(y.numpy(), want, atol=1e-12)


def test_reference_gradients_and_broadcast_positions():
    freq = nx.rotary_frequencies(4)
    q, k = _rand(2, 3, 4, 6).requires_grad_(True), _rand(2, 1, 4, 6).requires_grad_(True)
    pos = torch.tensor([[0, 1, 2, 3]], dtype=torch.int32)
    assert torch.autograd.gradcheck(lambda a, b: nx.rotary_embed(a, b, pos, freq), (q, k))
    a, _ = nx.rotary_embed(q, None, pos[0], freq)
    b, none = nx.rotary_embed(q, None, pos.expand(2, 4), freq)
    assert torch.equal(a, b) and none is None
    assert torch.equal(a, nx.rotary_embed(q, k, pos[0], freq)[0])


def test_distances_alone_count():
    """Scores of rotated queries and keys depend on the distance only."""
    freq = nx.rotary_frequencies(16)
    q, k = _rand(1, 1, 16), _rand(1, 1, 16, seed=3)
    scores = []
    for at in (0, 7, 100003):
        a, _ = nx.rotary_embed(q, None, torch.tensor([at + 11]), freq)
        b, _ = nx.rotary_embed(k, None, torch.tensor([at]), freq)
        scores.append(float((a * b).sum()))
    assert max(scores) - min(scores) < 1e-9


def test_frequencies():
    plain = nx.rotary_frequencies(64)
    assert plain.dtype == torch.float64 and plain.shape == (32,)
    assert plain[0] == 1 and math.isclose(plain[16], 10000 ** -0.5)
    assert torch.equal(nx.rotary_frequencies(64, scaling='linear', factor=4.0), plain / 4)
    base = nx.rotary_frequencies(64, scaling='base', factor=4.0)
    assert base[0] == 1 and math.isclose(base[-1], plain[-1] / 4)
    for scaling in ('ramp', 'bands'):
        w = nx.rotary_frequencies(64, scaling=scaling, factor=4.0, original_length=4096)
        turns = 4096 * plain / (2 * math.pi)
        ratio = w / plain
        fast, slow = turns > 64, turns < 0.5
        assert fast.any() and slow.any()
        assert (ratio[fast] == 1).all()
        torch.testing.assert_close(ratio[slow], torch.full_like(ratio[slow], 0.25))
        assert (ratio[1:] <= ratio[:-1] + 1e-15).all()
        same = nx.rotary_frequencies(64, scaling=scaling, factor=1.0, original_length=4096)
        torch.testing.assert_close(same, plain, rtol=1e-15, atol=0)


@pytest.mark.parametrize('scaling', ['ramp', 'bands'])
@pytest.mark.parametrize('length', [1, 6, 10, 64, 300, 10 ** 9, 10 ** 14])
def test_pairs_at_either_end(scaling, length):
    """Pairs that turn 32 times or more stay, those of one turn or less are divided,
    also where all of them do."""
    plain = nx.rotary_frequencies(16)
    ratio = nx.rotary_frequencies(16, scaling=scaling, factor=4.0, original_length=length) / plain
    turns = length * plain / (2 * math.pi)
    assert (ratio[turns >= 32 * (1 + 1e-12)] == 1).all()
    slow = ratio[turns <= 1 - 1e-12]
    torch.testing.assert_close(slow, torch.full_like(slow, 0.25))
    assert (ratio >= 0.25 - 1e-12).all() and (ratio <= 1).all()


def test_frequency_refusals():
    for kw in (
        {'dims': 7}, {'dims': 0}, {'dims': 8, 'base': 0.0}, {'dims': 8, 'factor': -1.0},
        {'dims': 8, 'scaling': 'cubic'}, {'dims': 2, 'scaling': 'base'},
        {'dims': 8, 'scaling': 'ramp'}, {'dims': 8, 'scaling': 'bands', 'original_length': 0},
        {'dims': 8, 'scaling': 'ramp', 'original_length': 9, 'fast_turns': 1.0},
        {'dims': 8, 'scaling': 'ramp', 'original_length': 9, 'base': 0.5},
    ):
        with pytest.raises(ValueError, match='rotary_frequencies'):
            nx.rotary_frequencies(**kw)


def test_packed_positions():
    off = torch.tensor([2, 4, 4, 7], dtype=torch.int32)
    start = torch.tensor([10, 20, 30], dtype=torch.int32)
    got = nx.packed_positions(off, 9, start)
    assert got.dtype == torch.int32 and got.tolist() == [0, 0, 10, 11, 30, 31, 32, 0, 0]
    assert nx.packed_positions(off, 9).tolist() == [0, 0, 0, 1, 0, 1, 2, 0, 0]
    assert nx.packed_positions(off, 0).shape == (0,)
    for args in ((off.long(), 9), (off[:1], 9), (off, -1), (off, 9, start[:2]), (off, 9, start.long())):
        with pytest.raises(ValueError, match='packed_positions'):
            nx.packed_positions(*args)


def test_refusals():
    q, k = torch.zeros(2, 3, 8), torch.zeros(1, 3, 8)
    pos, freq = torch.arange(3), nx.rotary_frequencies(8)
    for args in (
        (q[0], None, pos, freq), (q, k[:, :2], pos, freq), (q, k[..., :6], pos, freq),
        (q, k[None], pos, freq), (q, k.double(), pos, freq), (q.int(), None, pos, freq),
        (q, k, pos.float(), freq), (q, k, pos[:2], freq), (q, k, pos[:1], freq),
        (q, k, torch.tensor(1), freq), (q, k, pos[None, None], freq), (q, k, pos, freq[None]),
        (q, k, pos, freq.int()), (q, k, pos, nx.rotary_frequencies(10)), (q, k, pos, freq[:0]),
        (q, k, pos, freq.clone().requires_grad_(True)),
    ):
        with pytest.raises(ValueError, match='rotary_embed'):
            nx.rotary_embed(*args)


def _desc(B=1, T=5, H=4, Hk=2, D=64, R=64, dtype=_lib.NXA_BF16):
    d = _lib.NxaRotaryDesc()
    d.B, d.T, d.H, d.Hk, d.D, d.R, d.io_dtype, d.scale = B, T, H, Hk, D, R, dtype, 1.0
    d.pos_str[:] = (T, 1)
    for name, h in (('q', H), ('k', Hk)):
        for s in (getattr(d, f'{name}_str'), getattr(d, f'{name}_out_str')):
            s[:] = (h * T * D, T * D, D)
    return d


def test_check_codes():
    check = _lib.lib().nxa_rotary_check
    assert check(ctypes.byref(_desc())) == 0 and check(ctypes.byref(_desc(Hk=0, R=2, D=3))) == 0
    assert check(None) == _lib.NXA_E_ARG
    for bad, code in (
        (_desc(dtype=7), _lib.NXA_E_DTYPE), (_desc(T=0), _lib.NXA_E_SHAPE),
        (_desc(H=0), _lib.NXA_E_SHAPE), (_desc(D=257), _lib.NXA_E_UNSUPPORTED),
        (_desc(R=66), _lib.NXA_E_ARG), (_desc(R=3), _lib.NXA_E_ARG), (_desc(R=0), _lib.NXA_E_ARG),
        (_desc(B=1 << 20, T=1 << 10), _lib.NXA_E_SHAPE), (_desc(H=1 << 21), _lib.NXA_E_SHAPE),
    ):
        assert check(ctypes.byref(bad)) == code
    for field in ('q_str', 'k_out_str', 'pos_str'):
        d = _desc()
        getattr(d, field)[0] = -1
        assert check(ctypes.byref(d)) == _lib.NXA_E_LAYOUT
    run, ok = _lib.lib().nxa_rotary, 1 << 20
    d = ctypes.byref(_desc())
    assert run(d, None, ok, ok, ok, ok, ok, None) == _lib.NXA_E_ARG
    assert run(d, ok, None, ok, ok, ok, ok, None) == _lib.NXA_E_ARG
    assert run(d, ok, ok, ok, None, ok, ok, None) == _lib.NXA_E_ARG
    assert run(d, ok + 1, ok, ok, ok, ok, ok, None) == _lib.NXA_E_LAYOUT
