"""The largest calls of the paged caches and the rotary positions: refused before
anything is launched where a grid or a number would not hold them (CPU only)."""

from __future__ import annotations

import ctypes

import pytest
import torch

import nitrix_amd as nx
from nitrix_amd import _lib

OK = 1 << 20  # a pointer that no check looks behind


def _quant(Hk=2, PS=16, D=64, Dv=64):
    d = _lib.NxaQuantPoolDesc()
    d.P, d.Hk, d.PS, d.D, d.Dv, d.io_dtype, d.bits = 8, Hk, PS, D, Dv, _lib.NXA_BF16, 4
    d.k_str[:] = (Hk * PS * D // 2, PS * D // 2)
    d.v_str[:] = (Hk * PS * Dv // 2, PS * Dv // 2)
    d.s_str[:] = (Hk * PS * 4, PS * 4)
    return d


def _plain(Hk=2, PS=16, D=64, Dv=64):
    d = _lib.NxaPoolDesc()
    d.P, d.Hk, d.PS, d.D, d.Dv, d.io_dtype = 8, Hk, PS, D, Dv, _lib.NXA_BF16
    d.k_str[:] = (Hk * PS * D, PS * D, D)
    d.v_str[:] = (Hk * PS * Dv, PS * Dv, Dv)
    return d


@pytest.mark.parametrize('t', [(1 << 26) - 3, (1 << 26) - 1])
def test_tokens_whose_grid_has_2_32_threads(t):
    """Four tokens a block of 256 threads: 2^24 blocks are one too many."""
    lib, s2 = _lib.lib(), _lib.I64x2(64, 128)
    q, p = ctypes.byref(_quant()), ctypes.byref(_plain())
    for move in (lib.nxa_quant_write, lib.nxa_quant_read):
        assert move(q, OK, OK, OK, OK, s2, OK, s2, t, OK, 3, OK, OK, 2, 3,
                    None) == _lib.NXA_E_SHAPE
    assert lib.nxa_pages_write(p, OK, OK, OK, s2, OK, s2, t, OK, 3, OK, OK, 2, 3,
                               None) == _lib.NXA_E_SHAPE


@pytest.mark.parametrize('h', [(1 << 23) - 1, 1 << 23, (1 << 23) + 1, 1 << 24])
def test_heads_whose_zeros_pass_2_31(h):
    """A sequence without tokens is zeroed by 256 threads, whose count of H Dv
    elements steps past the last by up to 255."""
    lib, s2 = _lib.lib(), _lib.I64x2(64, 128)
    q, p = (ctypes.byref(f(Hk=1, D=256, Dv=256)) for f in (_quant, _plain))
    fits = h * 256 <= (1 << 31) - 256
    # (a table of 2 pages: a block a row in each, no workspace; of 200: some)
    assert (lib.nxa_quant_paged_workspace_bytes(q, 1, 200, h) > 0) == fits
    assert (lib.nxa_paged_workspace_bytes(p, 1, 200, h) > 0) == fits
    if not fits:
        assert lib.nxa_quant_paged_fwd(q, OK, OK, OK, OK, s2, OK, 2, OK, 1, 2, h, 1.0, OK, s2, None,
                                       0, None) == _lib.NXA_E_SHAPE
        assert lib.nxa_paged_fwd(p, OK, OK, OK, s2, OK, 2, OK, 1, 2, h, 1.0, OK, s2, None, 0,
                                 None) == _lib.NXA_E_SHAPE


def test_extents_past_31_bits_are_declined():
    """The C ABI's extents are 32-bit: 2^32 + 1 must not arrive as 1 (expanded
    tensors, so that nothing is that large)."""
    from nitrix_amd import paged, quantized, rotary
    from nitrix_amd.attention import HipNotTileable

    most, bf16 = (1 << 32) + 1, torch.bfloat16
    x = torch.zeros(1, 1, 1, 8, dtype=bf16)
    pos, freq = torch.zeros(1, dtype=torch.int32), torch.ones(4, dtype=torch.float64)
    for q, k in (
        (x.expand(most, 1, 1, 8), None), (x.expand(1, most, 1, 8), None),
        (x.expand(1, 1, most, 8), None), (x[0], x[0].expand(most, 1, 8)),
        (x.expand(1 << 16, 1, 1, 8)[:, None].expand(1 << 16, 1 << 16, 1, 1, 8), None),
    ):
        p = pos.expand(q.shape[-2])
        with pytest.raises(HipNotTileable, match='31 bits'):
            rotary._rotary_hip(q, k, p, freq, False, 1.0)
    pages = torch.zeros(2, 1, 16, 8, dtype=bf16)
    codes, sc = torch.zeros(2, 1, 16, 8, dtype=torch.uint8), torch.zeros(2, 1, 16, 4, dtype=bf16)
    table = torch.zeros(1, 1, dtype=torch.int32)
    for b, h in ((most, 1), (1, most)):
        q, t, n = x[0].expand(b, h, 8), table.expand(b, 1), pos.expand(b)
        with pytest.raises(HipNotTileable, match='31 bits'):
            paged._paged_hip(q, pages, pages, t, n, 1.0)
        with pytest.raises(HipNotTileable, match='31 bits'):
            quantized._attention_hip(q, codes, codes, sc, t, n, 1.0, 8)
