"""Checks and descriptor of a quantised pool (see :mod:`nitrix_amd.quantized`),
shared with the page operators of :mod:`nitrix_amd.paged`."""

from __future__ import annotations

import torch

from . import _lib
from .attention import _IO_DTYPES, _MAX_HEAD_DIM, HipNotTileable


def _check_quantized(name, k_pages, v_pages, scales, written=False) -> None:
    if k_pages.dtype != torch.uint8 or v_pages.dtype != torch.uint8:
        raise ValueError(
            f'{name}: k_pages and v_pages hold codes in uint8; got {k_pages.dtype}, '
            f'{v_pages.dtype}.'
        )
    if not scales.dtype.is_floating_point:
        raise ValueError(f'{name}: scales must be floating-point; got {scales.dtype}.')
    if k_pages.ndim != 4 or v_pages.ndim != 4 or scales.ndim != 4:
        raise ValueError(
            f'{name}: pages and scales must have four axes; got ndim {k_pages.ndim}, '
            f'{v_pages.ndim}, {scales.ndim}.'
        )
    slots = k_pages.shape[:3]
    if v_pages.shape[:3] != slots or scales.shape != (*slots, 4) or 0 in k_pages.shape or (
            0 in v_pages.shape):
        raise ValueError(
            f'{name}: k_pages, v_pages and scales (last axis 4) must hold the same, non-empty '
            f'pages; got {tuple(k_pages.shape)}, {tuple(v_pages.shape)} and '
            f'{tuple(scales.shape)}.'
        )
    if not k_pages.device == v_pages.device == scales.device:
        raise ValueError(
            f'{name}: k_pages, v_pages and scales must be on one device; got {k_pages.device}, '
            f'{v_pages.device}, {scales.device}.'
        )
    if written and any(
        s == 0 and n > 1
        for x in (k_pages, v_pages, scales)
        for s, n in zip(x.stride(), x.shape)
    ):
        raise ValueError(f'{name}: pages that share memory (a zero stride) cannot be written.')


def _bits_of(name, held: int, dims: int, which: str) -> int:
    """4 or 8: how many bits ``held`` bytes give each of ``dims`` elements."""
    for bits in (4, 8):
        if dims > 0 and dims * bits == 8 * held:
            return bits
    raise ValueError(
        f'{name}: {held} bytes a row of {which} hold {2 * held} elements in 4 bits or {held} in '
        f'8; got {dims}.'
    )


def _end_to_end(x: torch.Tensor, width: int) -> bool:
    """Whether the slots of each page and head lie end to end."""
    _, _, ps, _ = x.shape
    return x.stride(3) == 1 and (ps == 1 or x.stride(2) == width)


def _check_fused(k_pages, v_pages, scales, bits, *others) -> None:
    """Types, head dims and layouts of a pool the kernels read in place."""
    if scales.dtype not in _IO_DTYPES:
        raise HipNotTileable(
            f'fused quantised kernels support bfloat16, float16 and float32; got {scales.dtype}.'
        )
    for x in (k_pages, v_pages):
        d = x.shape[3] * 8 // bits
        if d > _MAX_HEAD_DIM or d % 8:
            raise HipNotTileable(
                f'fused quantised kernels require head dims <= {_MAX_HEAD_DIM} and multiples of '
                f'8; got {d}.'
            )
    for x in (k_pages, v_pages, scales):
        if not _end_to_end(x, x.shape[3]) or x.stride(0) % 4 or x.stride(1) % 4 or (
                x.data_ptr() % 16):
            raise HipNotTileable(
                'fused quantised kernels need a page and head\'s slots end to end, page and head '
                f'strides in multiples of 4 and 16-byte alignment; got strides {x.stride()}.'
            )
    p, hk, ps, _ = k_pages.shape
    if (p | ps) >> 30 or hk > 1 << 24:
        raise HipNotTileable('fused quantised kernels number up to 2^30 pages and slots.')
    for x in others:
        if x.dtype != scales.dtype:
            raise HipNotTileable(
                f'fused quantised kernels need the scales\' dtype {scales.dtype}; got {x.dtype}.'
            )
    _lib.lib()  # a missing library is an error, not a fallback


def _quant_desc(k_pages, v_pages, scales, bits) -> _lib.NxaQuantPoolDesc:
    desc = _lib.NxaQuantPoolDesc()
    desc.P, desc.Hk, desc.PS, width = k_pages.shape
    desc.D = width * 8 // bits
    desc.Dv = v_pages.shape[3] * 8 // bits
    desc.io_dtype = _IO_DTYPES[scales.dtype]
    desc.bits = bits
    desc.k_str[:] = k_pages.stride()[:2]
    desc.v_str[:] = v_pages.stride()[:2]
    desc.s_str[:] = scales.stride()[:2]
    return desc
