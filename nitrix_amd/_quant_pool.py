"""Checks and descriptor of a quantised pool (see :mod:`nitrix_amd.quantized`),
shared with the page operators of :mod:`nitrix_amd.paged`.

A decoding step's calls are bound by the host, so the checks are one condition
each for pools as they usually are, and what is wrong is found out afterwards."""

from __future__ import annotations

import torch

from . import _lib
from .attention import _IO_DTYPES, _MAX_HEAD_DIM, HipNotTileable

_U8 = torch.uint8


def _check_quantized(name, k_pages, v_pages, scales, written=False) -> None:
    ks, vs, ss = k_pages.shape, v_pages.shape, scales.shape
    if not (
        k_pages.dtype is _U8
        and v_pages.dtype is _U8
        and scales.dtype.is_floating_point
        and len(ks) == len(vs) == len(ss) == 4
        and ks[0] == vs[0] == ss[0] > 0
        and ks[1] == vs[1] == ss[1] > 0
        and ks[2] == vs[2] == ss[2] > 0
        and ks[3] > 0
        and vs[3] > 0
        and ss[3] == 4
        and k_pages.device == v_pages.device == scales.device
    ):
        _say_what_is_wrong(name, k_pages, v_pages, scales)
    if written and (0 in k_pages.stride() or 0 in v_pages.stride() or 0 in scales.stride()) and any(
        s == 0 and n > 1
        for x in (k_pages, v_pages, scales)
        for s, n in zip(x.stride(), x.shape)
    ):
        raise ValueError(f'{name}: pages that share memory (a zero stride) cannot be written.')


def _say_what_is_wrong(name, k_pages, v_pages, scales) -> None:
    if k_pages.dtype != _U8 or v_pages.dtype != _U8:
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
    raise ValueError(
        f'{name}: k_pages, v_pages and scales must be on one device; got {k_pages.device}, '
        f'{v_pages.device}, {scales.device}.'
    )


def _bits_of(name, held: int, dims: int, which: str) -> int:
    """4 or 8: how many bits ``held`` bytes give each of ``dims`` elements."""
    if dims == 2 * held:
        return 4
    if dims == held:
        return 8
    raise ValueError(
        f'{name}: {held} bytes a row of {which} hold {2 * held} elements in 4 bits or {held} in '
        f'8; got {dims}.'
    )


def _page_strides(x: torch.Tensor, heads: int, slots: int, width: int):
    """Page and head strides of a pool tensor whose slots lie end to end."""
    if x.is_contiguous():
        s0, s1 = heads * slots * width, slots * width
    else:
        s0, s1, s2, s3 = x.stride()
        if s3 != 1 or (slots > 1 and s2 != width):
            raise HipNotTileable(
                "fused quantised kernels need a page and head's slots end to end; got strides "
                f'{x.stride()}.'
            )
    if (s0 | s1) % 4:
        raise HipNotTileable(
            'fused quantised kernels need page and head strides in multiples of 4; got '
            f'{x.stride()}.'
        )
    return s0, s1


def _fused_pool(k_pages, v_pages, scales, bits):
    """Descriptor of a pool whose type, head dims and layout the kernels take,
    and its pointers."""
    io_dtype = _IO_DTYPES.get(scales.dtype)
    if io_dtype is None:
        raise HipNotTileable(
            f'fused quantised kernels support bfloat16, float16 and float32; got {scales.dtype}.'
        )
    p, hk, ps, kw = k_pages.shape
    vw = v_pages.shape[3]
    d, dv = (2 * kw, 2 * vw) if bits == 4 else (kw, vw)
    if d > _MAX_HEAD_DIM or dv > _MAX_HEAD_DIM or (d | dv) % 8:
        raise HipNotTileable(
            f'fused quantised kernels require head dims <= {_MAX_HEAD_DIM} and multiples of 8; '
            f'got {d} and {dv}.'
        )
    ptrs = k_pages.data_ptr(), v_pages.data_ptr(), scales.data_ptr()
    if (ptrs[0] | ptrs[1] | ptrs[2]) % 16:
        raise HipNotTileable('fused quantised kernels need pages and scales 16-byte aligned.')
    if (p | ps) >> 30 or hk > 1 << 24:
        raise HipNotTileable('fused quantised kernels number up to 2^30 pages and slots.')
    pair = _lib.I64x2
    desc = _lib.NxaQuantPoolDesc(
        p, hk, ps, d, dv, io_dtype, bits,
        pair(*_page_strides(k_pages, hk, ps, kw)), pair(*_page_strides(v_pages, hk, ps, vw)),
        pair(*_page_strides(scales, hk, ps, 4)),
    )
    return desc, ptrs


def _check_dtype(scales, *others) -> None:
    for x in others:
        if x.dtype != scales.dtype:
            raise HipNotTileable(
                f"fused quantised kernels need the scales' dtype {scales.dtype}; got {x.dtype}."
            )
