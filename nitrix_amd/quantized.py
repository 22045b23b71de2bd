"""A paged key-value cache of 4 or 8 bits an element.

The cache of :mod:`nitrix_amd.paged` with its pages quantised: for one row
(token and head) a scale ``s`` and a minimum ``z`` in the model's type, and for
each element a code ``c`` of ``bits`` bits, which stands for ``z + s c``.  Plain
tensors that the caller owns: ``k_pages`` uint8 ``(p, h_kv, page, d * bits / 8)``,
``v_pages`` uint8 ``(p, h_kv, page, d_v * bits / 8)`` (4 bits: element ``2 i`` in
the low half of byte ``i``) and ``scales`` ``(p, h_kv, page, 4)`` in the model's
type, a token's ``[s, z]`` of its key and of its value.  Page tables, lengths and
counts are those of :mod:`nitrix_amd.paged`.

* :func:`write_quantized_pages` -- new tokens' keys and values into their slots;
* :func:`read_quantized_pages` -- tokens back in the model's type, packed;
* :func:`quantized_paged_attention` -- one query token a sequence over its pages;
* :func:`~nitrix_amd.paged.fork_sequences`, ``compact_pages`` and ``copy_pages``
  move quantised pages where they are given ``scales=``.

At head dim 128 a token takes 136 bytes a head in 4 bits and 264 in 8, of 512 in
16.  The reference has no counterpart; engines and ``backend`` as in
:mod:`nitrix_amd.paged`, and the fused engine has no derivatives.
"""

from __future__ import annotations

import ctypes
import math
from typing import Optional

import torch

from . import _lib
from ._quant_pool import _bits_of, _check_dtype, _check_quantized, _fused_pool
from .attention import HipNotTileable, _has_tangent, default_scale
from .packed import _empty_like, _kernel_layout, _stream
from .paged import (
    _check_ints,
    _check_table,
    _check_written,
    _dispatch,
    _touched,
    _workspace,
)

__all__ = [
    'quantized_paged_attention',
    'read_quantized_pages',
    'write_quantized_pages',
]


# ---------------------------------------------------------------------------
# The format in stock tensor ops
# ---------------------------------------------------------------------------


def _quantise(x, bits):
    """Codes (one an element), scale and minimum of each row of ``x``."""
    top = (1 << bits) - 1
    lo, hi = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    acc = torch.promote_types(x.dtype, torch.float32)
    span = hi.to(acc) - lo.to(acc)
    good = torch.isfinite(x).all(-1, keepdim=True) & torch.isfinite(span)
    s = torch.where(good, span * (1 / top), math.nan).to(x.dtype)
    z = torch.where(good, lo, math.nan)
    live = torch.isfinite(s) & (s > 0)
    # (quotients in float64: a row next to a border)
    c = (x.double() - lo.double()) / torch.where(live, s, 1).double()
    c = torch.where(live, c, 0).round().clamp(0, top)
    return c.to(torch.uint8), s, z


def _pack(c, bits):
    return c if bits == 8 else c[..., 0::2] | c[..., 1::2] << 4


def _values(pages, scales, which, bits):
    """What the codes stand for, in at least float32."""
    acc = torch.promote_types(scales.dtype, torch.float32)
    c = pages if bits == 8 else torch.stack((pages & 15, pages >> 4), -1).flatten(-2)
    s, z = (scales[..., 2 * which + i, None].to(acc) for i in (0, 1))
    return c.to(acc) * s + z


def _slots(page_table, starts, offsets, t, p, ps):
    """Of each of t packed tokens the page and slot, and whether it has one."""
    b, m = page_table.shape
    tok = torch.arange(t, device=page_table.device)
    if offsets is None:
        seq, ok, pos = tok, torch.ones_like(tok, dtype=torch.bool), torch.zeros_like(tok)
    else:
        off = offsets.long()
        seq = torch.searchsorted(off, tok, right=True) - 1
        ok = (seq >= 0) & (seq < b)
        seq = seq.clamp(0, b - 1)
        pos = tok - off[seq]
    pos = pos + starts.long()[seq]
    ok = ok & (pos >= 0) & (pos < m * ps)
    pos = pos.clamp(0, m * ps - 1)
    page = page_table[seq, pos // ps].long()
    return page, pos % ps, ok & (page >= 0) & (page < p)


# ---------------------------------------------------------------------------
# Writing and reading back
# ---------------------------------------------------------------------------


def _reference_write(k_pages, v_pages, scales, k, v, page_table, starts, offsets, bits):
    page, slot, ok = _slots(page_table, starts, offsets, k.shape[1], k_pages.shape[0],
                            k_pages.shape[2])
    page, slot = page[ok], slot[ok]
    with torch.no_grad():
        for which, (pages, x) in enumerate(((k_pages, k), (v_pages, v))):
            c, s, z = _quantise(x.detach()[:, ok].transpose(0, 1).to(scales.dtype), bits)
            pages[page, :, slot] = _pack(c, bits)
            scales[page, :, slot, 2 * which] = s[..., 0]
            scales[page, :, slot, 2 * which + 1] = z[..., 0]


def _move(entry, pool, bits, k, v, page_table, starts, offsets) -> None:
    """Calls ``nxa_quant_write`` or ``nxa_quant_read``."""
    desc, ptrs = _fused_pool(*pool, bits)
    if page_table.stride(1) != 1:
        page_table = page_table.contiguous()
    starts = starts.contiguous()
    offsets = None if offsets is None else offsets.contiguous()
    b, m = page_table.shape
    ks, vs = k.stride(), v.stride()
    _lib.check(
        getattr(_lib.lib(), entry)(
            ctypes.byref(desc), *ptrs, k.data_ptr(), _lib.I64x2(ks[0], ks[1]), v.data_ptr(),
            _lib.I64x2(vs[0], vs[1]), k.shape[1], page_table.data_ptr(), page_table.stride(0),
            starts.data_ptr(), None if offsets is None else offsets.data_ptr(), b, m,
            _stream(k.device),
        )
    )


def _write_hip(k_pages, v_pages, scales, k, v, page_table, starts, offsets, bits):
    pool = (k_pages, v_pages, scales)
    _check_dtype(scales, k, v)
    k, v = _kernel_layout(k), _kernel_layout(v)
    _move('nxa_quant_write', pool, bits, k, v, page_table, starts, offsets)
    _touched(*pool)


def write_quantized_pages(
    k_pages: torch.Tensor,
    v_pages: torch.Tensor,
    scales: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    page_table: torch.Tensor,
    starts: torch.Tensor,
    offsets: Optional[torch.Tensor] = None,
    *,
    backend: str = 'auto',
) -> None:
    """Writes new tokens' keys and values into quantised pages, in place.

    k ``(h_kv, t, d)``, v ``(h_kv, t, d_v)`` in the scales' dtype, ``page_table``,
    ``starts`` and ``offsets`` as in :func:`~nitrix_amd.paged.write_pages`; bits a
    code (4 or 8) follow from the widths of the pages.  Of each row ``z`` is the
    minimum, ``s`` the range times ``1 / (2^bits - 1)`` (both in float32), rounded to
    the scales' dtype, and codes are the exact quotients ``(x - z) / s`` rounded to
    the nearest, ties to even.  A row that holds NaN or infinity, or whose range
    exceeds float32's, is NaN when it is read; a constant row is exact.

    The fused engine takes bfloat16, float16 and float32 and head dims up to 256
    in multiples of 8.  Two rows that share the page a token goes to write over
    each other: which of them a slot ends up with, codes and scales each, is not
    defined.
    """
    name = 'write_quantized_pages'
    _check_quantized(name, k_pages, v_pages, scales, written=True)
    hk = k_pages.shape[1]
    if k.ndim != 3 or v.ndim != 3 or k.shape[:2] != v.shape[:2] or k.shape[0] != hk:
        raise ValueError(
            f'{name}: k and v must be ({hk}, t, d) and ({hk}, t, d_v); got {tuple(k.shape)} and '
            f'{tuple(v.shape)}.'
        )
    bits = _bits_of(name, k_pages.shape[3], k.shape[2], 'k_pages')
    if _bits_of(name, v_pages.shape[3], v.shape[2], 'v_pages') != bits:
        raise ValueError(f'{name}: k_pages and v_pages must hold codes of as many bits.')
    if k.device != k_pages.device or v.device != k_pages.device:
        raise ValueError(
            f'{name}: k, v are on {k.device}, {v.device}, the pages on {k_pages.device}.'
        )
    _check_table(name, k.device, page_table, starts=(starts, (page_table.shape[0],)))
    b = page_table.shape[0]
    if offsets is not None:
        _check_ints(name, k.device, offsets=(offsets, (b + 1,)))
    elif k.shape[1] != b:
        raise ValueError(
            f'{name}: without offsets there is one token a sequence; got {k.shape[1]} tokens for '
            f'{b} sequences.'
        )
    _check_written(name, scales, k, v)
    if k.shape[1] == 0:
        return
    args = (k_pages, v_pages, scales, k, v, page_table, starts, offsets, bits)
    _dispatch(
        name, backend, k.device, lambda: _write_hip(*args), lambda: _reference_write(*args),
        (tuple(k.shape), tuple(k_pages.shape)), scales.dtype,
    )


def _reference_read(k_pages, v_pages, scales, page_table, starts, offsets, t, bits):
    page, slot, ok = _slots(page_table, starts, offsets, t, k_pages.shape[0], k_pages.shape[2])
    page = torch.where(ok, page, 0)
    with torch.no_grad():
        sc = scales[page, :, slot]
        out = []
        for which, pages in enumerate((k_pages, v_pages)):
            x = _values(pages[page, :, slot], sc, which, bits)
            # (a scale rounded up takes the largest code past the type's largest number)
            finite = (sc[..., 2 * which:2 * which + 2] < math.inf).all(-1, keepdim=True)
            top = torch.where(finite, torch.finfo(scales.dtype).max, math.inf).to(x.dtype)
            x = torch.minimum(x, top).to(scales.dtype)
            out.append(torch.where(ok[:, None, None], x, 0).transpose(0, 1))
    return tuple(out)


def _read_hip(k_pages, v_pages, scales, page_table, starts, offsets, t, bits):
    hk = k_pages.shape[1]
    # Tokens before heads, as a projection would leave them.
    k, v = (
        torch.empty((t, hk, x.shape[3] * 8 // bits), dtype=scales.dtype, device=x.device)
        .transpose(0, 1)
        for x in (k_pages, v_pages)
    )
    _move('nxa_quant_read', (k_pages, v_pages, scales), bits, k, v, page_table, starts, offsets)
    return k, v


def read_quantized_pages(
    k_pages: torch.Tensor,
    v_pages: torch.Tensor,
    scales: torch.Tensor,
    page_table: torch.Tensor,
    starts: torch.Tensor,
    offsets: Optional[torch.Tensor] = None,
    t: Optional[int] = None,
    *,
    bits: int = 4,
    backend: str = 'auto',
):
    """The keys ``(h_kv, t, d)`` and values ``(h_kv, t, d_v)`` that quantised
    pages of ``bits`` bits hold, in the scales' dtype.

    The mirror of :func:`write_quantized_pages`: with ``offsets`` ``(b + 1,)`` and
    the number ``t`` of tokens, token ``offsets[i] + j`` is the one at position
    ``starts[i] + j`` of sequence ``i``; without, there is one a sequence, at
    ``starts[i]``.  ``z + s c`` is rounded once, and where the rounding of ``s`` took it
    past the type's largest number it is that.  Tokens of no sequence, outside the
    table or in no page are zero.  For packed attention over tokens that a cache
    holds already, and for attention over what the cache holds of new ones.
    """
    name = 'read_quantized_pages'
    if bits not in (4, 8):
        raise ValueError(f'{name}: bits must be 4 or 8; got {bits}.')
    _check_quantized(name, k_pages, v_pages, scales)
    dev = k_pages.device
    _check_table(name, dev, page_table, starts=(starts, (page_table.shape[0],)))
    b = page_table.shape[0]
    if offsets is not None:
        _check_ints(name, dev, offsets=(offsets, (b + 1,)))
        if t is None:
            raise ValueError(f'{name}: with offsets the number t of tokens must be given.')
    elif t is not None and t != b:
        raise ValueError(
            f'{name}: without offsets there is one token a sequence; got t={t} for {b} sequences.'
        )
    t = b if t is None else int(t)
    if t < 0:
        raise ValueError(f'{name}: t must not be negative; got {t}.')
    _check_written(name, scales)
    args = (k_pages, v_pages, scales, page_table, starts, offsets, t, bits)
    if t == 0:
        return _reference_read(*args)
    return _dispatch(
        name, backend, dev, lambda: _read_hip(*args), lambda: _reference_read(*args),
        (t, tuple(k_pages.shape)), scales.dtype,
    )


# ---------------------------------------------------------------------------
# Attention
# ---------------------------------------------------------------------------


def _reference_attention(q, k_pages, v_pages, scales, page_table, lengths, scale, bits):
    p, hk, ps, _ = k_pages.shape
    b, h, _ = q.shape
    m = page_table.shape[1]
    acc = torch.promote_types(torch.promote_types(q.dtype, scales.dtype), torch.float32)
    real = (page_table >= 0) & (page_table < p)
    ids = torch.where(real, page_table, 0).long()
    seen = torch.arange(m * ps, device=q.device)[None] < lengths[:, None]
    seen = seen & real.repeat_interleave(ps, dim=1)

    def gather(pages, which):
        x = _values(pages[ids], scales[ids], which, bits).to(acc)
        x = x.transpose(1, 2).reshape(b, hk, m * ps, -1)
        return torch.where(seen[:, None, :, None], x, 0)  # whatever unused slots hold

    k, v = gather(k_pages, 0), gather(v_pages, 1)
    s = torch.matmul(q.to(acc).reshape(b, hk, h // hk, -1), k.transpose(-1, -2).contiguous()) * scale
    s = torch.where(seen[:, None, None, :], s, -math.inf)
    top = s.amax(-1, keepdim=True)
    w = torch.exp(s - torch.where(top == -math.inf, 0, top))
    total = w.sum(-1, keepdim=True)
    out = torch.matmul(w, v) / torch.where(total == 0, 1, total)
    return out.reshape(b, h, -1).to(torch.promote_types(q.dtype, scales.dtype))


def _attention_hip(q, k_pages, v_pages, scales, page_table, lengths, scale, bits):
    _check_dtype(scales, q)
    b, h, _ = q.shape
    if (b | h) >> 31:
        raise HipNotTileable('fused quantised attention numbers sequences and heads in 31 bits.')
    if torch.is_grad_enabled() and (q.requires_grad or scales.requires_grad):
        raise HipNotTileable('fused quantised attention has no backward pass.')
    if _has_tangent(q, scales):
        raise HipNotTileable('fused quantised attention has no forward-mode derivative.')
    desc, ptrs = _fused_pool(k_pages, v_pages, scales, bits)
    q = _kernel_layout(q)
    if page_table.stride(1) != 1:
        page_table = page_table.contiguous()
    lengths = lengths.contiguous()
    m = page_table.shape[1]
    o = _empty_like(q, desc.Dv)
    lib, at = _lib.lib(), ctypes.byref(desc)
    need = lib.nxa_quant_paged_workspace_bytes(at, b, m, h)  # (0: none, or it will say why)
    ws = _workspace(need, q.device) if need else None
    qs, os = q.stride(), o.stride()
    _lib.check(
        lib.nxa_quant_paged_fwd(
            at, *ptrs, q.data_ptr(), _lib.I64x2(qs[0], qs[1]), page_table.data_ptr(),
            page_table.stride(0), lengths.data_ptr(), b, m, h, scale, o.data_ptr(),
            _lib.I64x2(os[0], os[1]), None if ws is None else ws.data_ptr(), need,
            _stream(q.device),
        )
    )
    return o


def quantized_paged_attention(
    q: torch.Tensor,
    k_pages: torch.Tensor,
    v_pages: torch.Tensor,
    scales: torch.Tensor,
    page_table: torch.Tensor,
    lengths: torch.Tensor,
    *,
    scale: Optional[float] = None,
    backend: str = 'auto',
) -> torch.Tensor:
    """Attention of one new token a sequence over its quantised pages.

    :func:`~nitrix_amd.paged.paged_attention` of what the codes stand for: q
    ``(b, h, d)`` in the scales' dtype, the result ``(b, h, d_v)``.  Bits a code (4
    or 8) follow from ``d`` and the pages' width.  Keys and values are not rounded
    to the type on the way, and scores, weights and sums are float32's; tokens in no
    page, lengths outside the table's room and rows without tokens are treated as
    there.  A page row has room for less than 2^31 - 4096 tokens.  Keys past 2^100, and
    values whose sum over the tokens passes 2^119, leave float32; of values' scales
    below 2^-90 digits are lost.

    The fused engine takes bfloat16, float16 and float32, head dims up to 256 in
    multiples of 8 and pages of any number of slots (a multiple of 16 is fastest, as
    are head dims of 64, 128 and 256); derivatives are the reference engine's.
    """
    name = 'quantized_paged_attention'
    _check_quantized(name, k_pages, v_pages, scales)
    if q.ndim != 3:
        raise ValueError(f'{name}: q must be (b, h, d); got {tuple(q.shape)}.')
    bits = _bits_of(name, k_pages.shape[3], q.shape[2], 'k_pages')
    if q.shape[1] == 0 or q.shape[1] % k_pages.shape[1]:
        raise ValueError(
            f'{name}: query heads must be a multiple of the {k_pages.shape[1]} key-value heads; '
            f'got {q.shape[1]}.'
        )
    if q.device != k_pages.device:
        raise ValueError(f'{name}: q is on {q.device}, the pages on {k_pages.device}.')
    b = q.shape[0]
    _check_ints(name, q.device, page_table=(page_table, (b, None)), lengths=(lengths, (b,)))
    if not 0 < page_table.shape[1] < 1 << 30:
        raise ValueError(f'{name}: page_table has no columns, or 2^30 or more.')
    scale = float(default_scale(q.shape[2]) if scale is None else scale)
    if b == 0:
        return q.new_zeros(0, q.shape[1], v_pages.shape[3] * 8 // bits)
    args = (q, k_pages, v_pages, scales, page_table, lengths, scale, bits)
    return _dispatch(
        name, backend, q.device, lambda: _attention_hip(*args),
        lambda: _reference_attention(*args), (tuple(q.shape), tuple(k_pages.shape)), q.dtype,
    )
