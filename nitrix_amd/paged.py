"""A paged key-value cache: attention of one new token over it, and what fills
and manages its pages.

The cache is plain tensors that the caller owns.  A *pool* is ``k_pages``
``(p, h_kv, page, d)`` and ``v_pages`` ``(p, h_kv, page, d_v)``: ``p`` pages of
``page`` token slots (any strides with unit stride over the head dim).  A
*page table* ``(b, m)`` names each sequence's pages in order, ``lengths``
``(b,)`` its tokens: token ``j`` of sequence ``i`` is slot ``j % page`` of page
``page_table[i, j // page]``.  An entry outside ``0 .. p - 1`` (by convention
-1) is no page.  ``refs`` ``(p,)`` counts how many table entries name a page; a
page that none names is free.  All of these are int32 on the pool's device and
never read on the host by the fused engine, so calls can be captured in a
graph.

* :func:`paged_attention` -- one query token a sequence over its pages;
* :func:`write_pages` -- new tokens' keys and values into their slots;
* :func:`extend_sequences`, :func:`fork_sequences`, :func:`free_sequences` --
  tables and counts for growing, forking and ended sequences;
* :func:`compact_pages`, :func:`copy_pages` -- moving pages.

With :func:`~nitrix_amd.packed.packed_attention` for the prompts they serve a
model: prompt keys and values are written while their attention runs packed,
then each new token is written and attends its sequence's pages.  The fused
engine has no derivatives.  The reference has no counterpart; engines and
``backend`` as in :func:`~nitrix_amd.attention.scaled_dot_product_attention`
(``'jax'``: the same functions in stock tensor ops).

Page contents change in place (a cache fills most of the memory); tables,
lengths and counts are returned anew.
"""

from __future__ import annotations

import array
import ctypes
import math
from typing import Optional, Sequence, Union

import torch

from . import _lib
from ._backend import NitrixBackendError, fallback, resolve_backend
from .attention import (
    _IO_DTYPES,
    _MAX_HEAD_DIM,
    HipNotTileable,
    _has_tangent,
    _row_stride_ok,
    default_scale,
)
from .packed import _empty_like, _kernel_layout, _on, _stream

__all__ = [
    'compact_pages',
    'copy_pages',
    'extend_sequences',
    'fork_sequences',
    'free_sequences',
    'paged_attention',
    'write_pages',
]


# ---------------------------------------------------------------------------
# Checks
# ---------------------------------------------------------------------------


def _check_pool(name, k_pages, v_pages, written=False) -> None:
    if k_pages.ndim != 4 or v_pages.ndim != 4:
        raise ValueError(
            f'{name}: pages must be (p, h_kv, page, d); got ndim {k_pages.ndim}, {v_pages.ndim}.'
        )
    if k_pages.shape[:3] != v_pages.shape[:3] or 0 in k_pages.shape or 0 in v_pages.shape:
        raise ValueError(
            f'{name}: k_pages and v_pages must hold the same, non-empty pages; got '
            f'{tuple(k_pages.shape)} and {tuple(v_pages.shape)}.'
        )
    if k_pages.device != v_pages.device or k_pages.dtype != v_pages.dtype:
        raise ValueError(
            f'{name}: k_pages and v_pages must share device and dtype; got {k_pages.device} '
            f'{k_pages.dtype}, {v_pages.device} {v_pages.dtype}.'
        )
    if written and (0 in k_pages.stride() or 0 in v_pages.stride()) and any(
        s == 0 and n > 1 for x in (k_pages, v_pages) for s, n in zip(x.stride(), x.shape)
    ):
        raise ValueError(f'{name}: pages that share memory (a zero stride) cannot be written.')


def _check_ints(name, device, **arrays) -> None:
    """int32 arrays of the given shapes (None: any size) on ``device``."""
    for arg, (x, shape) in arrays.items():
        have = x.shape
        ok = have == shape or (
            len(have) == len(shape) and all(s is None or s == n for s, n in zip(shape, have))
        )
        if x.dtype != torch.int32 or not ok:
            want = ', '.join('n' if s is None else str(s) for s in shape)
            raise ValueError(
                f'{name}: {arg} must be int32 of shape ({want}); got {x.dtype} of shape {tuple(have)}.'
            )
        if x.device != device:
            raise ValueError(f'{name}: {arg} is on {x.device}, expected {device}.')


def _check_table(name, device, page_table, **arrays) -> None:
    _check_ints(name, device, page_table=(page_table, (None, None)), **arrays)
    if 0 in page_table.shape or max(page_table.shape) >> 30:
        raise ValueError(
            f'{name}: page_table must not be empty nor have 2^30 rows or columns; got '
            f'{tuple(page_table.shape)}.'
        )


def _check_written(name, *tensors) -> None:
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
        raise ValueError(f'{name} is not differentiable; detach its inputs or use no_grad.')
    if _has_tangent(*tensors):
        raise ValueError(f'{name} is not differentiable; its inputs carry forward-mode tangents.')


def _check_fused(k_pages, v_pages, *others) -> None:
    """Types, head dims and layouts of a pool the kernels read in place."""
    if k_pages.dtype not in _IO_DTYPES:
        raise HipNotTileable(
            f'fused paged kernels support bfloat16, float16 and float32; got {k_pages.dtype}.'
        )
    es = k_pages.element_size()
    epc = 16 // es
    for x in (k_pages, v_pages):
        d = x.shape[3]
        if d > _MAX_HEAD_DIM or d % epc:
            raise HipNotTileable(
                f'fused paged kernels require head dims <= {_MAX_HEAD_DIM} and multiples of '
                f'{epc}; got {d}.'
            )
        s0, s1, s2, s3 = x.stride()
        if (
            s3 != 1
            or (s0 | s1 | s2) % epc
            or x.data_ptr() % 16
            or not _row_stride_ok(s2, es)
        ):
            raise HipNotTileable(
                f'fused paged kernels need 16-byte aligned rows; got strides {x.stride()}.'
            )
    p, hk, ps, _ = k_pages.shape
    if (p | hk | ps) >> 30:
        raise HipNotTileable('fused paged kernels number up to 2^30 pages, heads and slots.')
    for x in others:
        if x.dtype != k_pages.dtype:
            raise HipNotTileable(f'fused paged kernels need one dtype; got {x.dtype}.')
    _lib.lib()  # a missing library is an error, not a fallback


def _pool_desc(k_pages, v_pages) -> _lib.NxaPoolDesc:
    desc = _lib.NxaPoolDesc()
    desc.P, desc.Hk, desc.PS, desc.D = k_pages.shape
    desc.Dv = v_pages.shape[3]
    desc.io_dtype = _IO_DTYPES[k_pages.dtype]
    desc.k_str[:] = k_pages.stride()[:3]
    desc.v_str[:] = v_pages.stride()[:3]
    return desc


def _workspace(nbytes: int, device) -> torch.Tensor:
    return torch.empty(max(nbytes, 16), dtype=torch.uint8, device=device)


def _touched(*pages) -> None:
    """Tell autograd that a kernel wrote these tensors."""
    for x in pages:
        if not x.is_inference():
            torch.autograd.graph.increment_version(x)


def _dispatch(name, backend, device, fused, reference, shapes, dtype):
    """Runs ``fused`` or, where it declines or another engine is asked for,
    ``reference``."""
    if resolve_backend(backend, device) == 'hip':
        try:
            with _on(device):
                return fused()
        except (HipNotTileable, _lib.NxaShapeError) as exc:
            fallback(
                function=name,
                requested='hip',
                resolved='jax',
                reason=f'the fused kernel does not support this input ({exc})',
                shapes=shapes,
                dtype=dtype,
            )
        except _lib.HipLibraryMissing as exc:
            raise NitrixBackendError(str(exc)) from exc
    return reference()


# ---------------------------------------------------------------------------
# Attention
# ---------------------------------------------------------------------------


def _reference_paged(q, k_pages, v_pages, page_table, lengths, scale):
    p, hk, ps, _ = k_pages.shape
    b, h, _ = q.shape
    m = page_table.shape[1]
    acc = torch.promote_types(torch.promote_types(q.dtype, k_pages.dtype), torch.float32)
    real = (page_table >= 0) & (page_table < p)
    ids = torch.where(real, page_table, 0).long()
    seen = torch.arange(m * ps, device=q.device)[None] < lengths[:, None]
    seen = seen & real.repeat_interleave(ps, dim=1)

    def gather(pages):
        x = pages[ids].to(acc).transpose(1, 2).reshape(b, hk, m * ps, -1)
        return torch.where(seen[:, None, :, None], x, 0)  # whatever unused slots hold

    k, v = gather(k_pages), gather(v_pages)
    s = torch.matmul(q.to(acc).reshape(b, hk, h // hk, -1), k.transpose(-1, -2).contiguous()) * scale
    s = torch.where(seen[:, None, None, :], s, -math.inf)
    top = s.amax(-1, keepdim=True)
    w = torch.exp(s - torch.where(top == -math.inf, 0, top))
    total = w.sum(-1, keepdim=True)
    out = torch.matmul(w, v) / torch.where(total == 0, 1, total)
    return out.reshape(b, h, -1).to(torch.promote_types(q.dtype, k_pages.dtype))


def _paged_hip(q, k_pages, v_pages, page_table, lengths, scale):
    _check_fused(k_pages, v_pages, q)
    if torch.is_grad_enabled() and any(x.requires_grad for x in (q, k_pages, v_pages)):
        raise HipNotTileable('fused paged attention has no backward pass.')
    if _has_tangent(q, k_pages, v_pages):
        raise HipNotTileable('fused paged attention has no forward-mode derivative.')
    q = _kernel_layout(q)
    if page_table.stride(1) != 1:
        page_table = page_table.contiguous()
    lengths = lengths.contiguous()
    b, h, _ = q.shape
    m = page_table.shape[1]
    o = _empty_like(q, v_pages.shape[3])
    lib = _lib.lib()
    desc = _pool_desc(k_pages, v_pages)
    ws = _workspace(lib.nxa_paged_workspace_bytes(ctypes.byref(desc), b, m, h), q.device)
    _lib.check(
        lib.nxa_paged_fwd(
            ctypes.byref(desc), k_pages.data_ptr(), v_pages.data_ptr(), q.data_ptr(),
            _lib.I64x2(*q.stride()[:2]), page_table.data_ptr(), page_table.stride(0),
            lengths.data_ptr(), b, m, h, scale, o.data_ptr(), _lib.I64x2(*o.stride()[:2]),
            ws.data_ptr(), ws.numel(), _stream(q.device),
        )
    )
    return o


def paged_attention(
    q: torch.Tensor,
    k_pages: torch.Tensor,
    v_pages: torch.Tensor,
    page_table: torch.Tensor,
    lengths: torch.Tensor,
    *,
    scale: Optional[float] = None,
    backend: str = 'auto',
) -> torch.Tensor:
    """Attention of one new token a sequence over its pages.

    q ``(b, h, d)``; the result ``(b, h, d_v)`` is ``softmax(scale * q k^T) v``
    over the first ``lengths[i]`` tokens of sequence ``i`` (the new token's key
    and value among them once :func:`write_pages` has put them there); query
    head ``j`` reads key-value head ``j // (h / h_kv)``; ``scale`` defaults to
    ``1/sqrt(d)``.  Lengths below zero count as zero, ones past the table's
    room as that room.  Tokens in no page take no part.  A row without tokens
    is zero (as is one whose scores are all -inf), and what unused slots hold,
    NaN or not, reaches no result.

    The fused engine takes bfloat16, float16 and float32, head dims up to 256
    (multiples of 8, 4 in float32) and pages of any number of slots (a
    multiple of 16 is fastest); derivatives, backward and forward mode, are the
    reference engine's.
    """
    _check_pool('paged_attention', k_pages, v_pages)
    if q.ndim != 3 or q.shape[2] != k_pages.shape[3]:
        raise ValueError(
            f'paged_attention: q must be (b, h, d) with d={k_pages.shape[3]}; got '
            f'{tuple(q.shape)}.'
        )
    if q.shape[1] == 0 or q.shape[1] % k_pages.shape[1]:
        raise ValueError(
            f'paged_attention: query heads must be a multiple of the {k_pages.shape[1]} '
            f'key-value heads; got {q.shape[1]}.'
        )
    if q.device != k_pages.device:
        raise ValueError(f'paged_attention: q is on {q.device}, the pages on {k_pages.device}.')
    b = q.shape[0]
    _check_ints('paged_attention', q.device, page_table=(page_table, (b, None)),
                lengths=(lengths, (b,)))
    if not 0 < page_table.shape[1] < 1 << 30:
        raise ValueError('paged_attention: page_table has no columns, or 2^30 or more.')
    scale = float(default_scale(q.shape[2]) if scale is None else scale)
    args = (q, k_pages, v_pages, page_table, lengths, scale)
    if b == 0:
        return q.new_zeros(0, q.shape[1], v_pages.shape[3])
    return _dispatch(
        'paged_attention', backend, q.device, lambda: _paged_hip(*args),
        lambda: _reference_paged(*args), (tuple(q.shape), tuple(k_pages.shape)), q.dtype,
    )


# ---------------------------------------------------------------------------
# Writing tokens
# ---------------------------------------------------------------------------


def _reference_write(k_pages, v_pages, k, v, page_table, starts, offsets):
    p, _, ps, _ = k_pages.shape
    b, m = page_table.shape
    t = k.shape[1]
    tok = torch.arange(t, device=k.device)
    pos = torch.zeros(t, dtype=torch.long, device=k.device)
    if offsets is None:
        seq, ok = tok, torch.ones(t, dtype=torch.bool, device=k.device)
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
    ok = ok & (page >= 0) & (page < p)
    page, slot = page[ok], (pos % ps)[ok]
    with torch.no_grad():
        k_pages[page, :, slot] = k.detach()[:, ok].transpose(0, 1).to(k_pages.dtype)
        v_pages[page, :, slot] = v.detach()[:, ok].transpose(0, 1).to(v_pages.dtype)


def _write_hip(k_pages, v_pages, k, v, page_table, starts, offsets):
    _check_fused(k_pages, v_pages, k, v)
    k, v = _kernel_layout(k), _kernel_layout(v)
    if page_table.stride(1) != 1:
        page_table = page_table.contiguous()
    starts = starts.contiguous()
    offsets = None if offsets is None else offsets.contiguous()
    desc = _pool_desc(k_pages, v_pages)
    b, m = page_table.shape
    _lib.check(
        _lib.lib().nxa_pages_write(
            ctypes.byref(desc), k_pages.data_ptr(), v_pages.data_ptr(), k.data_ptr(),
            _lib.I64x2(*k.stride()[:2]), v.data_ptr(), _lib.I64x2(*v.stride()[:2]), k.shape[1],
            page_table.data_ptr(), page_table.stride(0), starts.data_ptr(),
            None if offsets is None else offsets.data_ptr(), b, m, _stream(k.device),
        )
    )
    _touched(k_pages, v_pages)


def write_pages(
    k_pages: torch.Tensor,
    v_pages: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    page_table: torch.Tensor,
    starts: torch.Tensor,
    offsets: Optional[torch.Tensor] = None,
    *,
    backend: str = 'auto',
) -> None:
    """Writes new tokens' keys and values into their pages, in place.

    k ``(h_kv, t, d)``, v ``(h_kv, t, d_v)``, heads first as in
    :func:`~nitrix_amd.packed.packed_attention` and read in place from any
    strides.  With ``offsets`` ``(b + 1,)`` (packed prompts) token ``j`` of
    sequence ``i`` goes to position ``starts[i] + j - offsets[i]`` of that
    sequence; without, there is one token a sequence (``t == b``) and it goes to
    position ``starts[i]``.  Tokens of no sequence, with a position outside the
    table or in no page are dropped.

    Two rows that share the page a token goes to write over each other
    (:func:`fork_sequences` leaves no such pages): which of them a slot ends
    up with is not defined.
    """
    _check_pool('write_pages', k_pages, v_pages, written=True)
    p, hk, _, d = k_pages.shape
    if k.ndim != 3 or v.ndim != 3 or k.shape[:2] != v.shape[:2] or k.shape[0] != hk or (
            k.shape[2] != d or v.shape[2] != v_pages.shape[3]):
        raise ValueError(
            f'write_pages: k and v must be ({hk}, t, {d}) and ({hk}, t, {v_pages.shape[3]}); '
            f'got {tuple(k.shape)} and {tuple(v.shape)}.'
        )
    if k.device != k_pages.device or v.device != k_pages.device:
        raise ValueError(
            f'write_pages: k, v are on {k.device}, {v.device}, the pages on {k_pages.device}.'
        )
    _check_table('write_pages', k.device, page_table, starts=(starts, (page_table.shape[0],)))
    b = page_table.shape[0]
    if offsets is not None:
        _check_ints('write_pages', k.device, offsets=(offsets, (b + 1,)))
    elif k.shape[1] != b:
        raise ValueError(
            f'write_pages: without offsets there is one token a sequence; got {k.shape[1]} '
            f'tokens for {b} sequences.'
        )
    _check_written('write_pages', k_pages, v_pages, k, v)
    args = (k_pages, v_pages, k, v, page_table, starts, offsets)
    if k.shape[1] == 0:
        return
    _dispatch(
        'write_pages', backend, k.device, lambda: _write_hip(*args),
        lambda: _reference_write(*args), (tuple(k.shape), tuple(k_pages.shape)), k.dtype,
    )


# ---------------------------------------------------------------------------
# Page management
# ---------------------------------------------------------------------------


def _counted(table, refs, sign):
    """``refs`` with ``sign`` added for every time ``table`` names a page."""
    e = table.reshape(-1).long()
    e = e[(e >= 0) & (e < refs.numel())]
    return refs.index_add(0, e, torch.full_like(e, sign, dtype=torch.int32))


def _handed_out(refs, need):
    """The k-th free page, lowest first, for the k-th True of ``need``; -1
    where they run out."""
    free = torch.nonzero(refs <= 0).reshape(-1).to(torch.int32)
    free = torch.cat((free, free.new_full((1,), -1)))
    rank = need.reshape(-1).long().cumsum(0).reshape(need.shape) - 1
    return torch.where(need, free[rank.clamp(0, free.numel() - 1)], -1)


def _reference_free(page_table, lengths, refs, rows):
    b = page_table.shape[0]
    rows = rows[(rows >= 0) & (rows < b)].long().unique()
    table, lengths = page_table.clone(), lengths.clone()
    refs = _counted(table[rows], refs, -1)
    table[rows] = -1
    lengths[rows] = 0
    return table, lengths, refs


def _reference_extend(page_table, lengths, refs, counts, page_size):
    m = page_table.shape[1]
    room = m * page_size
    length = lengths.long().clamp(0, room)
    grown = (length + counts.long().clamp(min=0)).clamp(max=room)
    col = torch.arange(m, device=refs.device)[None]
    reached = (col >= -(-length // page_size)[:, None]) & (col < -(-grown // page_size)[:, None])
    missing = reached & ((page_table < 0) | (page_table >= refs.numel()))
    page = _handed_out(refs, missing)
    short = missing & (page < 0)
    first = torch.where(short, col, m).amin(1)
    table = torch.where(missing, page, page_table)
    refs = torch.where(
        _counted(page, torch.zeros_like(refs), 1) > 0, torch.ones_like(refs), refs
    )
    return table, torch.minimum(grown, first * page_size).to(torch.int32), refs


def _reference_fork(k_pages, v_pages, page_table, lengths, refs, src, dst):
    b, m = page_table.shape
    p, ps = refs.numel(), k_pages.shape[2]
    table, out_len = page_table.clone(), lengths.clone()
    idx = torch.arange(src.numel(), device=src.device)
    ok = (src >= 0) & (src < b) & (dst >= 0) & (dst < b) & (src != dst)
    last = torch.full((b,), -1, dtype=torch.long, device=src.device)
    last.scatter_reduce_(0, dst[ok].long(), idx[ok], 'amax')
    ok = ok & (last[dst.clamp(0, b - 1).long()] == idx)
    src, dst = src[ok].long(), dst[ok].long()
    length = lengths[src].long().clamp(0, m * ps)
    full, rest = length // ps, length % ps
    last_page = page_table[src, full.clamp(max=m - 1)]
    fresh = _handed_out(refs, (rest > 0) & (last_page >= 0) & (last_page < p))
    got = fresh >= 0
    col = torch.arange(m, device=src.device)[None]
    rows = torch.where(col < full[:, None], page_table[src], -1)
    rows = torch.where((rows >= 0) & (rows < p), rows, -1)
    rows = torch.where((col == full[:, None]) & got[:, None], fresh[:, None], rows)
    out_refs = _counted(rows, _counted(page_table[dst], refs, -1), 1)
    slot = torch.arange(ps, device=src.device)[None] < rest[:, None]
    f, s = torch.nonzero(got[:, None] & slot, as_tuple=True)
    with torch.no_grad():
        for pages in (k_pages, v_pages):
            pages[fresh[f].long(), :, s] = pages[last_page[f].long(), :, s]
    table[dst] = rows
    out_len[dst] = torch.where((rest > 0) & ~got, full * ps, length).to(torch.int32)
    return table, out_len, out_refs


def _reference_compact(k_pages, v_pages, page_table, refs):
    live = refs > 0
    at = torch.arange(refs.numel(), device=refs.device)
    n = live.sum()
    movers = torch.nonzero(live & (at >= n)).reshape(-1)
    holes = torch.nonzero(~live & (at < n)).reshape(-1)
    with torch.no_grad():
        for pages in (k_pages, v_pages):
            pages[holes] = pages[movers]
    where = at.clone()
    where[movers] = holes
    out = refs.clamp(min=0)
    out[holes] = refs[movers]
    out[movers] = 0
    real = (page_table >= 0) & (page_table < refs.numel())
    moved = where[torch.where(real, page_table, 0).long()].to(torch.int32)
    return torch.where(real, moved, page_table), out


def _outputs(page_table, lengths, refs):
    return torch.empty_like(page_table), torch.empty_like(lengths), torch.empty_like(refs)


def free_sequences(
    page_table: torch.Tensor,
    lengths: torch.Tensor,
    refs: torch.Tensor,
    rows: torch.Tensor,
    *,
    backend: str = 'auto',
):
    """Ends the sequences in ``rows`` (int32 ``(n,)``): each of their table
    entries no longer counts, the rows become -1 and of length zero.  A row
    listed twice is freed once; numbers outside the table are ignored.  Returns
    the new ``(page_table, lengths, refs)``."""
    dev = page_table.device
    _check_table('free_sequences', dev, page_table, lengths=(lengths, page_table.shape[:1]),
                 refs=(refs, (None,)), rows=(rows, (None,)))
    _check_refs('free_sequences', refs)

    def fused():
        lib = _lib.lib()
        t, n, c, r = (x.contiguous() for x in (page_table, lengths, refs, rows))
        out = _outputs(t, n, c)
        _lib.check(
            lib.nxa_pages_free(
                t.shape[0], t.shape[1], c.numel(), t.data_ptr(), n.data_ptr(), c.data_ptr(),
                r.data_ptr(), r.numel(), *(x.data_ptr() for x in out), _stream(dev),
            )
        )
        return out

    return _dispatch('free_sequences', backend, dev, fused,
                     lambda: _reference_free(page_table, lengths, refs, rows),
                     (tuple(page_table.shape),), torch.int32)


def _check_refs(name, refs) -> None:
    if refs.numel() == 0:
        raise ValueError(f'{name}: refs must count the pages of a pool; got none.')


def extend_sequences(
    page_table: torch.Tensor,
    lengths: torch.Tensor,
    refs: torch.Tensor,
    counts: torch.Tensor,
    page_size: int,
    *,
    backend: str = 'auto',
):
    """Room for ``counts[i]`` (int32 ``(b,)``) more tokens in each sequence.

    Columns behind the row's last token that the new ones reach and that hold
    no page take free pages, the lowest first, in row and then column order; lengths grow by the counts
    (below zero: none; at most to the table's room).  Where the pages run out, a
    row's length ends with its last token that has a page.  Returns the new
    ``(page_table, lengths, refs)``; the tokens themselves are then written at
    the old lengths with :func:`write_pages`."""
    dev = page_table.device
    b = page_table.shape[:1]
    _check_table('extend_sequences', dev, page_table, lengths=(lengths, b), refs=(refs, (None,)),
                 counts=(counts, b))
    _check_refs('extend_sequences', refs)
    page_size = int(page_size)
    if not 1 <= page_size < 1 << 31:
        raise ValueError(f'extend_sequences: page_size must be positive; got {page_size}.')
    if page_table.shape[1] * page_size >= 1 << 31:
        raise ValueError('extend_sequences: a row has room for 2^31 tokens or more.')

    def fused():
        lib = _lib.lib()
        t, n, c, k = (x.contiguous() for x in (page_table, lengths, refs, counts))
        out = _outputs(t, n, c)
        ws = _workspace(4 * c.numel(), dev)
        _lib.check(
            lib.nxa_pages_extend(
                t.shape[0], t.shape[1], c.numel(), page_size, t.data_ptr(), n.data_ptr(),
                c.data_ptr(), k.data_ptr(), *(x.data_ptr() for x in out), ws.data_ptr(),
                ws.numel(), _stream(dev),
            )
        )
        return out

    return _dispatch('extend_sequences', backend, dev, fused,
                     lambda: _reference_extend(page_table, lengths, refs, counts, page_size),
                     (tuple(page_table.shape),), torch.int32)


def fork_sequences(
    k_pages: torch.Tensor,
    v_pages: torch.Tensor,
    page_table: torch.Tensor,
    lengths: torch.Tensor,
    refs: torch.Tensor,
    src: torch.Tensor,
    dst: torch.Tensor,
    *,
    backend: str = 'auto',
):
    """Makes row ``dst[i]`` a copy of row ``src[i]`` (int32 ``(n,)`` each), for
    beam search or several answers to one prompt.

    Whole pages are shared (their counts grow).  The tokens in a partly filled
    last page are copied, in place, to a free page (the lowest first, in order
    of ``i``), so that the two rows can grow apart; where none is left, or the
    source's tokens there are in no page, the new row ends with its whole
    pages.  The target's former pages no longer count for it, but are not
    handed out by the same call.  Sources are taken as they were before the
    call.  Of several pairs with one target the last counts; ``src[i] ==
    dst[i]`` and numbers outside the table are ignored.  Returns the new ``(page_table, lengths, refs)``."""
    _check_pool('fork_sequences', k_pages, v_pages, written=True)
    dev = page_table.device
    _check_table('fork_sequences', k_pages.device, page_table,
                 lengths=(lengths, page_table.shape[:1]), refs=(refs, k_pages.shape[:1]),
                 src=(src, (None,)), dst=(dst, src.shape[:1]))
    _check_written('fork_sequences', k_pages, v_pages)
    if page_table.shape[1] * k_pages.shape[2] >= 1 << 31:
        raise ValueError('fork_sequences: a row has room for 2^31 tokens or more.')

    def fused():
        _check_fused(k_pages, v_pages)
        lib = _lib.lib()
        desc = _pool_desc(k_pages, v_pages)
        t, n, c, s, d = (x.contiguous() for x in (page_table, lengths, refs, src, dst))
        out = _outputs(t, n, c)
        ws = _workspace(lib.nxa_pages_fork_workspace_bytes(t.shape[0], c.numel(), s.numel()), dev)
        _lib.check(
            lib.nxa_pages_fork(
                ctypes.byref(desc), k_pages.data_ptr(), v_pages.data_ptr(), t.shape[0],
                t.shape[1], t.data_ptr(), n.data_ptr(), c.data_ptr(), s.data_ptr(), d.data_ptr(),
                s.numel(), *(x.data_ptr() for x in out), ws.data_ptr(), ws.numel(), _stream(dev),
            )
        )
        _touched(k_pages, v_pages)
        return out

    return _dispatch(
        'fork_sequences', backend, dev, fused,
        lambda: _reference_fork(k_pages, v_pages, page_table, lengths, refs, src, dst),
        (tuple(k_pages.shape), tuple(page_table.shape)), k_pages.dtype,
    )


def compact_pages(
    k_pages: torch.Tensor,
    v_pages: torch.Tensor,
    page_table: torch.Tensor,
    refs: torch.Tensor,
    *,
    backend: str = 'auto',
):
    """Moves the ``n`` pages in use (``refs > 0``) to the pool's first ``n``.

    The k-th page in use from ``n`` on is copied, in place, to the k-th free
    page below ``n``; the other pages stay where they are, and what the movers
    leave behind is free but unchanged.  Returns the new ``(page_table, refs)``;
    entries that name no page, or a free one, stay as they are."""
    _check_pool('compact_pages', k_pages, v_pages, written=True)
    dev = page_table.device
    _check_table('compact_pages', k_pages.device, page_table, refs=(refs, k_pages.shape[:1]))
    _check_written('compact_pages', k_pages, v_pages)

    def fused():
        _check_fused(k_pages, v_pages)
        lib = _lib.lib()
        desc = _pool_desc(k_pages, v_pages)
        t, c = page_table.contiguous(), refs.contiguous()
        out = torch.empty_like(t), torch.empty_like(c)
        ws = _workspace(lib.nxa_pages_compact_workspace_bytes(c.numel()), dev)
        _lib.check(
            lib.nxa_pages_compact(
                ctypes.byref(desc), k_pages.data_ptr(), v_pages.data_ptr(), t.numel(),
                t.data_ptr(), c.data_ptr(), out[0].data_ptr(), out[1].data_ptr(), ws.data_ptr(),
                ws.numel(), _stream(dev),
            )
        )
        _touched(k_pages, v_pages)
        return out

    return _dispatch(
        'compact_pages', backend, dev, fused,
        lambda: _reference_compact(k_pages, v_pages, page_table, refs),
        (tuple(k_pages.shape), tuple(page_table.shape)), k_pages.dtype,
    )


def _page_list(arg, pages, limit) -> array.array:
    """A list or host tensor of page numbers as C ints."""
    if isinstance(pages, torch.Tensor):
        if pages.device.type != 'cpu':
            raise ValueError(f'copy_pages: {arg} must be on the host; it is on {pages.device}.')
        pages = pages.tolist()
    try:
        x = array.array('i', pages)
    except (TypeError, OverflowError) as exc:
        raise ValueError(f'copy_pages: {arg} must be a list of page numbers ({exc}).') from None
    if x and (min(x) < 0 or max(x) >= limit):
        raise ValueError(f'copy_pages: {arg} names pages outside the pool of {limit}.')
    return x


def copy_pages(
    k_pages: torch.Tensor,
    v_pages: torch.Tensor,
    src: Union[Sequence[int], torch.Tensor],
    dst: Union[Sequence[int], torch.Tensor],
    *,
    backend: str = 'auto',
) -> None:
    """Copies page ``src[i]`` to page ``dst[i]``, in place, for lists on the
    host (a program that keeps its own page lists has them there).

    No page may be a target twice, or both a target and a source
    (``ValueError``): every order of the copies then gives the same.  A
    captured graph replays the pages named at capture."""
    _check_pool('copy_pages', k_pages, v_pages, written=True)
    _check_written('copy_pages', k_pages, v_pages)
    s = _page_list('src', src, k_pages.shape[0])
    d = _page_list('dst', dst, k_pages.shape[0])
    if len(s) != len(d):
        raise ValueError(f'copy_pages: {len(s)} sources for {len(d)} targets.')
    targets = set(d)
    if len(targets) != len(d):
        raise ValueError('copy_pages: a page is the target of two copies.')
    if not targets.isdisjoint(s):
        raise ValueError('copy_pages: a page is both a source and a target.')
    if not s:
        return
    dev = k_pages.device

    def fused():
        _check_fused(k_pages, v_pages)
        desc = _pool_desc(k_pages, v_pages)
        _lib.check(
            _lib.lib().nxa_pages_copy(
                ctypes.byref(desc), k_pages.data_ptr(), v_pages.data_ptr(), s.buffer_info()[0],
                d.buffer_info()[0], len(s), _stream(dev),
            )
        )
        _touched(k_pages, v_pages)

    def reference():
        with torch.no_grad():
            for pages in (k_pages, v_pages):
                pages[torch.tensor(d, device=dev)] = pages[torch.tensor(s, device=dev)]

    _dispatch('copy_pages', backend, dev, fused, reference, (tuple(k_pages.shape),), k_pages.dtype)
