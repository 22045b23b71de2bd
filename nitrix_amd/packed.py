"""Attention over packed sequences, with grouped heads.

Sequences of different lengths laid end to end along one token axis, without
padding: what a prompt batch, packed training documents or the tokens of
differently sized volumes are.  :func:`packed_attention` stands next to
:func:`~nitrix_amd.attention.scaled_dot_product_attention` (the same heads
before tokens, the same dispatch over engines) for inputs that have no batch
axis; the reference has no counterpart.

* :func:`packed_attention` -- the public dispatcher;
* :func:`packed_attention_hip` -- the fused gfx950 engine, differentiable
  (``nxa_packed_fwd`` / ``nxa_packed_bwd``);
* :func:`reference_packed_attention` -- stock tensor ops, one sequence at a
  time (``backend='jax'``).
"""

from __future__ import annotations

import contextlib
import ctypes
from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from ._backend import NitrixBackendError, fallback, resolve_backend
from .attention import (
    _IO_DTYPES,
    _MAX_HEAD_DIM,
    HipNotTileable,
    _has_tangent,
    _no_tangent_back,
    _ptr,
    _row_stride_ok,
    default_scale,
    reference_scaled_dot_product_attention,
)

__all__ = [
    'packed_attention',
    'packed_attention_hip',
    'reference_packed_attention',
]


def _validate(q, k, v, offsets) -> None:
    if q.ndim != 3 or k.ndim != 3 or v.ndim != 3:
        raise ValueError(
            'packed_attention: q, k, v must be (h, t, d); got ndim '
            f'{q.ndim}, {k.ndim}, {v.ndim}.'
        )
    if q.shape[-1] != k.shape[-1]:
        raise ValueError(
            f'packed_attention: q/k head-dim mismatch (q d={q.shape[-1]}, k d={k.shape[-1]}).'
        )
    if not q.shape[1] == k.shape[1] == v.shape[1]:
        raise ValueError(
            'packed_attention: q, k, v must hold the same tokens; got '
            f't={q.shape[1]}, {k.shape[1]}, {v.shape[1]}.'
        )
    if k.shape[0] != v.shape[0] or k.shape[0] == 0 or q.shape[0] % k.shape[0] or q.shape[0] == 0:
        raise ValueError(
            'packed_attention: query heads must be a multiple of the key-value heads; got '
            f'{q.shape[0]} query, {k.shape[0]} key and {v.shape[0]} value heads.'
        )
    if offsets.ndim != 1 or offsets.dtype != torch.int32 or offsets.numel() < 2:
        raise ValueError(
            'packed_attention: offsets must be int32 of shape (sequences + 1,), at least one '
            f'sequence; got {offsets.dtype} of shape {tuple(offsets.shape)}.'
        )
    if not (q.device == k.device == v.device == offsets.device):
        raise ValueError(
            'packed_attention: q, k, v and offsets must be on one device; got '
            f'{q.device}, {k.device}, {v.device}, {offsets.device}.'
        )


def reference_packed_attention(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    offsets: torch.Tensor,
    *,
    scale: Optional[float] = None,
    causal: bool = False,
) -> torch.Tensor:
    """The unfused engine: :func:`reference_scaled_dot_product_attention` on
    each sequence, key-value heads repeated; rows of no sequence are zero.
    (Reads the offsets on the host, so it waits for the device.)"""
    if scale is None:
        scale = default_scale(q.shape[-1])
    t, g = q.shape[1], q.shape[0] // k.shape[0]
    dtype = torch.promote_types(torch.promote_types(q.dtype, k.dtype), v.dtype)
    ends = [min(max(x, 0), t) for x in offsets.tolist()]
    # (a sum of padded pieces, so that gradients reach every input even where
    # no row belongs to a sequence)
    pieces, at = [], 0
    for a, b in zip(ends[:-1], ends[1:]):
        if b <= a or a < at:
            continue
        if a > at:
            pieces.append(q.new_zeros(q.shape[0], a - at, v.shape[-1], dtype=dtype))
        ks = k[:, a:b].repeat_interleave(g, dim=0)
        vs = v[:, a:b].repeat_interleave(g, dim=0)
        pieces.append(
            reference_scaled_dot_product_attention(
                q[:, a:b], ks, vs, scale=scale, causal=causal
            )
        )
        at = b
    if at < t or not pieces:
        pieces.append(q.new_zeros(q.shape[0], t - at, v.shape[-1], dtype=dtype))
    out = torch.cat(pieces, dim=1)
    if not out.requires_grad and torch.is_grad_enabled():
        tied = [x for x in (q, k, v) if x.requires_grad]
        for x in tied:  # no sequence at all: zero gradients, not missing ones
            out = out + (x.reshape(-1)[:0].sum() * 0).to(dtype)
    return out


# ---------------------------------------------------------------------------
# Fused HIP engine
# ---------------------------------------------------------------------------


def _check_tileable(q, k, v) -> None:
    """Types and head dims the gfx950 kernels take: those of the dense
    attention (``attention._check_tileable``)."""
    if q.dtype not in _IO_DTYPES:
        raise HipNotTileable(
            f'fused packed attention supports bfloat16, float16 and float32; got {q.dtype}.'
        )
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise HipNotTileable(
            f'fused packed attention needs one dtype for q, k, v; got {q.dtype}, {k.dtype}, '
            f'{v.dtype}.'
        )
    if q.shape[1] >> 31:
        raise HipNotTileable(f'fused packed attention numbers rows in 31 bits; got t={q.shape[1]}.')
    epc = 16 // q.element_size()
    for name, n in (('d', q.shape[-1]), ('d_v', v.shape[-1])):
        if n > _MAX_HEAD_DIM or n % epc != 0 or n == 0:
            raise HipNotTileable(
                f'fused packed attention requires head dims <= {_MAX_HEAD_DIM} and multiples '
                f'of {epc}; got {name}={n}.'
            )


def _kernel_layout(x: torch.Tensor) -> torch.Tensor:
    """``x`` (h, t, d) itself where the kernels can read it in place, else a
    contiguous copy.  (``contiguous()`` would be no copy of a contiguous view
    off a 16-byte boundary, nor of one whose only odd stride is that of an
    axis of size one.)"""
    h_str, t_str, d_str = x.stride()
    epc = 16 // x.element_size()
    if (
        d_str == 1
        and h_str % epc == 0
        and t_str % epc == 0
        and x.data_ptr() % 16 == 0
        and _row_stride_ok(t_str, x.element_size())
    ):
        return x
    return x.clone(memory_format=torch.contiguous_format)


def _empty_like(x: torch.Tensor, d: int) -> torch.Tensor:
    """Uninitialised (h, t, d) in the memory order of ``x``: tokens before
    heads where a projection's output was viewed with heads first."""
    h, t, _ = x.shape
    if x.stride(0) < x.stride(1):
        return torch.empty((t, h, d), dtype=x.dtype, device=x.device).transpose(0, 1)
    return torch.empty((h, t, d), dtype=x.dtype, device=x.device)


_SAME_DEVICE = contextlib.nullcontext()
# (the public current_stream() builds a Stream object, 2 us of a call's 20)
_raw_stream = getattr(torch._C, '_cuda_getCurrentRawStream', None)


def _on(device: torch.device):
    """Context in which ``device`` is current, for launches on its streams."""
    if device.index == torch.cuda.current_device():
        return _SAME_DEVICE
    return torch.cuda.device(device)


def _stream(device: torch.device) -> int:
    if _raw_stream is None or device.index is None:
        return torch.cuda.current_stream(device).cuda_stream
    return _raw_stream(device.index)


def _desc(q, k, v, o, offsets, scale, causal) -> _lib.NxaPackedDesc:
    desc = _lib.NxaPackedDesc()
    desc.H, desc.T, desc.D = q.shape
    desc.Hk, desc.Dv = v.shape[0], v.shape[2]
    desc.nseq = offsets.numel() - 1
    desc.io_dtype = _IO_DTYPES[q.dtype]
    desc.causal = 1 if causal else 0
    desc.scale = scale
    desc.q_str[:] = q.stride()[:2]
    desc.k_str[:] = k.stride()[:2]
    desc.v_str[:] = v.stride()[:2]
    desc.o_str[:] = o.stride()[:2]
    return desc


def _forward(q, k, v, offsets, scale, causal, train):
    """The output and, for a backward, what the rounding of the output left
    (16-bit types), the log-sum-exp and the bytes of the backward's workspace."""
    o = _empty_like(q, v.shape[2])
    lse = o_lo = need = None
    if train:
        lse = torch.empty(q.shape[:2], dtype=torch.float32, device=q.device)
        if q.dtype != torch.float32:
            o_lo = _empty_like(q, v.shape[2])
    desc = _desc(q, k, v, o, offsets, scale, causal)
    lib = _lib.lib()
    if train:
        need = lib.nxa_packed_workspace_bytes(ctypes.byref(desc))
        if need == 0:
            raise HipNotTileable(lib.nxa_last_error().decode('utf-8', 'replace'))
    with _on(q.device):
        _lib.check(
            lib.nxa_packed_fwd(
                ctypes.byref(desc), q.data_ptr(), k.data_ptr(), v.data_ptr(),
                offsets.data_ptr(), o.data_ptr(), _ptr(o_lo), _ptr(lse),
                _stream(q.device),
            )
        )
    return o, o_lo, lse, need


class _PackedHip(torch.autograd.Function):
    """``(q, k, v, offsets) -> out``; the residuals are the inputs as the
    kernels read them, the output with its rounding, and the log-sum-exp, kept with
    ``save_for_backward`` (an in-place change between forward and backward
    raises); the backward is not itself differentiable."""

    @staticmethod
    def forward(ctx, q, k, v, offsets, scale, causal):
        kq, kk, kv = _kernel_layout(q), _kernel_layout(k), _kernel_layout(v)
        o, o_lo, lse, ctx.need = _forward(kq, kk, kv, offsets, scale, causal, True)
        ctx.args = (scale, causal)
        ctx.save_for_backward(kq, kk, kv, offsets, o, o_lo, lse)
        return o

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        q, k, v, offsets, o, o_lo, lse = ctx.saved_tensors
        _no_tangent_back('packed_attention', dout)
        dout = _kernel_layout(dout)
        dq, dk, dv = (_empty_like(x, x.shape[2]) for x in (q, k, v))
        desc = _desc(q, k, v, o, offsets, *ctx.args)
        lib = _lib.lib()
        ws = torch.empty(ctx.need, dtype=torch.uint8, device=q.device)
        strides = [_lib.I64x2(*x.stride()[:2]) for x in (dout, dq, dk, dv)]
        with _on(q.device):
            _lib.check(
                lib.nxa_packed_bwd(
                    ctypes.byref(desc), q.data_ptr(), k.data_ptr(), v.data_ptr(),
                    offsets.data_ptr(), o.data_ptr(), _ptr(o_lo), lse.data_ptr(), dout.data_ptr(),
                    strides[0], dq.data_ptr(), strides[1], dk.data_ptr(), strides[2],
                    dv.data_ptr(), strides[3], ws.data_ptr(), ws.numel(),
                    _stream(q.device),
                )
            )
        return dq, dk, dv, None, None, None


def packed_attention_hip(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    offsets: torch.Tensor,
    *,
    scale: float,
    causal: bool = False,
) -> torch.Tensor:
    """Fused packed attention on gfx950.  Raises :class:`HipNotTileable` for
    types and head dims outside the supported set and for forward-mode
    derivatives; differentiable in q, k and v."""
    _check_tileable(q, k, v)
    if _has_tangent(q, k, v):
        raise HipNotTileable('fused packed attention has no forward-mode derivative.')
    _lib.lib()  # a missing library is an error here, not a fallback
    offsets = offsets.contiguous()
    scale, causal = float(scale), bool(causal)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        return _PackedHip.apply(q, k, v, offsets, scale, causal)
    return _forward(
        _kernel_layout(q), _kernel_layout(k), _kernel_layout(v), offsets, scale, causal, False
    )[0]


def packed_attention(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    offsets: torch.Tensor,
    *,
    scale: Optional[float] = None,
    causal: bool = False,
    backend: str = 'auto',
) -> torch.Tensor:
    """Attention inside each of several sequences packed along one token axis.

    q ``(h, t, d)``, k ``(h_kv, t, d)``, v ``(h_kv, t, d_v)``, any strides
    (a projection's ``(t, h, d)`` output transposed is read in place); ``h``
    a multiple of ``h_kv``: query head ``i`` reads key-value head
    ``i // (h / h_kv)``.  ``offsets`` int32 ``(sequences + 1,)`` on the same
    device, non-decreasing within ``0 .. t``: sequence ``s`` is tokens
    ``offsets[s] .. offsets[s + 1] - 1`` and may be empty.  The result
    ``(h, t, d_v)`` is ``softmax(scale * q k^T) v`` over the keys of a
    query's own sequence, with ``causal`` those up to the query itself;
    ``scale`` defaults to ``1/sqrt(d)``.  Tokens of no sequence (before
    ``offsets[0]``, from ``offsets[-1]`` on) give zero, take no part in
    anything and get zero gradients, whatever they hold; a NaN or infinity
    inside a sequence stays in that sequence.  Differentiable
    in q, k and v; gradients of k and v are summed over the heads that share
    them.

    ``backend`` as in :func:`scaled_dot_product_attention`; forward-mode
    derivatives are left to the reference engine.  The fused engine
    never reads the offsets on the host: a captured graph may be replayed
    with other offsets (and lengths) in the same tensor.  Capture forward and
    backward together, with no eager graph of the same leaves alive: torch ties
    a leaf's accumulation to the stream of the first graph that uses it.
    """
    _validate(q, k, v, offsets)
    resolved_scale = default_scale(q.shape[-1]) if scale is None else scale
    resolved = resolve_backend(backend, q.device)
    if resolved == 'hip' and q.shape[1] > 0:
        try:
            return packed_attention_hip(q, k, v, offsets, scale=resolved_scale, causal=causal)
        except (HipNotTileable, _lib.NxaShapeError) as exc:
            fallback(
                function='packed_attention',
                requested='hip',
                resolved='jax',
                reason=f'the fused packed-attention kernel does not support this input ({exc})',
                shapes=(tuple(q.shape), tuple(k.shape), tuple(v.shape)),
                dtype=q.dtype,
            )
        except _lib.HipLibraryMissing as exc:
            raise NitrixBackendError(str(exc)) from exc
    return reference_packed_attention(q, k, v, offsets, scale=resolved_scale, causal=causal)
