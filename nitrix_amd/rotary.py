"""Rotary positions of queries and keys.

What tells attention where a token stands: pairs of a query's or key's elements
turned by an angle that grows with the position.  :func:`rotary_embed` takes
queries and keys heads first, as :func:`~nitrix_amd.packed.packed_attention`
and :func:`~nitrix_amd.attention.scaled_dot_product_attention` do, or those of
one new token a sequence (``(h, b, d)``, transposed views of what
:func:`~nitrix_amd.paged.paged_attention` reads), and the position of each token.
The reference has no counterpart.

* :func:`rotary_embed` -- the public dispatcher (``nxa_rotary``), differentiable;
* :func:`rotary_frequencies` -- the angle a position of each pair, plain or for
  contexts longer than the model was trained on;
* :func:`packed_positions` -- the positions of packed sequences' tokens;
* :func:`reference_rotary_embed` -- stock tensor ops (``backend='jax'``).
"""

from __future__ import annotations

import ctypes
import math
from typing import Optional

import torch

from . import _lib
from ._backend import NitrixBackendError, fallback, resolve_backend
from .attention import _IO_DTYPES, HipNotTileable, _has_tangent, _no_tangent_back
from .packed import _on, _stream

__all__ = [
    'packed_positions',
    'reference_rotary_embed',
    'rotary_embed',
    'rotary_frequencies',
]

_MAX_ROTARY_DIM = 256


def rotary_frequencies(
    dims: int,
    *,
    base: float = 10000.0,
    scaling: str = 'none',
    factor: float = 1.0,
    original_length: Optional[int] = None,
    fast_turns: float = 32.0,
    slow_turns: float = 1.0,
    device=None,
) -> torch.Tensor:
    """Radians a position of each pair of ``dims`` rotated elements, float64
    ``(dims / 2,)``: ``w_i = base ** (-2 i / dims)``, and for a context ``factor``
    times as long as the one of ``original_length`` tokens trained on, by
    ``scaling``:

    * ``'none'`` -- as it is;
    * ``'linear'`` -- ``w_i / factor``: positions interpolated;
    * ``'base'`` -- the base raised to ``base * factor ** (dims / (dims - 2))``: the
      slowest pair interpolates, the fastest stays (``dims`` of at least 4);
    * ``'ramp'`` -- pairs that turn ``fast_turns`` times or more in
      ``original_length`` stay, those of ``slow_turns`` or fewer are divided by the
      factor, with a ramp linear in the pair's number between (YaRN);
    * ``'bands'`` -- the same ends, with a ramp linear in the number of turns.

    Where attention of a longer context is sharpened as well (YaRN's ``0.1
    ln(factor) + 1``), that is :func:`rotary_embed`'s ``scale``.
    """
    if dims <= 0 or dims % 2:
        raise ValueError(f'rotary_frequencies: dims must be a positive even number; got {dims}.')
    if not base > 0 or not factor > 0:
        raise ValueError(
            f'rotary_frequencies: base and factor must be positive; got {base}, {factor}.'
        )
    i = torch.arange(dims // 2, dtype=torch.float64)
    if scaling == 'base':
        if dims < 4:
            raise ValueError("rotary_frequencies: scaling='base' needs at least 4 dims.")
        base = base * factor ** (dims / (dims - 2))
    w = base ** (-2.0 * i / dims)
    if scaling == 'linear':
        w = w / factor
    elif scaling in ('ramp', 'bands'):
        if original_length is None or original_length <= 0:
            raise ValueError(f'rotary_frequencies: scaling={scaling!r} needs an original_length.')
        if not fast_turns > slow_turns > 0:
            raise ValueError(
                'rotary_frequencies: fast_turns must exceed slow_turns, both positive; got '
                f'{fast_turns}, {slow_turns}.'
            )
        if scaling == 'ramp':
            if not base > 1:
                raise ValueError("rotary_frequencies: scaling='ramp' needs a base above 1.")
            lo, hi = (
                dims * math.log(original_length / (2 * math.pi * t)) / (2 * math.log(base))
                for t in (fast_turns, slow_turns)
            )
            lo, hi = max(math.floor(lo), 0), min(math.ceil(hi), dims - 1)
            # (no pair turns even slow_turns times: all are divided)
            slow = torch.ones_like(i) if hi <= 0 else ((i - lo) / max(hi - lo, 0.001)).clamp(0, 1)
        else:
            turns = original_length * w / (2 * math.pi)
            slow = ((fast_turns - turns) / (fast_turns - slow_turns)).clamp(0, 1)
        w = w * (1 - slow) + w / factor * slow
    elif scaling not in ('none', 'base'):
        raise ValueError(
            "rotary_frequencies: scaling must be 'none', 'linear', 'base', 'ramp' or 'bands'; "
            f'got {scaling!r}.'
        )
    return w.to(device) if device is not None else w


def packed_positions(
    offsets: torch.Tensor, t: int, starts: Optional[torch.Tensor] = None
) -> torch.Tensor:
    """Positions int32 ``(t,)`` of packed tokens: token ``j`` of sequence ``i``
    (``offsets`` int32 ``(sequences + 1,)`` as in
    :func:`~nitrix_amd.packed.packed_attention`) stands at ``starts[i] + j -
    offsets[i]`` (``starts`` int32 ``(sequences,)``, zeros if None, as in
    :func:`~nitrix_amd.paged.write_pages`); tokens of no sequence at 0."""
    if offsets.ndim != 1 or offsets.dtype != torch.int32 or offsets.numel() < 2:
        raise ValueError(
            'packed_positions: offsets must be int32 of shape (sequences + 1,), at least one '
            f'sequence; got {offsets.dtype} of shape {tuple(offsets.shape)}.'
        )
    n = offsets.numel() - 1
    if starts is not None and (starts.shape != (n,) or starts.dtype != torch.int32):
        raise ValueError(
            f'packed_positions: starts must be int32 of shape ({n},); got {starts.dtype} of '
            f'shape {tuple(starts.shape)}.'
        )
    if starts is not None and starts.device != offsets.device:
        raise ValueError(
            f'packed_positions: starts is on {starts.device}, offsets on {offsets.device}.'
        )
    if t < 0:
        raise ValueError(f'packed_positions: t must not be negative; got {t}.')
    token = torch.arange(t, dtype=torch.int32, device=offsets.device)
    seq = torch.searchsorted(offsets, token, right=True, out_int32=True) - 1
    ok = (seq >= 0) & (seq < n)
    seq = seq.clamp(0, n - 1)
    at = token - offsets[seq]
    if starts is not None:
        at = at + starts[seq]
    return torch.where(ok, at, 0)


def _validate(q, k, positions, frequencies) -> None:
    qs = q.shape
    if len(qs) < 3:
        raise ValueError(f'rotary_embed: q must be (..., h, t, d); got ndim {q.ndim}.')
    if not q.dtype.is_floating_point:
        raise ValueError(f'rotary_embed: q must be floating-point; got {q.dtype}.')
    if k is not None:
        ks = k.shape
        if len(ks) != len(qs) or ks[-2:] != qs[-2:] or ks[:-3] != qs[:-3]:
            raise ValueError(
                'rotary_embed: q and k must agree in all but their heads; got '
                f'{tuple(qs)} and {tuple(ks)}.'
            )
        if k.dtype != q.dtype:
            raise ValueError(
                f'rotary_embed: q and k must share a dtype; got {q.dtype} and {k.dtype}.'
            )
    if frequencies.ndim != 1 or not frequencies.dtype.is_floating_point or not (
            1 <= frequencies.shape[0] <= qs[-1] // 2):
        raise ValueError(
            f'rotary_embed: frequencies must be floating-point of shape (r / 2,) with r up to '
            f'd={qs[-1]}; got {frequencies.dtype} of shape {tuple(frequencies.shape)}.'
        )
    if positions.dtype != torch.int32 and positions.dtype != torch.int64:
        raise ValueError(f'rotary_embed: positions must be int32 or int64; got {positions.dtype}.')
    ps = positions.shape
    # (broadcast: axes from the last on, each as long as q's or 1; every token its own)
    if not 1 <= len(ps) <= len(qs) - 2 or ps[-1] != qs[-2] or any(
        n != 1 and n != m for n, m in zip(ps[-2::-1], qs[-4::-1])
    ):
        raise ValueError(
            f'rotary_embed: positions must broadcast to {(*qs[:-3], qs[-2])} with one for each '
            f'token; got {tuple(ps)}.'
        )
    device = q.device
    if not positions.device == frequencies.device == device or (
            k is not None and k.device != device):
        for name, x in (('k', k), ('positions', positions), ('frequencies', frequencies)):
            if x is not None and x.device != device:
                raise ValueError(f'rotary_embed: {name} is on {x.device}, q on {device}.')
    if frequencies.requires_grad and torch.is_grad_enabled():
        raise ValueError('rotary_embed is not differentiable in the frequencies; detach them.')


def reference_rotary_embed(q, k, positions, frequencies, *, interleaved=False, scale=1.0):
    """The unfused engine: angles in float64, the rotation in at least
    float32."""
    acc = torch.promote_types(q.dtype, torch.float32)
    angle = positions.double()[..., None, :, None] * frequencies.double()
    cos, sin = (angle.cos() * scale).to(acc), (angle.sin() * scale).to(acc)
    n = frequencies.shape[0]

    def turn(x):
        y = x[..., :2 * n].to(acc)
        a, b = (y[..., 0::2], y[..., 1::2]) if interleaved else (y[..., :n], y[..., n:])
        a, b = a * cos - b * sin, b * cos + a * sin
        y = torch.stack((a, b), -1).flatten(-2) if interleaved else torch.cat((a, b), -1)
        return torch.cat((y.to(x.dtype), x[..., 2 * n:]), -1)

    return turn(q), None if k is None else turn(k)


# ---------------------------------------------------------------------------
# Fused HIP engine
# ---------------------------------------------------------------------------


def _rows(x: torch.Tensor):
    """``x`` (h, t, d) or (b, h, t, d) with unit stride over d, its strides (batch,
    head, token), and an uninitialised tensor of its shape in its memory order:
    tokens before heads where a projection's output was viewed with heads first."""
    if x.stride(-1) != 1:
        x = x.contiguous()
    str_ = x.stride()
    *lead, h, t, d = x.shape
    if str_[-3] < str_[-2]:
        out = torch.empty((*lead, t, h, d), dtype=x.dtype, device=x.device).transpose(-3, -2)
    else:
        out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    if lead:
        return x, _lib.I64x3(*str_[:3]), out, _lib.I64x3(*out.stride()[:3])
    out_str = out.stride()
    return (x, _lib.I64x3(0, str_[0], str_[1]), out, _lib.I64x3(0, out_str[0], out_str[1]))


_NO_STRIDES = _lib.I64x3(0, 0, 0)


def _turn(q, k, positions, frequencies, interleaved, scale, inverse):
    """The fused kernel on (h, t, d) or (b, h, t, d) rows, k None or of the same
    b, t, d; positions of the batch and token axes."""
    q, q_str, q_out, q_out_str = _rows(q)
    k_out, hk, k_str, k_out_str = None, 0, _NO_STRIDES, _NO_STRIDES
    if k is not None:
        k, k_str, k_out, k_out_str = _rows(k)
        hk = k.shape[-3]
    *lead, h, t, d = q.shape
    pos_str = positions.stride()
    desc = _lib.NxaRotaryDesc(
        lead[0] if lead else 1, t, h, hk, d, 2 * frequencies.shape[0], _IO_DTYPES[q.dtype],
        interleaved, inverse, positions.dtype == torch.int64, scale,
        _lib.I64x2(pos_str[0] if lead else 0, pos_str[-1]), q_str, k_str, q_out_str, k_out_str,
    )
    with _on(q.device):
        _lib.check(
            _lib.lib().nxa_rotary(
                ctypes.byref(desc), q.data_ptr(), None if k is None else k.data_ptr(),
                positions.data_ptr(), frequencies.data_ptr(), q_out.data_ptr(),
                None if k is None else k_out.data_ptr(), _stream(q.device),
            )
        )
    return q_out, k_out


class _RotaryHip(torch.autograd.Function):
    """``(q, k) -> (q', k')``.  Linear, so the backward is the same turned the
    other way round, and is itself differentiable."""

    @staticmethod
    def forward(ctx, q, k, positions, frequencies, interleaved, scale, inverse):
        ctx.set_materialize_grads(False)
        ctx.args = (interleaved, scale, not inverse)
        ctx.save_for_backward(positions, frequencies)
        out = _turn(q, k, positions, frequencies, interleaved, scale, inverse)
        # (keys of a frozen projection beside queries that are trained)
        ctx.mark_non_differentiable(*(
            y for y, need in zip(out, ctx.needs_input_grad) if y is not None and not need
        ))
        return out

    @staticmethod
    def backward(ctx, dq, dk):
        args = (*ctx.saved_tensors, *ctx.args)
        if not ctx.needs_input_grad[0]:
            dq = None
        if not ctx.needs_input_grad[1]:
            dk = None
        for x in (dq, dk):
            if x is not None:
                _no_tangent_back('rotary_embed', x)
        # (a graph of the gradients themselves where one is asked for)
        turn = _RotaryHip.apply if torch.is_grad_enabled() else _turn
        if dq is not None:
            dq, dk = turn(dq, dk, *args)
        elif dk is not None:
            dk, _ = turn(dk, None, *args)
        return dq, dk, None, None, None, None, None


def _rotary_hip(q, k, positions, frequencies, interleaved, scale):
    if q.dtype not in _IO_DTYPES:
        raise HipNotTileable(
            f'fused rotary positions support bfloat16, float16 and float32; got {q.dtype}.'
        )
    shape = q.shape
    if shape[-1] > _MAX_ROTARY_DIM:
        raise HipNotTileable(
            f'fused rotary positions take head dims up to {_MAX_ROTARY_DIM}; got {shape[-1]}.'
        )
    if q.numel() >> 31 and max(math.prod(shape[:-3]), *shape[-3:]) >> 31 or (
            k is not None and k.shape[-3] >> 31):
        raise HipNotTileable('fused rotary positions number sequences, heads and tokens in 31 bits.')
    if _has_tangent(q, k):
        raise HipNotTileable('fused rotary positions have no forward-mode derivative.')
    _lib.lib()  # a missing library is an error here, not a fallback
    ndim = len(shape)
    if ndim > 3:
        positions = positions.expand(*shape[:-3], shape[-2])
    elif positions.ndim != 1:
        positions = positions.reshape(-1)
    k_shape = None if k is None else k.shape
    if ndim > 4:
        q = q.reshape(-1, *shape[-3:])
        k = None if k is None else k.reshape(-1, *k_shape[-3:])
        positions = positions.reshape(-1, shape[-2])
    if frequencies.dtype != torch.float64 or not frequencies.is_contiguous():
        frequencies = frequencies.double().contiguous()
    args = (positions, frequencies, bool(interleaved), float(scale), False)
    if torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)):
        q, k = _RotaryHip.apply(q, k, *args)
    else:
        q, k = _turn(q, k, *args)
    if ndim > 4:
        q = q.reshape(shape)
        k = None if k is None else k.reshape(k_shape)
    return q, k


def rotary_embed(
    q: torch.Tensor,
    k: Optional[torch.Tensor],
    positions: torch.Tensor,
    frequencies: torch.Tensor,
    *,
    interleaved: bool = False,
    scale: float = 1.0,
    backend: str = 'auto',
):
    """Queries and keys turned by their tokens' positions.

    q ``(..., h, t, d)`` and k ``(..., h_kv, t, d)`` (or None) of one dtype, any
    strides; ``positions`` int32 or int64, one a token, broadcast to ``(..., t)``
    (:func:`packed_positions` for packed sequences; for one new token a sequence,
    its length before it), negative ones too; ``frequencies``
    :func:`rotary_frequencies` of the ``r`` elements to rotate, ``r <= d``, kept on
    the same device (float64; others are cast by every call).  Pair ``i`` of a
    row, elements ``i`` and ``i + r / 2``, or ``2 i`` and ``2 i + 1`` with
    ``interleaved``, turns by ``position * frequencies[i]`` and is multiplied by
    ``scale``; elements from ``r`` on are copied.  Returns ``(q', k')`` (None for
    None).

    Angles are formed in float64 (off by 2^-53 of themselves in the reference engine,
    by less than a float32's last place in the fused one up to positions of 2^53), the
    rotation in float32 (float64 inputs, which the reference engine takes: float64) and
    rounded once.  Differentiable in q and
    k, any number of times; forward-mode derivatives are left to the reference
    engine.  The fused engine takes bfloat16, float16 and float32 and head dims up
    to 256; ``d`` and ``r`` (half layout: ``r / 2``) in whole 16-byte chunks are
    fastest.  Positions and frequencies are never read on the host: a captured
    graph may be replayed with others in the same tensors.  Capture forward and
    backward together, with no eager graph of the same leaves alive.
    """
    _validate(q, k, positions, frequencies)
    if resolve_backend(backend, q.device) == 'hip' and q.numel() > 0 and (
            k is None or k.numel() > 0):
        try:
            return _rotary_hip(q, k, positions, frequencies, interleaved, scale)
        except (HipNotTileable, _lib.NxaShapeError) as exc:
            fallback(
                function='rotary_embed',
                requested='hip',
                resolved='jax',
                reason=f'the fused kernel does not support this input ({exc})',
                shapes=(tuple(q.shape), None if k is None else tuple(k.shape)),
                dtype=q.dtype,
            )
        except _lib.HipLibraryMissing as exc:
            raise NitrixBackendError(str(exc)) from exc
    return reference_rotary_embed(
        q, k, positions, frequencies, interleaved=interleaved, scale=scale
    )
