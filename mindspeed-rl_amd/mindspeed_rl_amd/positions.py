"""Rotary positions of queries and keys: the position ids that :func:`preprocess_packed_seqs` hands out (or a batch's, or those of
single tokens) turn pairs of entries of every head.  The reference leaves them to the model below it.
"""
import array
import ctypes
import math

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .vocab_ops import _transformed

_CODES = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}
_INTS = {torch.int64: _lib.I64, torch.int32: _lib.I32}


class RotarySide(ctypes.Structure):
    """struct mrl_rotary_side"""
    _fields_ = [("x", ctypes.c_void_p), ("out", ctypes.c_void_p)] + [
        (name, ctypes.c_int64) for name in ("heads", "dim", "start", "stride_outer", "stride_inner", "stride_head")]


def _turn(xs, positions, inv_freq, interleaved, start, scale, back):
    """The turned tensors of `xs`, dense."""
    words, outs, kept = [], [], []
    for x in xs:
        strides = x.stride()
        if strides[-1] != 1:
            x = x.contiguous()
            kept.append(x)                  # until the launch: the next copy may not take its memory
            strides = x.stride()
        shape = x.shape
        out = x.new_empty(shape)
        outs.append(out)
        dim = shape[-1]
        words += (x.data_ptr(), out.data_ptr(), shape[-2], dim, start if start >= 0 else dim + start)
        words += strides[:3] if len(shape) == 4 else (0, strides[0], strides[1])
    pos = positions.stride()
    if len(shape) == 4:
        n_outer, n_inner, pos_outer, pos_inner = shape[0], shape[1], pos[0], pos[1]
    else:
        n_outer, n_inner, pos_outer, pos_inner = 1, shape[0], 0, pos[0]
    sides = array.array("q", words)         # struct mrl_rotary_side, one or two
    at = sides.buffer_info()[0]
    _lib.call("mrl_rotary", at, at + 64 if len(outs) > 1 else None, _CODES[out.dtype], positions.data_ptr(), _INTS[positions.dtype],
              pos_outer, pos_inner, n_outer, n_inner, inv_freq.data_ptr(), 2 * inv_freq.shape[0], interleaved, scale, back,
              _lib.stream(out.device))
    return outs


def _rotary_backward(ctx, dq, dk):
    positions, inv_freq = ctx.saved_tensors
    need = ctx.needs_input_grad
    q, k = need[0] and dq is not None, need[1] and dk is not None
    outs = iter(_turn([g for g, wanted in ((dq, q), (dk, k)) if wanted], positions, inv_freq, *ctx.meta, True) if q or k else ())
    return next(outs) if q else None, next(outs) if k else None, None, None, None, None, None


_rotary_backward_once = once_differentiable(_rotary_backward)


class _Rotary(torch.autograd.Function):
    """(q, k or None) -> the same turned; the backward turns the gradients back."""

    @staticmethod
    def forward(ctx, q, k, positions, inv_freq, interleaved, start, scale):
        ctx.save_for_backward(positions, inv_freq)
        ctx.meta = (interleaved, start, scale)
        ctx.set_materialize_grads(False)
        if k is None:
            return _turn([q], positions, inv_freq, interleaved, start, scale, False)[0], None
        return tuple(_turn([q, k], positions, inv_freq, interleaved, start, scale, False))

    @staticmethod
    def backward(ctx, dq, dk):
        return _rotary_backward_once(ctx, dq, dk) if torch.is_grad_enabled() else _rotary_backward(ctx, dq, dk)


def rotary(q, k, position_ids, inv_freq, interleaved=False, start=0, scale=1.0):
    """``(q, k)`` turned by their positions: a pair of entries ``(a, b)`` of every head becomes ``scale * (a cos t - b sin t, b cos t + a sin
    t)`` with ``t = position * inv_freq[i]``.

    ``q`` and ``k``: ``[tokens, heads, dim]`` (packed) or ``[batch, tokens, heads, dim]``, fp32, bf16 or fp16, of any strides (views of one
    projection's output); heads and ``dim`` may differ between them, and ``k`` may be None.  ``position_ids``: integers, ``[tokens]`` or ``[1,
    tokens]``, or ``[batch, tokens]``.  ``inv_freq``: ``[part / 2]``, fp64 (:func:`rotary_frequencies`) or fp32; the angle is formed in 64
    bits.  ``part`` entries of a head from ``start`` on (from its end, if negative) are turned, entries ``i`` and ``i + part / 2`` of them
    or, with ``interleaved``, ``2 i`` and ``2 i + 1``; the others are copied.  Results are dense; entries are turned in fp32 and rounded once.
    Differentiable (once) with respect to ``q`` and ``k``."""
    dtype, lead = q.dtype, q.shape[:-2]
    part = 2 * inv_freq.numel()
    start, scale = int(start), float(scale)
    if inv_freq.dim() != 1 or part < 2 or inv_freq.dtype not in (torch.float64, torch.float32):
        raise TypeError("inv_freq must be float64 or float32 of one dimension, not %s %s" % (inv_freq.dtype, tuple(inv_freq.shape)))
    for name, x in (("q", q), ("k", k)) if k is not None else (("q", q),):
        shape = x.shape
        if dtype not in _CODES or x.dtype is not dtype:
            raise TypeError("%s must be float32, bfloat16 or float16, and of one type with q: %s" % (name, x.dtype))
        if len(shape) not in (3, 4) or shape[:-2] != lead or shape[-2] < 1:
            raise ValueError("%s must be [tokens, heads, dim] or [batch, tokens, heads, dim], of one batch with q: %s and %s"
                             % (name, tuple(shape), tuple(q.shape)))
        begin = start if start >= 0 else shape[-1] + start
        if begin < 0 or begin + part > shape[-1]:
            raise ValueError("%s: %d entries from %d on are not in a head of %d" % (name, part, start, shape[-1]))
    if not math.isfinite(scale):
        raise ValueError("scale must be finite, not %r" % scale)
    if position_ids.dtype not in _INTS:
        raise TypeError("position_ids must be int64 or int32, not %s" % position_ids.dtype)
    if position_ids.shape != lead:
        if position_ids.dim() == 2 and len(lead) == 1 and position_ids.shape[0] == 1:
            position_ids = position_ids[0]
        if position_ids.dim() not in (1, len(lead)) or position_ids.shape[-1] != lead[-1] or (
                position_ids.dim() == 2 and position_ids.shape[0] not in (1, lead[0])):
            raise ValueError("position_ids must be [tokens] or [batch, tokens] of q: %s and %s" % (tuple(position_ids.shape), tuple(q.shape)))
        position_ids = position_ids.expand(lead)
    _lib.require_device(q, k, position_ids, inv_freq)
    if inv_freq.requires_grad:
        raise ValueError("inv_freq is not differentiable here: detach it")
    if inv_freq.dtype is not torch.float64 or not inv_freq.is_contiguous():
        inv_freq = inv_freq.to(torch.float64).contiguous()
    interleaved = bool(interleaved)
    if torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)) or _transformed():
        return _Rotary.apply(q, k, position_ids, inv_freq, interleaved, start, scale)
    outs = _turn([q] if k is None else [q, k], position_ids, inv_freq, interleaved, start, scale, False)
    return (outs[0], outs[1] if k is not None else None)


def rotary_frequencies(part, base=10000.0, scaling=None, factor=1.0, trained=None, fast=None, slow=1.0, device=None):
    """``(inv_freq, scale)`` for :func:`rotary`: ``base^(-2 i / part)``, ``i < part / 2``, in fp64, for contexts ``factor`` times as long as the
    ``trained`` positions (``scaling``):

    * None: as they are, ``scale`` 1
    * "linear": all divided by ``factor``
    * "yarn": those that turn more than ``fast`` times within the ``trained`` positions stay, those that turn less than ``slow`` times are divided by
      ``factor``, in between (by index) a share of both; ``scale`` is ``0.1 ln(factor) + 1``
    * "bands": the same with the share in between by the number of turns, and ``scale`` 1

    ``fast`` is 32 for "yarn" and 4 for "bands" unless it is given, as the models that use them have it.
    """
    part = int(part)
    if part < 2 or part % 2:
        raise ValueError("part must be an even number from 2 on, not %r" % part)
    if not base > 1.0 or not factor >= 1.0:
        raise ValueError("base must be above 1 and factor at least 1, not %r and %r" % (base, factor))
    own = float(base) ** (-torch.arange(0, part, 2, dtype=torch.float64) / part)
    scale = 1.0
    if scaling is None:
        inv_freq = own
    elif scaling == "linear":
        inv_freq = own / factor
    elif scaling in ("yarn", "bands"):
        fast = (32.0 if scaling == "yarn" else 4.0) if fast is None else fast
        if trained is None or not trained > 0 or not fast > slow > 0:
            raise ValueError("scaling %r needs trained positions and fast > slow > 0: %r, %r, %r" % (scaling, trained, fast, slow))
        if scaling == "yarn":
            # where a pair turns so many times within the trained positions, as a fraction of an index
            place = [part * math.log(trained / (n * 2 * math.pi)) / (2 * math.log(base)) for n in (fast, slow)]
            lo, hi = max(math.floor(place[0]), 0), min(math.ceil(place[1]), part - 1)
            kept = 1 - ((torch.arange(part // 2, dtype=torch.float64) - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
            scale = 0.1 * math.log(factor) + 1.0
        else:
            kept = ((trained * own / (2 * math.pi) - slow) / (fast - slow)).clamp(0, 1)
        inv_freq = own * kept + own / factor * (1 - kept)
    else:
        raise ValueError("scaling must be None, 'linear', 'yarn' or 'bands', not %r" % (scaling,))
    return inv_freq.to(device), scale
