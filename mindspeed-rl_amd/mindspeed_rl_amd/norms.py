"""Layer norm and RMS norm of hidden states, forward and backward: what a model's last stage does to the hidden states
that :func:`lmhead_logprob` and the loss objects with ``lm_head_weight=`` take.

The reference leaves them to the model below it; the loss objects call them with ``final_norm_weight=``.
"""
import functools

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .vocab_ops import _flat_rows, _transformed

_FLOATS = (torch.float32, torch.bfloat16, torch.float16)


@functools.lru_cache(maxsize=256)
def _workspace_bytes(n_rows, hidden):
    """mrl_norm_bwd_workspace_bytes: a function of its arguments alone."""
    return _lib.load().mrl_norm_bwd_workspace_bytes(n_rows, hidden)


def _forward(x, weight, bias, eps, layer, keep):
    """y, and what the backward takes if `keep`: the rows, their stride, the weight, [mean and] rstd of the rows."""
    dev, hidden = x.device, x.shape[-1]
    if x.is_contiguous():
        flat, n_rows, x_stride, y = x, x.numel() // hidden, hidden, torch.empty_like(x)
    else:
        flat, x_stride = _flat_rows(x)
        n_rows, y = flat.shape[0], torch.empty(x.shape, dtype=x.dtype, device=dev)
    w, b = weight.contiguous(), None if bias is None else bias.contiguous()
    stats = p_mean = p_rstd = None
    if keep:
        stats = weight.new_empty((2 if layer else 1, n_rows), dtype=torch.float32)
        p_rstd = stats.data_ptr()
        p_mean = p_rstd + 4 * n_rows if layer else None
    _lib.call("mrl_norm_fwd", flat.data_ptr(), _lib.dtype_code(x), n_rows, hidden, x_stride, w.data_ptr(), _lib.ptr(b),
              _lib.dtype_code(w), 1 if layer else 0, eps, y.data_ptr(), p_mean, p_rstd, _lib.stream(dev))
    return y, flat, x_stride, w, stats


def _backward(ctx, dy):
    flat, w, stats = ctx.saved_tensors
    shape, n_rows, hidden, x_stride, layer = ctx.meta
    dev = flat.device
    if dy.is_contiguous():
        dy_stride = hidden
    else:
        dy, dy_stride = _flat_rows(dy)
    need_x, need_w, need_b = ctx.needs_input_grad[:3]
    dx = dw = db = workspace = None
    if need_x:
        dx = torch.empty_like(flat) if flat.is_contiguous() and flat.shape == shape else torch.empty(shape, dtype=flat.dtype, device=dev)
    ws_bytes = 0
    if need_w or need_b:
        dw = torch.empty_like(w) if need_w else None
        db = torch.empty_like(w) if need_b else None
        ws_bytes = _workspace_bytes(n_rows, hidden)
        workspace = w.new_empty(ws_bytes, dtype=torch.uint8)
    p_rstd = stats.data_ptr()
    _lib.call("mrl_norm_bwd", dy.data_ptr(), dy_stride, flat.data_ptr(), x_stride, _lib.dtype_code(flat), n_rows, hidden,
              w.data_ptr(), _lib.dtype_code(w), p_rstd + 4 * n_rows if layer else None, p_rstd, _lib.ptr(dx), _lib.ptr(dw),
              _lib.ptr(db), _lib.ptr(workspace), ws_bytes, _lib.stream(dev))
    return dx, dw, db, None, None


_backward_once = once_differentiable(_backward)


class _Norm(torch.autograd.Function):
    """(x[..., H], weight[H], bias[H] or None) -> y[..., H]; mean and rstd of the rows are kept for the backward."""

    @staticmethod
    def forward(ctx, x, weight, bias, eps, layer):
        y, flat, x_stride, w, stats = _forward(x, weight, bias, eps, layer, True)
        ctx.save_for_backward(flat, w, stats)
        ctx.meta = (x.shape, stats.shape[1], x.shape[-1], x_stride, layer)
        return y

    @staticmethod
    def backward(ctx, dy):
        # the wrapper that refuses a second differentiation costs as much as a launch: only where there may be one
        return _backward_once(ctx, dy) if torch.is_grad_enabled() else _backward(ctx, dy)


def _norm(x, weight, bias, eps, layer):
    if x.dtype not in _FLOATS:
        raise TypeError("x must be float32, bfloat16 or float16, not %s" % x.dtype)
    if weight.dtype is not x.dtype and weight.dtype is not torch.float32:
        raise TypeError("weight must have the type of x (%s) or float32, not %s" % (x.dtype, weight.dtype))
    if x.dim() < 1 or x.shape[-1] < 1 or weight.dim() != 1 or weight.shape[0] != x.shape[-1]:
        raise ValueError("weight must have the shape of x's last dimension: x %s, weight %s"
                         % (tuple(x.shape), tuple(weight.shape)))
    if bias is not None and (bias.shape != weight.shape or bias.dtype is not weight.dtype):
        raise ValueError("bias must have the shape and type of weight: %s %s and %s %s"
                         % (tuple(bias.shape), bias.dtype, tuple(weight.shape), weight.dtype))
    eps = float(eps)
    if not 0.0 < eps < float("inf"):
        raise ValueError("eps must be positive and finite, not %r" % eps)
    _lib.require_device(x, weight, bias)
    if (torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or (bias is not None and bias.requires_grad))
            or _transformed()):
        return _Norm.apply(x, weight, bias, eps, layer)
    return _forward(x, weight, bias, eps, layer, False)[0]          # nothing for autograd to see


def layer_norm(x, weight, bias=None, eps=1e-5):
    """``(x - mean) * (var + eps)^(-1/2) * weight + bias`` over the last dimension of ``x`` ``[..., H]`` (fp32, bf16
    or fp16; rows of any stride), in fp32, rounded once to the type of ``x``.  ``weight`` and ``bias`` ``[H]`` have the type of
    ``x`` or fp32.  Differentiable (once) with respect to all three; sums over rows are taken in an order that the
    sizes set.  A row's squares have to add up inside fp32, which they do up to a root mean square of 1.8e19 / sqrt(H); a row
    beyond it gives zeros (and the bias) and no gradient, or NaN where its mean overflows too."""
    return _norm(x, weight, bias, eps, True)


def rms_norm(x, weight, eps=1e-6):
    """``x * (mean(x^2) + eps)^(-1/2) * weight`` over the last dimension, otherwise as :func:`layer_norm`."""
    return _norm(x, weight, None, eps, False)


def final_norm(hidden, kwargs):
    """The hidden states that the lm_head takes: ``hidden`` itself, or normalised if the caller of a loss object says
    how (``final_norm_weight=``; ``final_norm_type=`` "rms" (default) or "layer", ``final_norm_bias=``, ``final_norm_eps=``)."""
    weight = kwargs.get("final_norm_weight")
    kind, bias = kwargs.get("final_norm_type", "rms"), kwargs.get("final_norm_bias")
    if kind not in ("rms", "layer"):
        raise ValueError("final_norm_type must be 'rms' or 'layer', not %r" % (kind,))
    if weight is None:
        if bias is not None:
            raise ValueError("final_norm_bias= needs final_norm_weight=")
        return hidden
    if kind == "rms":
        if bias is not None:
            raise ValueError("final_norm_bias= needs final_norm_type='layer'")
        return rms_norm(hidden, weight, kwargs.get("final_norm_eps", 1e-6))
    return layer_norm(hidden, weight, bias, kwargs.get("final_norm_eps", 1e-5))
