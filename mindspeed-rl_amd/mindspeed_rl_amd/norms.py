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
_CODES = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}


@functools.lru_cache(maxsize=256)
def _workspace_bytes(n_rows, hidden):
    """mrl_norm_bwd_workspace_bytes: a function of its arguments alone."""
    return _lib.load().mrl_norm_bwd_workspace_bytes(n_rows, hidden)


@functools.lru_cache(maxsize=256)
def _add_workspace_bytes(n_rows, hidden):
    """mrl_add_norm_bwd_workspace_bytes: a function of its arguments alone."""
    return _lib.load().mrl_add_norm_bwd_workspace_bytes(n_rows, hidden)


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


def _added(x, residual, weight, eps):
    """What :func:`add_rms_norm` and :func:`rms_norm_fp8` ask of their arguments."""
    dtype, shape = x.dtype, x.shape
    if dtype not in _FLOATS:
        raise TypeError("x must be float32, bfloat16 or float16, not %s" % dtype)
    if weight.dtype is not dtype and weight.dtype is not torch.float32:
        raise TypeError("weight must have the type of x (%s) or float32, not %s" % (dtype, weight.dtype))
    if len(shape) < 1 or shape[-1] < 1 or weight.dim() != 1 or weight.shape[0] != shape[-1]:
        raise ValueError("weight must have the shape of x's last dimension: x %s, weight %s" % (tuple(shape), tuple(weight.shape)))
    if residual is not None:
        if residual.dtype is not dtype and residual.dtype is not torch.float32:
            raise TypeError("residual must have the type of x (%s) or float32, not %s" % (dtype, residual.dtype))
        if residual.shape != shape:
            raise ValueError("residual must have the shape of x: %s and %s" % (tuple(residual.shape), tuple(shape)))
    eps = float(eps)
    if not 0.0 < eps < float("inf"):
        raise ValueError("eps must be positive and finite, not %r" % eps)
    _lib.require_device(x, residual, weight)
    return eps


def _add_forward(x, residual, weight, eps, keep):
    """y, h and, if `keep`, rstd of the rows; the weight as the kernels read it."""
    dev, hidden, w = x.device, x.shape[-1], weight.contiguous()
    n_rows, flat, res, x_stride, r_stride = x.numel() // hidden, x, residual, hidden, hidden
    if x.is_contiguous() and residual.is_contiguous():
        y, h = torch.empty_like(x), torch.empty_like(residual)
    else:
        flat, x_stride = _flat_rows(x)
        res, r_stride = _flat_rows(residual)
        y, h = x.new_empty(x.shape), residual.new_empty(x.shape)
    rstd = w.new_empty(n_rows, dtype=torch.float32) if keep else None
    _lib.call("mrl_add_norm_fwd", flat.data_ptr(), _CODES[x.dtype], x_stride, res.data_ptr(), _CODES[residual.dtype], r_stride,
              n_rows, hidden, w.data_ptr(), _CODES[w.dtype], eps, h.data_ptr(), y.data_ptr(), _lib.ptr(rstd), _lib.stream(dev))
    return y, h, w, rstd


def _add_backward(ctx, dy, dh):
    h, w, rstd = ctx.saved_tensors
    shape, dtype = ctx.meta
    dev, hidden, n_rows = h.device, shape[-1], rstd.shape[0]
    need_x, need_r, need_w = ctx.needs_input_grad[:3]
    if dy is None:                          # nothing came back through the norm
        dw = torch.zeros_like(w) if need_w else None
        if dh is None:
            return None, None, dw, None
        return dh.to(dtype) if need_x else None, dh if need_r else None, dw, None
    dy_stride = dh_stride = hidden
    if not dy.is_contiguous():
        dy, dy_stride = _flat_rows(dy)
    if dh is not None and not dh.is_contiguous():
        dh, dh_stride = _flat_rows(dh)
    # dy has the type of x, and its shape unless it was spread out
    dx = (torch.empty_like(dy) if dy.shape == shape and dy_stride == hidden else dy.new_empty(shape)) if need_x else None
    dr = torch.empty_like(h) if need_r and not (need_x and h.dtype is dtype) else None
    dw = workspace = None
    ws_bytes = 0
    if need_w:
        dw = torch.empty_like(w)
        ws_bytes = _add_workspace_bytes(n_rows, hidden)
        workspace = w.new_empty(ws_bytes, dtype=torch.uint8)
    _lib.call("mrl_add_norm_bwd", dy.data_ptr(), dy_stride, _lib.ptr(dh), dh_stride, h.data_ptr(), _CODES[h.dtype], _CODES[dtype],
              n_rows, hidden, w.data_ptr(), _CODES[w.dtype], rstd.data_ptr(), _lib.ptr(dx), _lib.ptr(dr), _lib.ptr(dw),
              _lib.ptr(workspace), ws_bytes, _lib.stream(dev))
    return dx, dr if dr is not None or not need_r else dx, dw, None


_add_backward_once = once_differentiable(_add_backward)


class _AddNorm(torch.autograd.Function):
    """(x[..., H], residual[..., H], weight[H]) -> y, h; h itself and rstd of the rows are kept for the backward."""

    @staticmethod
    def forward(ctx, x, residual, weight, eps):
        y, h, w, rstd = _add_forward(x, residual, weight, eps, True)
        ctx.save_for_backward(h, w, rstd)
        ctx.meta = (x.shape, x.dtype)
        ctx.set_materialize_grads(False)
        return y, h

    @staticmethod
    def backward(ctx, dy, dh):
        return _add_backward_once(ctx, dy, dh) if torch.is_grad_enabled() else _add_backward(ctx, dy, dh)


def add_rms_norm(x, residual, weight, eps=1e-6):
    """``(y, h)``: the residual stream behind a layer, ``h = x + residual``, and its RMS norm ``y = h * (mean(h^2) + eps)^(-1/2) *
    weight`` for the next one, in one pass.  ``x`` ``[..., H]`` is fp32, bf16 or fp16, ``residual`` of the same shape and of the type of
    ``x`` or fp32 (rows of any stride), ``weight`` ``[H]`` of the type of ``x`` or fp32; ``h`` has the residual's type and ``y`` that of ``x``.
    The norm is that of ``h`` as it is returned, so the call gives what ``rms_norm(x + residual, weight)`` gives but for the order
    of the sums.  Differentiable (once) with respect to all three, from gradients of either output or both; the same limits
    as :func:`layer_norm`'s, and fewer than 2^24 rows."""
    eps = _added(x, residual, weight, eps)
    if torch.is_grad_enabled() and (x.requires_grad or residual.requires_grad or weight.requires_grad) or _transformed():
        return _AddNorm.apply(x, residual, weight, eps)
    return _add_forward(x, residual, weight, eps, False)[:2]


def rms_norm_fp8(x, weight, eps=1e-6, residual=None, block=None):
    """``(q, scale)``: the RMS norm of ``x`` in 8 bits, for a product that takes OCP e4m3 operands: ``q`` (``torch.float8_e4m3fn``, the shape of
    ``x``) times ``scale`` (fp32) is the norm.  ``block=None``: a scale for each row, ``[..., 1]``; ``block=128``: one for each 128 entries, ``[..., H /
    128]`` (``H`` a multiple of 128).  ``scale`` is the largest magnitude times 1/448, at least 2^-126, and ``q`` the fp32 quotient by it rounded to the
    nearest, ties to even.  With ``residual`` the norm is that of ``h = x + residual`` as in :func:`add_rms_norm`, and ``(q, scale, h)`` is returned.
    A pass without gradients: with inputs that require one it is refused."""
    eps = _added(x, residual, weight, eps)
    if block is not None and block != 128:
        raise ValueError("block must be None (a scale for each row) or 128, not %r" % (block,))
    hidden = x.shape[-1]
    if block and hidden % block:
        raise ValueError("rows of %d entries are not whole blocks of %d" % (hidden, block))
    if (torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or (residual is not None and residual.requires_grad))
            or _transformed()):
        raise RuntimeError("rms_norm_fp8 has no gradient: call it under torch.no_grad() or with detached tensors")
    dev, w, x_stride = x.device, weight.contiguous(), hidden
    flat, n_rows = x, x.numel() // hidden
    if not x.is_contiguous():
        flat, x_stride = _flat_rows(x)
    res, r_stride, h = None, hidden, None
    if residual is not None:
        res, r_stride = (residual, hidden) if residual.is_contiguous() else _flat_rows(residual)
        h = residual.new_empty(x.shape)
    q = x.new_empty(x.shape, dtype=torch.float8_e4m3fn)
    scale = x.new_empty((*x.shape[:-1], hidden // block if block else 1), dtype=torch.float32)
    _lib.call("mrl_norm_fp8_fwd", flat.data_ptr(), _CODES[x.dtype], x_stride, _lib.ptr(res), _CODES[(x if res is None else res).dtype],
              r_stride, n_rows, hidden, w.data_ptr(), _CODES[w.dtype], eps, block or 0, _lib.ptr(h), q.data_ptr(), scale.data_ptr(),
              _lib.stream(dev))
    return (q, scale) if h is None else (q, scale, h)


def final_norm(hidden, kwargs):
    """The hidden states that the lm_head takes: ``hidden`` itself, or normalised if the caller of a loss object says
    how (``final_norm_weight=``; ``final_norm_type=`` "rms" (default) or "layer", ``final_norm_bias=``, ``final_norm_eps=``;
    ``final_norm_residual=``: the residual stream that the RMS norm adds the last layer's output ``hidden`` to)."""
    weight = kwargs.get("final_norm_weight")
    kind, bias = kwargs.get("final_norm_type", "rms"), kwargs.get("final_norm_bias")
    residual = kwargs.get("final_norm_residual")
    if kind not in ("rms", "layer"):
        raise ValueError("final_norm_type must be 'rms' or 'layer', not %r" % (kind,))
    if weight is None:
        if bias is not None:
            raise ValueError("final_norm_bias= needs final_norm_weight=")
        if residual is not None:
            raise ValueError("final_norm_residual= needs final_norm_weight=")
        return hidden
    if kind == "rms":
        if bias is not None:
            raise ValueError("final_norm_bias= needs final_norm_type='layer'")
        eps = kwargs.get("final_norm_eps", 1e-6)
        return rms_norm(hidden, weight, eps) if residual is None else add_rms_norm(hidden, residual, weight, eps)[0]
    if residual is not None:
        raise ValueError("final_norm_residual= needs final_norm_type='rms'")
    return layer_norm(hidden, weight, bias, kwargs.get("final_norm_eps", 1e-5))
