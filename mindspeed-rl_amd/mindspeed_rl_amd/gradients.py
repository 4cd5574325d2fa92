"""The global norm of a step's gradients and clipping by it, without a wait for the device.

The reference's optimizer reports the norm of every update (``grad_norm``) and clips by it before the weights move; it takes
both from the training framework below it.  Here they work on the gradients that :func:`fused_lmhead_policy_loss`,
:func:`token_embedding` and the norms leave behind, whatever their types.
"""
import array

import torch

from . import _lib

_PARTIALS = 2048            # MRL_GRAD_NORM_PARTIALS
_CODES = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}


def _listed(grads):
    grads = [grads] if isinstance(grads, torch.Tensor) else [g for g in grads if g is not None]
    for g in grads:
        if not isinstance(g, torch.Tensor):
            raise TypeError("gradients must be tensors, not %s" % type(g).__name__)
        if g.layout is not torch.strided or g.dtype not in _CODES:
            raise TypeError("gradients must be dense float32, bfloat16 or float16 tensors, not %s of %s" % (g.layout, g.dtype))
    return grads


def _steps(t):
    """(stride, size) of the dimensions that move, the closest entries first."""
    return sorted((st, n) for st, n in zip(t.stride(), t.shape) if n > 1)


def _fills(t):
    """True where the entries fill their stretch of memory, in whatever order."""
    if t.is_contiguous():
        return True
    extent = 1
    for st, n in _steps(t):
        if st != extent:
            return False
        extent *= n
    return True


def _table(pairs):
    """The list as mrl_grad structures: ``pairs`` of (gradient, output or None), dense."""
    words = array.array("q")
    for g, o in pairs:
        code = _CODES[g.dtype]
        if o is None:
            words.extend((g.data_ptr(), 0, g.numel(), code | code << 32))
        else:
            words.extend((g.data_ptr(), o.data_ptr(), g.numel(), code | _CODES[o.dtype] << 32))
    return words


def _result(dev):
    """Where the norm goes, and the partial sums."""
    return torch.empty((), dtype=torch.float32, device=dev), torch.empty(_PARTIALS, dtype=torch.float64, device=dev)


def global_grad_norm(grads):
    """The 2-norm over all entries of ``grads`` (a tensor, or an iterable of them; None is skipped) as an fp32 scalar on their
    device: squares and sums in fp64, in an order that the sizes set.  A tensor that is listed twice counts twice.  Not
    differentiable."""
    grads = _listed(grads)
    if not grads:
        raise ValueError("no gradients")
    dev = _lib.require_device(*grads)
    pairs = [(g if _fills(g) else g.detach().contiguous(), None) for g in grads]
    words = _table(pairs)
    norm, partial = _result(dev)
    _lib.call("mrl_grad_norm", words.buffer_info()[0], len(pairs), norm.data_ptr(), partial.data_ptr(), _lib.stream(dev))
    return norm


def clip_grad_norm_(grads, max_norm, out=None):
    """Scales all ``grads`` by ``min(1, max_norm / (norm + 1e-6))`` and returns ``norm`` (:func:`global_grad_norm`), without
    a host synchronisation.  In place - gradients below the limit are then not touched - or into the tensors of ``out``, one
    for each of ``grads``, of the same shape and of the gradient's type or fp32 (an optimizer's main gradients).  What is written
    may not share memory with anything else in the lists.  A norm that is not finite gives what the formula gives."""
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError("max_norm must not be negative: %r" % max_norm)
    if out is None:
        grads = _listed(grads)
        outs = grads
    else:
        grads = [grads] if isinstance(grads, torch.Tensor) else list(grads)
        outs = [out] if isinstance(out, torch.Tensor) else list(out)
        if len(grads) != len(outs):
            raise ValueError("%d gradients and %d outputs" % (len(grads), len(outs)))
        both = [(g, o) for g, o in zip(grads, outs) if g is not None]
        grads, outs = _listed([g for g, _ in both]), _listed([o for _, o in both])
        if len(grads) != len(outs):
            raise ValueError("a gradient without an output")
        for g, o in zip(grads, outs):
            if g.shape != o.shape or (o.dtype is not g.dtype and o.dtype is not torch.float32):
                raise ValueError("an output must have the shape of its gradient, and its type or float32: %s %s and %s %s"
                                 % (tuple(g.shape), g.dtype, tuple(o.shape), o.dtype))
    if not grads:
        raise ValueError("no gradients")
    dev = _lib.require_device(*grads, *([] if out is None else outs))
    pairs, back = [], []
    for g, o in zip(grads, outs):
        g, o = g.detach(), o.detach()
        if o.data_ptr() == g.data_ptr() and o.dtype is g.dtype and o.stride() == g.stride() and _fills(g):
            pairs.append((g, g))
            continue
        # entries lie in another order than their outputs, or apart: by way of dense tensors
        source, target = g.contiguous(), o
        if not o.is_contiguous():
            extent = 1
            for st, n in _steps(o):
                if st < extent:
                    raise ValueError("an output's entries share memory")
                extent += (n - 1) * st
            target = source if out is None else torch.empty(o.shape, dtype=o.dtype, device=dev)
            back.append((o, target))
        pairs.append((source, target))
    words = _table(pairs)
    norm, partial = _result(dev)
    _lib.call("mrl_grad_clip", words.buffer_info()[0], len(pairs), max_norm, norm.data_ptr(), partial.data_ptr(),
              _lib.stream(dev))
    for o, target in back:
        o.copy_(target)
    return norm
