"""The global norm of a step's gradients and clipping by it, without a wait for the device.

The reference's optimizer reports the norm of every update (``grad_norm``) and clips by it before the weights move; it takes
both from the training framework below it.  Here they work on the gradients that :func:`fused_lmhead_policy_loss`,
:func:`token_embedding` and the norms leave behind, whatever their types.
"""
import array
import operator

import torch
from torch.autograd.graph import increment_version

from . import _lib

_PARTIALS = 2304            # MRL_GRAD_NORM_PARTIALS
# names that every tensor of a list is met with: the host's time is what a short list takes
_TENSOR, _STRIDED, _GET_DEVICE = torch.Tensor, torch.strided, torch.Tensor.get_device
_REQUIRES_GRAD = operator.attrgetter("requires_grad")
_CODES = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}


def _code(g):
    """The dtype code of a gradient that can be taken."""
    if not isinstance(g, _TENSOR):
        raise TypeError("gradients must be tensors, not %s" % type(g).__name__)
    code = _CODES.get(g.dtype)
    if code is None or g.layout is not _STRIDED:
        raise TypeError("gradients must be dense float32, bfloat16 or float16 tensors, not %s of %s" % (g.layout, g.dtype))
    return code


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


def _device(tensors):
    """Their one device, as :func:`_lib.require_device` would have it."""
    if not tensors:
        raise ValueError("no gradients")
    indices = set(map(_GET_DEVICE, tensors))
    if len(indices) != 1 or -1 in indices:
        _lib.require_device(*tensors)       # raises
    return _lib.require_device(tensors[0])


def _result(dev):
    """Where the norm goes, and the partial sums."""
    return torch.empty((), dtype=torch.float32, device=dev), torch.empty(_PARTIALS, dtype=torch.float64, device=dev)


def global_grad_norm(grads):
    """The 2-norm over all entries of ``grads`` (a tensor, or an iterable of them; None is skipped) as an fp32 scalar on their
    device: squares and sums in fp64, in an order that the sizes set.  A tensor that is listed twice counts twice.  Not
    differentiable."""
    grads = [grads] if isinstance(grads, torch.Tensor) else [g for g in grads if g is not None]
    words, kept = [], []
    for g in grads:
        code = _code(g)
        if not _fills(g):
            g = g.detach().contiguous()
            kept.append(g)
        words += (g.data_ptr(), 0, g.numel(), code | code << 32)
    dev = _device(grads)
    table = array.array("q", words)
    norm, partial = _result(dev)
    _lib.call("mrl_grad_norm", table.buffer_info()[0], len(grads), norm.data_ptr(), partial.data_ptr(), _lib.stream(dev))
    return norm


def _places(t):
    """(first byte, bytes that lie together, [(step in bytes, how many), the widest first]) of the entries."""
    together, steps = t.element_size(), []
    for st, n in _steps(t):
        st *= t.element_size()
        if st == together and not steps:
            together *= n
        elif st > 0:                        # entries of an expanded dimension are the same ones
            steps.insert(0, (st, n))
    return t.data_ptr(), together, steps


def _end(places):
    at, together, steps = places
    return at + together + sum((n - 1) * st for st, n in steps)


def _meet(a, b):
    """Whether two :func:`_places` have a byte in common."""
    if a[0] >= _end(b) or b[0] >= _end(a):
        return False
    if not a[2] or (b[2] and b[2][0][0] > a[2][0][0]):
        a, b = b, a
    if not a[2]:
        return True
    (st, n), least = a[2][0], 0
    a = a[0], a[1], a[2][1:]
    if b[2] and b[2][0][0] == st:           # of two equal steps their difference counts
        least, b = 1 - b[2][0][1], (b[0], b[1], b[2][1:])
    # the blocks of a that begin in front of b's end and end behind its begin
    first, last = max(least, (b[0] - _end(a)) // st + 1), min(n - 1, (_end(b) - 1 - a[0]) // st)
    return any(_meet((a[0] + d * st, a[1], a[2]), b) for d in range(first, last + 1))


def _refuse_shared(pairs):
    """What the entry point sees to for dense tensors, for (gradient, output) some of which it gets as copies."""
    everything = []
    for g, o in pairs:
        if g.numel() > 0:
            everything.append((_places(o), True))
            if g.data_ptr() != o.data_ptr() or g.dtype is not o.dtype or any(
                    n > 1 and p != q for p, q, n in zip(g.stride(), o.stride(), g.shape)):
                everything.append((_places(g), False))
    everything.sort()
    reach = []                              # those that may reach the next one
    for places, written in everything:
        reach = [r for r in reach if _end(r[0]) > places[0]]
        if any((written or r[1]) and _meet(r[0], places) for r in reach):
            raise ValueError("a tensor shares memory with another that is written")
        reach.append((places, written))


def _spaced(g, o, in_place):
    """(gradient, output) as dense tensors of one order, by copies where they are not."""
    source = g.detach().contiguous()
    if o.is_contiguous():
        return source, o
    extent = 1
    for st, n in _steps(o):
        if st < extent:
            raise ValueError("an output's entries share memory")
        extent += (n - 1) * st
    return source, source if in_place else torch.empty(o.shape, dtype=o.dtype, device=o.device)


def clip_grad_norm_(grads, max_norm, out=None):
    """Scales all ``grads`` by ``min(1, max_norm / (norm + 1e-6))`` and returns ``norm`` (:func:`global_grad_norm`), without
    a host synchronisation.  In place - gradients below the limit are then not touched - or into the tensors of ``out``, one
    for each of ``grads``, of the same shape and of the gradient's type or fp32 (an optimizer's main gradients).  What is written
    may not share memory with anything else in the lists, nor be part of a graph (the gradients are meant, not the parameters).
    A norm that is not finite gives what the formula gives."""
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError("max_norm must not be negative: %r" % max_norm)
    grads = [grads] if isinstance(grads, torch.Tensor) else list(grads)
    words, back, tensors, written = [], [], [], []
    if out is None:
        written = tensors
        for g in grads:
            if g is None:
                continue
            code = _code(g)
            tensors.append(g)
            p = q = g.data_ptr()
            if not _fills(g):
                source, target = _spaced(g, g, True)
                back.append((g, target))
                p, q = source.data_ptr(), target.data_ptr()
            words += (p, q, g.numel(), code | code << 32)
    else:
        outs = [out] if isinstance(out, torch.Tensor) else list(out)
        if len(grads) != len(outs):
            raise ValueError("%d gradients and %d outputs" % (len(grads), len(outs)))
        for g, o in zip(grads, outs):
            if g is None:
                continue
            if o is None:
                raise ValueError("a gradient without an output")
            code, to = _code(g), _code(o)
            if g.shape != o.shape or (to != code and to != _lib.F32):
                raise ValueError("an output must have the shape of its gradient, and its type or float32: %s %s and %s %s"
                                 % (tuple(g.shape), g.dtype, tuple(o.shape), o.dtype))
            tensors += (g, o)
            written.append(o)
            p, q = g.data_ptr(), o.data_ptr()
            if not (g.is_contiguous() and o.is_contiguous()) and not (p == q and g.stride() == o.stride() and _fills(g)):
                source, target = _spaced(g, o, False)
                back.append((o, target, source))
                p, q = source.data_ptr(), target.data_ptr()
            words += (p, q, g.numel(), code | to << 32)
    if back:
        _refuse_shared(zip(tensors, tensors) if out is None else zip(tensors[::2], written))
    if True in map(_REQUIRES_GRAD, written):
        raise ValueError("what is written is part of a graph: give the gradients (p.grad, not p) or detached tensors")
    dev = _device(tensors)
    table = array.array("q", words)
    norm, partial = _result(dev)
    _lib.call("mrl_grad_clip", table.buffer_info()[0], len(words) // 4, max_norm, norm.data_ptr(), partial.data_ptr(),
              _lib.stream(dev))
    increment_version(written)              # autograd looks whether what it kept has been written to
    for o, target, *_ in back:
        if target is not o:
            o.detach().copy_(target)
    return norm
