"""The update's last step: AdamW over all parameters at once, clipped by the norm of the gradients on the way, without a wait for
the device; moments in 32 or in 8 bits.

The reference takes its optimizer from the training framework below it.  Here it works on what :func:`global_grad_norm` has seen:
the clipped gradients are never written.
"""
import array
import itertools
import operator

import torch
from torch.autograd.graph import increment_version

from . import _lib

_BLOCK = 128                # entries that share a scale
_E4M3 = torch.float8_e4m3fn
_CODES = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}


# what every tensor of a list is asked: the host's time is what a short list takes
_DATA_PTR, _NUMEL, _CONTIGUOUS, _GET_DEVICE = torch.Tensor.data_ptr, torch.Tensor.numel, torch.Tensor.is_contiguous, torch.Tensor.get_device
_DTYPE, _SHAPE, _LAYOUT, _REQUIRES_GRAD, _IS_LEAF = map(operator.attrgetter, ("dtype", "shape", "layout", "requires_grad", "is_leaf"))


_USUAL = {torch.Tensor, torch.nn.Parameter}


def _are_tensors(ts):
    return _USUAL.issuperset(map(type, ts)) or all(isinstance(t, torch.Tensor) for t in ts)


def _blocks(n):
    return -(-n // _BLOCK)


def adamw_state(params, bits=32, master=True):
    """What :func:`adamw_` keeps for ``params`` from one step to the next, as its keyword arguments: ``exp_avg``, ``exp_avg_sq`` (zeros), ``step`` (an
    int64 scalar on the device, 0), with ``bits=8`` ``exp_avg_scale`` and ``exp_avg_sq_scale``, and with ``master`` fp32 copies of the bf16 and
    fp16 parameters (None for those of fp32).  Plain lists of tensors, which ``torch.save`` takes."""
    params = list(params)
    if bits not in (8, 32):
        raise ValueError("bits must be 32 or 8, not %r" % (bits,))
    if not params:
        raise ValueError("no parameters")
    _check_params(params)
    dev = _lib.require_device(*params)
    state = {"exp_avg": [], "exp_avg_sq": [], "step": torch.zeros((), dtype=torch.int64, device=dev)}
    dtype = torch.float32 if bits == 32 else _E4M3
    for name in ("exp_avg", "exp_avg_sq"):
        state[name] = [torch.zeros(p.shape, dtype=dtype, device=dev) for p in params]
        if bits == 8:
            state[name + "_scale"] = [torch.full((_blocks(p.numel()),), 2.0 ** -126, device=dev) for p in params]
    if master:
        state["master"] = [None if p.dtype is torch.float32 else p.detach().float() for p in params]
    return state


def _check_params(params):
    """Their shapes and types."""
    if not _are_tensors(params):
        raise TypeError("parameters must be tensors, not %s" % sorted({type(p).__name__ for p in params}))
    dtypes = [*map(_DTYPE, params)]
    if not _CODES.keys() >= set(dtypes) or {*map(_LAYOUT, params)} - {torch.strided}:
        raise TypeError("parameters must be dense float32, bfloat16 or float16 tensors")
    shapes = [*map(_SHAPE, params)]
    if False in map(_CONTIGUOUS, params):
        raise ValueError("parameters must be contiguous: of the shapes %s not all are" % [tuple(s) for s in shapes])
    if False in map(_IS_LEAF, params):
        raise ValueError("a parameter is the result of a graph: give leaves or detached tensors")
    return shapes, dtypes


def _check_held(name, held, shapes, dtype):
    """What the step keeps: tensors of `dtype` and the parameters' shapes, as they lie in memory."""
    if not _are_tensors(held) or {*map(_DTYPE, held)} - {dtype} or [*map(_SHAPE, held)] != shapes or False in map(_CONTIGUOUS, held):
        raise ValueError("%s must hold contiguous tensors of %s with the parameters' shapes" % (name, dtype))
    if True in map(_REQUIRES_GRAD, held):
        raise ValueError("what the step keeps is part of a graph: give detached tensors")


def _check_grads(grads, shapes, dtypes):
    """Their types."""
    if not _are_tensors(grads) or {*map(_LAYOUT, grads)} - {torch.strided}:
        raise ValueError("gradients must be dense tensors")
    types = [*map(_DTYPE, grads)]
    if [*map(_SHAPE, grads)] != shapes or (types != dtypes and any(g is not p and g is not torch.float32 for g, p in zip(types, dtypes))):
        raise ValueError("a gradient must have the shape of its parameter, and its type or float32")
    return types


def adamw_(params, grads, exp_avg, exp_avg_sq, step, lr, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01, master=None,
           exp_avg_scale=None, exp_avg_sq_scale=None, grad_norm=None, max_norm=None):
    """One step of AdamW (decoupled weight decay) for every tensor of ``params``, in place:

        ``m = b1 m + (1 - b1) g``, ``v = b2 v + (1 - b2) g^2``,
        ``p = p (1 - lr weight_decay) - m / (sqrt(v) / sqrt(1 - b2^t) + eps) * lr / (1 - b1^t)``, ``t`` the number of this step

    ``params``: contiguous fp32, bf16 or fp16 tensors (leaves that require gradients are meant; what a graph has computed is refused), ``grads``: for each a gradient of the
    same shape and of the parameter's type or fp32, or None, which leaves its parameter alone.  The others are those of :func:`adamw_state`:
    ``adamw_(params, grads, **state, lr=...)``; parameters with another ``lr`` or ``weight_decay`` take a call and a state of their own.
    ``master``: fp32 weights that the step is taken on; the parameter is their rounded value.  ``exp_avg_scale`` and ``exp_avg_sq_scale``
    belong to moments in 8 bits (``torch.float8_e4m3fn``: of ``m`` and ``sqrt(v)`` over their scales, blocks of 128 entries, rounded
    up or down by a hash of the step and the place, so that the same call gives the same bits; ``v`` is then held a few percent too large, as
    the square of what is rounded).  One ``step`` counts for all: a parameter whose gradient was None until now has its first moments corrected as if they had
    been formed from the beginning.

    ``grad_norm`` (the fp32 scalar of :func:`global_grad_norm`) and ``max_norm``: gradients are multiplied by ``min(1, max_norm / (grad_norm + 1e-6))``
    first, as :func:`clip_grad_norm_` would have it (but for the factor's last bit, which is that of torch's clipping: ``max_norm`` times the
    reciprocal).  ``lr`` may be an fp32 scalar on the device.  ``step`` is counted up on the device, and a
    captured call can be replayed.  Gradients have to be finite.  Nothing that is written may share memory with anything else of the call."""
    params, grads, exp_avg, exp_avg_sq = list(params), list(grads), list(exp_avg), list(exp_avg_sq)
    small = exp_avg_scale is not None or exp_avg_sq_scale is not None
    if small and (exp_avg_scale is None or exp_avg_sq_scale is None):
        raise ValueError("exp_avg_scale and exp_avg_sq_scale belong together")
    lists = [params, grads, exp_avg, exp_avg_sq]
    lists += [list(x) for x in (master, exp_avg_scale, exp_avg_sq_scale) if x is not None]
    if len(set(map(len, lists))) != 1:
        raise ValueError("lists of one length are wanted: %s" % ([len(x) for x in lists],))
    lr_at = None
    if isinstance(lr, torch.Tensor):
        if lr.dtype is not torch.float32 or lr.numel() != 1:
            raise TypeError("lr must be a number or one float32 on the device, not %s %s" % (lr.dtype, tuple(lr.shape)))
        lr_at, lr_value = lr.data_ptr(), 0.0
    else:
        lr_value = float(lr)
    b1, b2 = map(float, betas)
    eps, weight_decay = float(eps), float(weight_decay)
    if not (0.0 <= b1 < 1.0 and 0.0 <= b2 < 1.0):
        raise ValueError("betas must lie in [0, 1): %r" % (betas,))
    if not (0.0 <= lr_value < float("inf") and 1e-30 <= eps < float("inf") and 0.0 <= weight_decay < float("inf")):
        raise ValueError("lr and weight_decay must not be negative, and eps at least 1e-30: %r, %r, %r" % (lr, weight_decay, eps))
    if not isinstance(step, torch.Tensor) or step.dtype is not torch.int64 or step.numel() != 1:
        raise TypeError("step must be one int64 on the device")
    if (grad_norm is None) != (max_norm is None):
        raise ValueError("grad_norm and max_norm belong together")
    if grad_norm is not None:
        max_norm = float(max_norm)
        if not isinstance(grad_norm, torch.Tensor) or grad_norm.dtype is not torch.float32 or grad_norm.numel() != 1:
            raise TypeError("grad_norm must be one float32 on the device")
        if not max_norm >= 0.0:
            raise ValueError("max_norm must not be negative: %r" % max_norm)
    shapes, dtypes = _check_params(params)
    if any(g is None for g in grads):
        kept = [k for k, g in enumerate(grads) if g is not None]
        lists = [[x[k] for k in kept] for x in lists]
        params, grads = lists[:2]
        shapes, dtypes = [shapes[k] for k in kept], [dtypes[k] for k in kept]
    held = lists[2:4]
    types = _check_grads(grads, shapes, dtypes)
    for name, x in zip(("exp_avg", "exp_avg_sq"), held):
        _check_held(name, x, shapes, _E4M3 if small else torch.float32)
    sizes = [*map(_NUMEL, params)]
    columns = [[*map(_DATA_PTR, params)], None, itertools.repeat(0), *([*map(_DATA_PTR, x)] for x in held)]
    if master is not None:
        main = lists[4]
        if any(w is not None and p is torch.float32 for w, p in zip(main, dtypes)):
            raise ValueError("a float32 parameter is its own main weight: its entry of master must be None")
        there = [k for k, w in enumerate(main) if w is not None]
        only = [main[k] for k in there]
        _check_held("master", only, [shapes[k] for k in there], torch.float32)
        columns[2] = [0 if w is None else w.data_ptr() for w in main]
        held = [*held, only]
    if small:
        counts = [torch.Size((_blocks(n),)) for n in sizes]
        for name, x in zip(("exp_avg_scale", "exp_avg_sq_scale"), lists[-2:]):
            _check_held(name, x, counts, torch.float32)
            columns.append([*map(_DATA_PTR, x)])
        held = [*held, *lists[-2:]]
    else:
        columns += [itertools.repeat(0)] * 2
    codes = [_CODES[p] | _CODES[g] << 32 for p, g in zip(dtypes, types)]
    written = [step, *params, *itertools.chain.from_iterable(held)]
    devices = set(map(_GET_DEVICE, itertools.chain(written, grads)))
    if len(devices) != 1 or -1 in devices:
        _lib.require_device(*written, *grads)       # raises
    dev = _lib.require_device(step, grad_norm, lr if lr_at is not None else None)
    dense = grads if False not in map(_CONTIGUOUS, grads) else [g.detach().contiguous() for g in grads]
    columns[1] = [*map(_DATA_PTR, dense)]
    table = array.array("q", itertools.chain.from_iterable(zip(*columns, sizes, codes)))
    coefs = torch.empty(8, dtype=torch.float32, device=dev)
    _lib.call("mrl_adamw_step", table.buffer_info()[0], len(sizes), 8 if small else 32, step.data_ptr(), lr_value, lr_at, b1, b2, eps,
              weight_decay, _lib.ptr(grad_norm), max_norm or 0.0, coefs.data_ptr(), _lib.stream(dev))
    try:
        increment_version(written)          # autograd looks whether what it kept has been written to
    except RuntimeError:                    # of tensors of inference mode it keeps none
        increment_version([t for t in written if not t.is_inference()])
