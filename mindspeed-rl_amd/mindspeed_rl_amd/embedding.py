"""Rows of the token table and the table's gradient: the other end of the ``[V, H]`` weight that the lm_head functions
(:mod:`lmhead`) project with.

A table that both ends share has two gradients: the lm_head's, which is dense, and the tokens'.  :func:`token_embedding_grad`
with ``accumulate=True`` adds the latter to the former and touches the named rows alone.
"""
import functools
import math

import torch
from torch.autograd.function import once_differentiable
from torch.autograd.graph import increment_version

from . import _lib
from .vocab_ops import _transformed

_FLOATS = (torch.float32, torch.bfloat16, torch.float16)


def _check(ids, scale, vocab_start):
    if ids.dtype.is_floating_point or ids.dtype.is_complex or ids.dtype is torch.bool:
        raise TypeError("ids must be integers, not %s" % ids.dtype)
    scale, vocab_start = float(scale), int(vocab_start)
    if not math.isfinite(scale):
        raise ValueError("scale must be finite, not %r" % scale)
    if not 0 <= vocab_start < 1 << 63:
        raise ValueError("vocab_start must not be negative, nor beyond 64 bits: %d" % vocab_start)
    return scale, vocab_start


@functools.lru_cache(maxsize=256)
def _workspace_bytes(n_tokens, vocab, hidden):
    """mrl_embedding_bwd_workspace_bytes: a function of its arguments alone."""
    return _lib.load().mrl_embedding_bwd_workspace_bytes(n_tokens, vocab, hidden)


def _add_up(ids, dy, scale, vocab_start, out, accumulate):
    """mrl_embedding_bwd: ``dy`` of ``ids`` (both dense) into ``out`` ``[V, H]``."""
    dev = out.device
    vocab, hidden = out.shape
    n = ids.numel()
    ws_bytes = _workspace_bytes(n, vocab, hidden)
    workspace = out.new_empty(ws_bytes, dtype=torch.uint8) if ws_bytes else None
    _lib.call("mrl_embedding_bwd", ids.data_ptr(), _lib.dtype_code(ids), n, vocab_start, dy.data_ptr(), _lib.dtype_code(dy), vocab,
              hidden, scale, out.data_ptr(), _lib.dtype_code(out), 1 if accumulate else 0, _lib.ptr(workspace), ws_bytes,
              _lib.stream(dev))
    return out


def _look_up(ids, weight, scale, vocab_start):
    """The rows, and the ids as the kernels take them."""
    dev = weight.device
    table, flat = weight.contiguous(), _lib.index_column(ids, dev)
    vocab, hidden = table.shape
    out = table.new_empty((*ids.shape, hidden))
    _lib.call("mrl_embedding_fwd", flat.data_ptr(), _lib.dtype_code(flat), flat.numel(), vocab_start, table.data_ptr(),
              _lib.dtype_code(table), vocab, hidden, scale, out.data_ptr(), _lib.stream(dev))
    return out, flat


def _backward(ctx, dy):
    (flat,) = ctx.saved_tensors
    shape, dtype, scale, vocab_start = ctx.meta
    out = dy.new_empty(shape, dtype=dtype)
    return None, _add_up(flat, dy.contiguous(), scale, vocab_start, out, False), None, None


_backward_once = once_differentiable(_backward)


class _TokenEmbedding(torch.autograd.Function):
    """(ids[...], weight[V, H]) -> [..., H]; the backward gives the dense gradient of the table."""

    @staticmethod
    def forward(ctx, ids, weight, scale, vocab_start):
        out, flat = _look_up(ids, weight, scale, vocab_start)
        ctx.save_for_backward(flat)
        ctx.meta = (weight.shape, weight.dtype, scale, vocab_start)
        return out

    @staticmethod
    def backward(ctx, dy):
        # the wrapper that refuses a second differentiation costs as much as a launch: only where there may be one
        return _backward_once(ctx, dy) if torch.is_grad_enabled() else _backward(ctx, dy)


def token_embedding(ids, weight, scale=1.0, vocab_start=0):
    """``scale * weight[ids - vocab_start]``: ``ids`` ``[...]`` integers, ``weight`` ``[V, H]`` (fp32, bf16 or fp16) ->
    ``[..., H]``.  Ids outside ``[vocab_start, vocab_start + V)`` give zeros and take no part in the gradient: another rank's
    share of a table, or positions without a token (-1, say).  Differentiable (once) with respect to ``weight``: the dense
    gradient, tokens sorted by row and summed in fp32, the same bits from run to run."""
    if weight.dtype not in _FLOATS:
        raise TypeError("weight must be float32, bfloat16 or float16, not %s" % weight.dtype)
    if weight.dim() != 2 or weight.shape[0] < 1 or weight.shape[1] < 1:
        raise ValueError("weight must have shape (vocab, hidden_dim), not %s" % (tuple(weight.shape),))
    scale, vocab_start = _check(ids, scale, vocab_start)
    _lib.require_device(ids, weight)
    if torch.is_grad_enabled() and weight.requires_grad or _transformed():
        return _TokenEmbedding.apply(ids, weight, scale, vocab_start)
    return _look_up(ids, weight, scale, vocab_start)[0]             # nothing for autograd to see


def token_embedding_grad(ids, grad, out, scale=1.0, vocab_start=0, accumulate=False):
    """The table's gradient without autograd, into ``out`` ``[V, H]`` (dense, of ``grad``'s type or fp32): ``out[v] = scale *
    sum of grad over the tokens with ids - vocab_start == v``, or ``out[v] +=`` that, with the other rows untouched, if
    ``accumulate``.  ``grad`` is ``ids.shape + (H,)`` and shares no memory with ``out``.  Returns ``out``."""
    if grad.dtype not in _FLOATS or (out.dtype is not grad.dtype and out.dtype is not torch.float32):
        raise TypeError("grad must be float32, bfloat16 or float16 and out of its type or float32: %s and %s"
                        % (grad.dtype, out.dtype))
    if out.dim() != 2 or out.shape[0] < 1 or out.shape[1] < 1 or not out.is_contiguous():
        raise ValueError("out must be a dense (vocab, hidden_dim) tensor")
    if tuple(grad.shape) != tuple(ids.shape) + (out.shape[1],):
        raise ValueError("grad must have shape %s, not %s" % (tuple(ids.shape) + (out.shape[1],), tuple(grad.shape)))
    if out.requires_grad:
        raise ValueError("out is part of a graph: give its gradient or a detached tensor")
    scale, vocab_start = _check(ids, scale, vocab_start)
    dev = _lib.require_device(ids, grad, out)
    _add_up(_lib.index_column(ids, dev), grad.detach().contiguous(), scale, vocab_start, out, accumulate)
    increment_version(out)
    return out
