"""ctypes binding of libmrl_hip.so (the C ABI declared in include/mrl_hip.h).

The library is the only compute path of this package: if it is missing, loading raises - there
is no CPU or eager-torch fallback.  torch is used for device memory and streams only.
"""
import ctypes
import functools
import os

import torch

from . import _build

# enum mrl_dtype
F32, BF16, F16, I32, I64, U8, F64 = 0, 1, 2, 3, 4, 5, 6
# enum mrl_kl_penalty
KL_NONE, KL_KL, KL_ABS, KL_MSE, KL_LOW_VAR = 0, 1, 2, 3, 4
KL_BY_NAME = {"kl": KL_KL, "abs": KL_ABS, "mse": KL_MSE, "low_var_kl": KL_LOW_VAR}

_TORCH_DTYPE = {
    torch.float32: F32, torch.bfloat16: BF16, torch.float16: F16, torch.int32: I32,
    torch.int64: I64, torch.uint8: U8, torch.bool: U8, torch.float64: F64,
}

_vp = ctypes.c_void_p
_i64 = ctypes.c_int64
_int = ctypes.c_int
_f32 = ctypes.c_float
_f64 = ctypes.c_double

class RaggedColumn(ctypes.Structure):
    """struct mrl_ragged_column"""
    _fields_ = [(name, _vp) for name in ("lengths", "eff_len", "cu", "info", "src", "dst")] + [
        ("pad_bits", ctypes.c_uint64)] + [
        (name, _i64) for name in ("batch", "width", "multiple", "first_dim", "src_stride", "total")] + [
        (name, _int) for name in ("lengths_dtype", "elem_bytes", "left_pad", "reserved")]


RAGGED_COLUMNS = 16         # MRL_RAGGED_COLUMNS
ERR_LAUNCH = -4             # MRL_ERR_LAUNCH


# name -> argtypes; the order is that of include/mrl_hip.h
SIGNATURES = {
    "mrl_version": [],
    "mrl_last_error": [],
    "mrl_host_wait": [_vp, _i64, _vp],
    "mrl_vocab_logprob_fwd": [_vp, _int, _i64, _i64, _i64, _vp, _int, _vp, _f32, _vp, _vp, _vp, _vp],
    "mrl_vocab_logprob_bwd": [_vp, _int, _i64, _i64, _i64, _vp, _int, _f32, _vp, _vp, _vp, _vp, _vp, _int, _i64, _vp],
    "mrl_pack_index_build": [_vp, _int, _i64, _i64, _i64, _vp, _vp, _vp, _vp],
    "mrl_pack_rows": [_vp, _vp, _vp, _vp, _int, _i64, _i64, _vp, _vp, _i64, _vp, _vp],
    "mrl_unpad_gather": [_vp, _int, _i64, _i64, _vp, _vp, _vp, _int, _i64, _i64, _vp, _vp],
    "mrl_pad_scatter": [_vp, _i64, _i64, _vp, _vp, _vp, _int, _i64, _vp, _vp],
    "mrl_window_gather": [_vp, _int, _i64, _i64, _i64, _vp, _int, _i64, ctypes.c_uint64, _vp, _vp],
    "mrl_window_scatter": [_vp, _i64, _i64, _vp, _int, _i64, _vp, _vp],
    "mrl_window_rows": [_int, _i64, _i64, _i64, _vp, _vp, _i64, _vp, _int, _vp, _int, _vp, _vp],
    "mrl_window_cut": [_int, _i64, _i64, _i64, _vp, _vp, _i64, _vp, _int, _vp, _int, _vp, _vp, _vp, _vp, _vp],
    "mrl_window_logprob": [_vp, _int, _i64, _i64, _i64, _vp, _int, _f32, _int, _i64, _i64, _vp, _vp, _i64, _vp, _int, _vp,
                           _int, _int, _vp, _vp, _vp],
    "mrl_window_cells": [_int, _i64, _i64, _i64, _vp, _vp, _i64, _vp, _int, _vp, _int, _int, _vp, _vp, _vp, _vp, _vp, _vp],
    "mrl_generate_mask": [_vp, _int, _i64, _i64, _vp, _vp],
    "mrl_live_rows": [_vp, _int, _i64, _i64, _vp, _vp, _vp, _vp, _vp],
    "mrl_move_rows": [_vp, _i64, _vp, _vp, _i64, _vp, _vp, _i64, _vp, _vp, _int, _vp],
    "mrl_spread_scalars": [_vp, _i64, _int, _vp, _i64, _vp, _vp],
    "mrl_ragged_layouts": [_vp, _int, _vp],
    "mrl_ragged_columns": [_int, _vp, _int, _vp],
    "mrl_ragged_layout": [_vp, _int, _i64, _i64, _vp, _int, _i64, _int, _vp, _vp, _vp, _vp],
    "mrl_ragged_to_padded": [_vp, _int, _i64, _i64, _vp, _i64, _i64, ctypes.c_uint64, _vp, _vp],
    "mrl_padded_to_ragged": [_vp, _int, _i64, _i64, _vp, _int, _i64, _vp, _vp],
    "mrl_group_advantage": [_vp, _int, _i64, _i64, _vp, _int, _i64, _vp, _vp, _vp],
    "mrl_group_keep_mask": [_vp, _int, _i64, _i64, _vp, _vp],
    "mrl_policy_loss_fwd": [_vp, _vp, _vp, _vp, _vp, _vp, _int, _vp, _int, _i64, _i64, _f32, _f32, _int, _f32, _f32,
                            _int, _f32, _vp, _vp, _vp],
    "mrl_policy_loss_bwd": [_vp, _vp, _vp, _vp, _vp, _int, _vp, _int, _i64, _i64, _f32, _f32, _int, _f32, _f32, _int,
                            _f32, _vp, _vp, _vp, _vp, _vp, _vp],
    "mrl_fused_max_vocab": [_int],
    "mrl_fused_loss_prepare": [_int, _i64, _i64, _i64, _vp, _vp, _i64, _vp, _int, _vp, _int, _vp, _vp, _vp, _vp, _int,
                               _int, _vp, _vp, _vp, _vp, _vp, _i64, _vp, _f32, _vp, _vp],
    "mrl_fused_workspace_bytes": [_int, _i64, _i64],
    "mrl_fused_logprob_loss": [_vp, _int, _i64, _i64, _i64, _vp, _int, _f32, _vp, _int, _f32, _f32, _int, _f32, _f32,
                               _f32, _vp, _vp, _i64, _vp, _vp, _vp, _vp, _i64, _int, _vp],
    "mrl_fused_logprob_regrad": [_vp, _int, _i64, _i64, _i64, _vp, _int, _f32, _vp, _int, _f32, _f32, _int, _f32, _f32,
                                 _f32, _vp, _vp, _vp, _vp, _int, _vp, _i64, _vp, _i64, _int, _vp],
    "mrl_set_wide_spin_limit": [_i64],
    "mrl_fused_loss_reduce": [_vp, _vp, _vp, _i64, _i64, _vp, _vp, _vp, _vp, _int, _vp, _int, _f32, _f32, _int, _f32,
                              _f32, _int, _f32, _vp, _vp, _vp, _vp, _vp],
    "mrl_fused_loss_reduce_host": [_vp, _vp, _vp, _i64, _i64, _vp, _vp, _vp, _vp, _int, _vp, _int, _f32, _f32, _int, _f32,
                              _f32, _int, _f32, _vp, _vp, _vp, _vp, _vp, _vp],
    "mrl_scale_rows": [_vp, _int, _i64, _i64, _i64, _vp, _vp, _vp],
    "mrl_grad_scale_note": [_vp, _vp, _vp, _vp, _vp],
    "mrl_scale_rows_note": [_vp, _int, _i64, _i64, _i64, _vp, _vp, _vp, _vp, _vp],
    "mrl_lmhead_workspace_bytes": [_i64, _i64],
    "mrl_lmhead_logprob_fwd": [_vp, _vp, _i64, _i64, _i64, _vp, _int, _f32, _vp, _vp, _vp, _vp, _i64, _vp],
    "mrl_lmhead_logprob_fwd_cells": [_vp, _vp, _i64, _i64, _i64, _vp, _int, _f32, _vp, _vp, _vp, _vp, _i64, _vp],
    "mrl_lmhead_logits": [_vp, _vp, _i64, _i64, _i64, _vp, _i64, _vp],
    "mrl_lmhead_logprob_bwd": [_vp, _vp, _vp, _i64, _i64, _i64, _i64, _vp, _vp, _vp],
    "mrl_lmhead_bwd_workspace_bytes": [_i64, _i64, _i64],
    "mrl_lmhead_logprob_bwd_chunk": [_vp, _vp, _vp, _i64, _i64, _i64, _i64, _vp, _vp, _vp, _int, _int, _vp, _i64, _vp],
    "mrl_lmhead_static_max_tokens": [],
    "mrl_lmhead_logprob_fwd_static": [_vp, _vp, _i64, _i64, _i64, _vp, _int, _f32, _vp, _vp, _vp, _vp],
    "mrl_group_standardize": [_vp, _int, _i64, _i64, ctypes.c_double, _vp, _vp],
    "mrl_first_match": [_vp, _int, _i64, _i64, _i64, _int, _vp, _vp],
    "mrl_kl_token_rewards": [_vp, _vp, _vp, _int, _vp, _i64, _i64, _int, _f32, _vp, _vp, _vp],
    "mrl_gae_scan": [_vp, _vp, _i64, _i64, _f32, _f32, _vp, _vp, _vp],
    "mrl_gae_whiten_workspace_bytes": [_i64],
    "mrl_gae_whiten": [_vp, _vp, _vp, _int, _i64, _i64, _f32, _f32, _vp, _vp, _vp, _vp, _i64, _vp],
    "mrl_gae_whiten_host": [_vp, _vp, _vp, _int, _i64, _i64, _f32, _f32, _vp, _vp, _vp, _vp, _vp, _i64, _vp],
    "mrl_masked_whiten": [_vp, _vp, _int, _i64, _int, _vp, _vp, _vp],
    "mrl_value_loss_fwd": [_vp, _vp, _vp, _vp, _int, _vp, _int, _i64, _i64, _f32, _f32, _vp, _vp],
    "mrl_value_loss_workspace_bytes": [_i64],
    "mrl_value_loss_fwd_split": [_vp, _vp, _vp, _vp, _int, _vp, _int, _i64, _i64, _f32, _f32, _vp, _vp, _vp, _i64, _vp],
    "mrl_critic_loss_fwd_slope": [_vp, _i64, _i64, _vp, _int, _vp, _int, _vp, _vp, _i64, _f32, _f32, _vp, _vp, _vp, _vp, _i64, _vp],
    "mrl_critic_loss_fwd_slope_host": [_vp, _i64, _i64, _vp, _int, _vp, _int, _vp, _vp, _i64, _f32, _f32, _vp, _vp, _vp, _vp, _vp, _i64, _vp],
    "mrl_critic_loss_bwd_slope": [_vp, _i64, _i64, _vp, _int, _vp, _int, _i64, _f32, _vp, _vp, _vp, _vp],
    "mrl_value_loss_bwd": [_vp, _vp, _vp, _vp, _int, _vp, _int, _i64, _i64, _f32, _f32, _vp, _vp, _vp, _vp],
    "mrl_norm_fwd": [_vp, _int, _i64, _i64, _i64, _vp, _vp, _int, _int, _f32, _vp, _vp, _vp, _vp],
    "mrl_norm_bwd_workspace_bytes": [_i64, _i64],
    "mrl_norm_bwd": [_vp, _i64, _vp, _i64, _int, _i64, _i64, _vp, _int, _vp, _vp, _vp, _vp, _vp, _vp, _i64, _vp],
    "mrl_embedding_fwd": [_vp, _int, _i64, _i64, _vp, _int, _i64, _i64, _f32, _vp, _vp],
    "mrl_embedding_bwd_workspace_bytes": [_i64, _i64, _i64],
    "mrl_embedding_bwd": [_vp, _int, _i64, _i64, _vp, _int, _i64, _i64, _f32, _vp, _int, _int, _vp, _i64, _vp],
    "mrl_grad_norm": [_vp, _i64, _vp, _vp, _vp],
    "mrl_grad_clip": [_vp, _i64, _f32, _vp, _vp, _vp],
    "mrl_add_norm_fwd": [_vp, _int, _i64, _vp, _int, _i64, _i64, _i64, _vp, _int, _f32, _vp, _vp, _vp, _vp],
    "mrl_norm_fp8_fwd": [_vp, _int, _i64, _vp, _int, _i64, _i64, _i64, _vp, _int, _f32, _i64, _vp, _vp, _vp, _vp],
    "mrl_add_norm_bwd_workspace_bytes": [_i64, _i64],
    "mrl_add_norm_bwd": [_vp, _i64, _vp, _i64, _vp, _int, _int, _i64, _i64, _vp, _int, _vp, _vp, _vp, _vp, _vp, _i64, _vp],
    "mrl_rotary": [_vp, _vp, _int, _vp, _int, _i64, _i64, _i64, _i64, _vp, _i64, _int, _f32, _int, _vp],
    "mrl_adamw_step": [_vp, _i64, _int, _vp, _f64, _vp, _f64, _f64, _f64, _f64, _vp, _f32, _vp, _vp],
    "mrl_copy_bytes": [_vp, _vp, _i64, _vp],
    "mrl_bandwidth_probe": [_int, _vp, _vp, _i64, _i64, _vp],
}
_RESTYPES = {"mrl_last_error": ctypes.c_char_p, "mrl_fused_workspace_bytes": ctypes.c_int64, "mrl_fused_max_vocab": ctypes.c_int64,
             "mrl_lmhead_workspace_bytes": ctypes.c_int64, "mrl_lmhead_static_max_tokens": ctypes.c_int64,
             "mrl_set_wide_spin_limit": ctypes.c_int64, "mrl_gae_whiten_workspace_bytes": ctypes.c_int64,
             "mrl_value_loss_workspace_bytes": ctypes.c_int64, "mrl_lmhead_bwd_workspace_bytes": ctypes.c_int64,
             "mrl_norm_bwd_workspace_bytes": ctypes.c_int64, "mrl_add_norm_bwd_workspace_bytes": ctypes.c_int64,
             "mrl_embedding_bwd_workspace_bytes": ctypes.c_int64}

_lib = None
_entry = {}             # name -> bound function, looked up once


class MrlError(RuntimeError):
    """A libmrl_hip entry point returned a negative status."""

    def __init__(self, fn, code, message):
        super().__init__("%s failed (%d): %s" % (fn, code, message))
        self.code = code


def library_path():
    """The in-tree library; MRL_LIB_PATH points at another build of the same ABI (for experiments)."""
    return os.environ.get("MRL_LIB_PATH") or _build.LIB_PATH


def load():
    """Loads libmrl_hip.so once and declares every prototype.  Raises if it is not built."""
    global _lib
    if _lib is not None:
        return _lib
    path = library_path()
    if not os.path.exists(path):
        raise RuntimeError(
            "libmrl_hip.so is not built (%s missing): run `python -m mindspeed_rl_amd._build`; "
            "this package has no fallback path" % path)
    lib = ctypes.CDLL(path)
    for name, argtypes in SIGNATURES.items():
        fn = getattr(lib, name)       # AttributeError if the library lacks a declared symbol
        fn.argtypes = argtypes
        fn.restype = _RESTYPES.get(name, ctypes.c_int)
        _entry[name] = fn
    _lib = lib
    return lib


def call(name, *args):
    """Calls an entry point; a negative status becomes MrlError (ValueError-like codes included)."""
    if _lib is None:
        load()
    rc = _entry[name](*args)
    if rc != 0:
        raise MrlError(name, rc, _lib.mrl_last_error().decode("utf-8", "replace"))


def dtype_code(t):
    try:
        return _TORCH_DTYPE[t.dtype]
    except KeyError:
        raise TypeError("unsupported tensor dtype %s" % t.dtype) from None


@functools.lru_cache(maxsize=256)
def fused_workspace_bytes(dtype, n_rows, vocab):
    """mrl_fused_workspace_bytes: a function of its arguments alone."""
    return load().mrl_fused_workspace_bytes(dtype, n_rows, vocab)


def ptr(t):
    """Device pointer of a tensor (None -> NULL)."""
    return None if t is None else t.data_ptr()


# without the checks that the device has been initialised (a tensor on it is there) and other detours
_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device
_capturing = getattr(torch._C, "_cuda_isCurrentStreamCapturing", None) or torch.cuda.is_current_stream_capturing


def require_device(*tensors):
    """All given tensors (None skipped) must live on one HIP device; returns it."""
    dev = None
    for t in tensors:
        if t is None:
            continue
        if not t.is_cuda:
            raise RuntimeError("mindspeed_rl_amd runs on the GPU only: got a %s tensor (no CPU fallback exists)"
                               % t.device)
        if dev is None:
            dev = t.device
        elif t.device != dev:
            raise RuntimeError("tensors on different devices: %s and %s" % (dev, t.device))
    if dev is not None and dev.index is not None and dev.index != _current_device():
        # kernels are launched on the current device's context: one process drives one GPU here
        raise RuntimeError("tensors live on %s but the current device is cuda:%d (call torch.cuda.set_device first)"
                           % (dev, torch.cuda.current_device()))
    return dev


# the handle alone, without a Stream object around it (3 us of a call that takes 10); part of every torch that
# compiles for this device, and where it is not, the public way serves
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def stream(device):
    """Raw hipStream_t of torch's current stream on `device` (kernels are enqueued there)."""
    if _raw_stream is not None and device.index is not None:
        return _raw_stream(device.index)
    return torch.cuda.current_stream(device).cuda_stream


def dense(t, dtype, dev):
    """`t` as a contiguous tensor of `dtype` on `dev`; None stays None.  The usual case is that it is one already."""
    if t is None or (t.dtype is dtype and t.device == dev and t.is_contiguous()):
        return t
    return t.to(dev).to(dtype).contiguous()


def index_column(t, dev):
    """A length column as a dense int32 / int64 tensor on `dev`, flat unless it was dense already: what the kernels
    get is its address.  None stays None."""
    if t is None:
        return None
    if (t.dtype is torch.int64 or t.dtype is torch.int32) and t.is_contiguous() and t.device == dev:
        return t
    if t.dtype is not torch.int32 and t.dtype is not torch.int64:
        t = t.to(torch.int64)
    if t.device != dev:
        t = t.to(dev)
    return (t if t.dim() == 1 else t.reshape(-1)).contiguous()


# ------------------------------------------------------------------------------------ results for the host
class HostWords:
    """A slot of pinned host memory that a kernel leaves a few numbers in: the host watches it instead of copying
    from the device and waiting for the copy.  ``addr`` goes to the kernel as the address of its output, by ``launch``;
    one of the readers waits for the numbers, takes them and gives the slot back.  A slot that is never read, or not
    to its end, is not used again: a kernel may still write to it.  So its memory is not freed either."""

    BYTES = 4096
    _free = {}                  # device index -> slots that nothing writes to (list operations are atomic)
    _blocks = []                # all memory that slots lie in, as long as the process lives
    _BLOCK = 16                 # slots that are allocated together; there are as many as were ever taken at once
    _MOST_BLOCKS = 64           # 4 MiB; where they are all taken or lost, results are copied

    def __init__(self, f32, key):
        self.f32, self.addr, self._key = f32, f32.data_ptr(), key

    @classmethod
    def take(cls, dev, n_bytes):
        """An empty slot of ``n_bytes``, or None: more than a slot holds, no more slots, or the stream is being
        captured (the numbers will be there after a replay, not now)."""
        if n_bytes > cls.BYTES or _capturing():
            return None
        free = cls._free.setdefault(dev.index, [])
        try:
            slot = free.pop()
        except IndexError:
            if len(cls._blocks) >= cls._MOST_BLOCKS:
                return None
            block = torch.empty((cls._BLOCK, cls.BYTES // 4), dtype=torch.float32, pin_memory=True)
            cls._blocks.append(block)
            slot, *more = [cls(row, dev.index) for row in block.unbind(0)]
            free.extend(more)
        ctypes.memset(slot.addr, 0xff, n_bytes)
        return slot

    def launch(self, name, *args):
        """:func:`call` of an entry point that gets ``addr``.  One that refuses its arguments has launched nothing, and
        the slot goes back; what a failed launch leaves behind is not known."""
        try:
            call(name, *args)
        except Exception as e:
            if getattr(e, "code", None) != ERR_LAUNCH:
                self._free[self._key].append(self)
            raise

    def _arrived(self, n_bytes, stream):
        call("mrl_host_wait", self.addr, n_bytes // 4, stream)

    def read(self, ctype, n, stream):
        """``n`` numbers of a ctypes type, as a list."""
        kind = ctype * n
        self._arrived(ctypes.sizeof(kind), stream)
        values = kind.from_address(self.addr)[:]
        self._free[self._key].append(self)
        return values

    def read_doubles_of(self, n, stream):
        """``n`` fp32 numbers as a host tensor of doubles."""
        self._arrived(4 * n, stream)
        values = self.f32[:n].double()
        self._free[self._key].append(self)
        return values
