"""ctypes binding of libdynconv.so (the C ABI declared in include/dynconv.h).

The shared library is built in-tree (``python -m dynamic_conv1d_b200.build``) and
loaded from this directory.  There is no fallback: if the library is missing or
cannot be loaded, every op raises.
"""
from __future__ import annotations

import contextlib
import ctypes
import functools
import os
import threading

import torch
from torch.autograd import forward_ad

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "libdynconv.so")

DTYPE_BF16 = 0
DTYPE_F32 = 1
# added to the dtype: the norms' weights and scales, the gated delta rule's log decays and rates are float32
WEIGHTS_F32 = GATES_F32 = 256
_TORCH_DTYPES = {torch.bfloat16: DTYPE_BF16, torch.float32: DTYPE_F32}

_c_i64 = ctypes.c_int64
_c_int = ctypes.c_int
_c_vp = ctypes.c_void_p
_c_size = ctypes.c_size_t

_SIGNATURES = {
    "dynconv_abi_version": (_c_int, []),
    "dynconv_status_string": (ctypes.c_char_p, [_c_int]),
    "dynconv_last_error": (ctypes.c_char_p, []),
    "dynconv_check_device": (_c_int, [_c_vp]),
    "dynconv_launch_count": (ctypes.c_uint64, []),
    "dynconv_hw_fwd": (_c_int, [_c_vp] * 4 + [_c_i64] * 5 + [_c_int, _c_int, _c_vp]),
    "dynconv_hw_bwd_workspace_bytes": (_c_size, [_c_i64] * 5 + [_c_int, _c_int]),
    "dynconv_hw_bwd": (_c_int, [_c_vp] * 8 + [_c_vp, _c_size] + [_c_i64] * 5 + [_c_int, _c_int, _c_vp]),
    "dynconv_lr_fwd_workspace_bytes": (_c_size, [_c_i64] * 5 + [_c_int, _c_int]),
    "dynconv_lr_fwd": (_c_int, [_c_vp] * 5 + [_c_vp, _c_size] + [_c_i64] * 5 + [_c_int, _c_int, _c_vp]),
    "dynconv_lr_fwd_noalloc": (_c_int, [_c_vp] * 5 + [_c_i64] * 5 + [_c_int, _c_int, _c_vp]),
    "dynconv_lr_bwd_workspace_bytes": (_c_size, [_c_i64] * 5 + [_c_int, _c_int]),
    "dynconv_lr_bwd": (_c_int, [_c_vp] * 10 + [_c_vp, _c_size] + [_c_i64] * 5 + [_c_int, _c_int, _c_vp]),
    "dynconv_lr_fwd_grouped_workspace_bytes": (_c_size, [_c_i64] * 6 + [_c_int, _c_int]),
    "dynconv_lr_fwd_grouped": (_c_int, [_c_vp] * 5 + [_c_vp, _c_size] + [_c_i64] * 6 + [_c_int, _c_int, _c_vp]),
    "dynconv_lr_bwd_grouped_workspace_bytes": (_c_size, [_c_i64] * 6 + [_c_int, _c_int]),
    "dynconv_lr_bwd_grouped": (_c_int, [_c_vp] * 10 + [_c_vp, _c_size] + [_c_i64] * 6 + [_c_int, _c_int, _c_vp, _c_vp]),
    "dynconv_comm_blob_bytes": (_c_size, []),
    "dynconv_comm_create": (_c_int, [_c_int, _c_int, _c_i64, ctypes.POINTER(_c_vp), _c_vp]),
    "dynconv_comm_connect": (_c_int, [_c_vp, _c_vp]),
    "dynconv_comm_destroy": (_c_int, [_c_vp]),
    "dynconv_lr_bwd_grouped_dp": (_c_int, [_c_vp] * 10 + [_c_vp, _c_size] + [_c_i64] * 6
                                  + [_c_int, _c_int, _c_vp, _c_vp, _c_vp]),
    "dynconv_lr_step": (_c_int, [_c_vp] * 7 + [_c_int] + [_c_i64] * 6 + [_c_int, _c_int, _c_vp]),
    "dynconv_hw_step": (_c_int, [_c_vp] * 6 + [_c_int] + [_c_i64] * 5 + [_c_int, _c_int, _c_vp]),
    "dynconv_la_workspace_bytes": (_c_size, [_c_i64] * 5 + [_c_int, _c_int]),
    "dynconv_la_fwd": (_c_int, [_c_vp] * 8 + [_c_vp, _c_size] + [_c_i64] * 5 + [ctypes.c_float, _c_int, _c_vp]),
    "dynconv_la_bwd": (_c_int, [_c_vp] * 12 + [_c_vp, _c_size] + [_c_i64] * 5 + [ctypes.c_float, _c_int, _c_vp]),
    "dynconv_la_step": (_c_int, [_c_vp] * 7 + [_c_int, _c_vp] + [_c_i64] * 5 + [ctypes.c_float, _c_int, _c_vp]),
    "dynconv_delta_kept_bytes": (_c_size, [_c_i64] * 5 + [_c_int]),
    "dynconv_delta_fwd": (_c_int, [_c_vp] * 9 + [_c_size, _c_vp, _c_vp, _c_size] + [_c_i64] * 5 + [ctypes.c_float, _c_int, _c_vp]),
    "dynconv_delta_workspace_bytes": (_c_size, [_c_i64] * 5 + [_c_int] * 2),
    "dynconv_delta_bwd": (_c_int, [_c_vp] * 5 + [_c_size] + [_c_vp] * 10 + [_c_size] + [_c_i64] * 5
                          + [ctypes.c_float, _c_int, _c_vp]),
    "dynconv_delta_step": (_c_int, [_c_vp] * 8 + [_c_int, _c_vp] + [_c_i64] * 5 + [ctypes.c_float, _c_int, _c_vp]),
    "dynconv_norm_workspace_bytes": (_c_size, [_c_i64]),
    "dynconv_gated_norm_fwd": (_c_int, [_c_vp] * 5 + [_c_i64] * 3 + [ctypes.c_float] * 2 + [_c_int, _c_vp]),
    "dynconv_gated_norm_bwd": (_c_int, [_c_vp] * 9 + [_c_size] + [_c_i64] * 3 + [ctypes.c_float] * 2 + [_c_int, _c_vp]),
    "dynconv_residual_norm_fwd": (_c_int, [_c_vp] * 4 + [ctypes.c_float] + [_c_vp] * 2 + [_c_i64] * 2
                                  + [ctypes.c_float, _c_int, _c_vp]),
    "dynconv_residual_norm_bwd": (_c_int, [_c_vp] * 4 + [ctypes.c_float] + [_c_vp] * 7 + [_c_size] + [_c_i64] * 2
                                  + [ctypes.c_float, _c_int, _c_vp]),
    "dynconv_vocab_loss_fwd_workspace_bytes": (_c_size, [_c_i64] * 3 + [_c_int]),
    "dynconv_vocab_loss_fwd": (_c_int, [_c_vp] * 7 + [_c_size] + [_c_i64] * 4 + [_c_int, _c_int, _c_vp]),
    "dynconv_vocab_loss_bwd_workspace_bytes": (_c_size, [_c_i64] * 3 + [_c_int] * 3),
    "dynconv_vocab_loss_bwd": (_c_int, [_c_vp] * 9 + [_c_size] + [_c_i64] * 4 + [_c_int, _c_int, _c_vp]),
    "dynconv_cast_f32": (_c_int, [_c_vp, _c_vp, _c_i64, _c_int, _c_vp]),
    "dynconv_umma_selftest": (_c_int, [_c_vp, _c_vp, _c_vp] + [_c_int] * 12 + [_c_vp]),
    "dynconv_wait_selftest": (_c_int, [ctypes.c_uint64, _c_vp, _c_vp]),
}

EXPORTED_SYMBOLS = tuple(_SIGNATURES)

_lock = threading.Lock()
_lib = None


class DynconvError(RuntimeError):
    """A libdynconv entry point returned a non-zero status."""

    def __init__(self, status: int, message: str):
        super().__init__(message)
        self.status = status


def load() -> ctypes.CDLL:
    """Load libdynconv.so (once) and declare its prototypes."""
    global _lib
    if _lib is not None:
        return _lib
    with _lock:
        if _lib is None:
            if not os.path.exists(LIB_PATH):
                raise RuntimeError(
                    f"{LIB_PATH} is missing: build it with `python -m dynamic_conv1d_b200.build` "
                    "(there is no CPU or non-CUDA fallback)"
                )
            lib = ctypes.CDLL(LIB_PATH)
            for name, (res, args) in _SIGNATURES.items():
                fn = getattr(lib, name)
                fn.restype = res
                fn.argtypes = args
            if lib.dynconv_abi_version() != 1:
                raise RuntimeError("libdynconv ABI version mismatch")
            _lib = lib
    return _lib


def check(status: int) -> None:
    if status != 0:
        lib = load()
        msg = lib.dynconv_last_error().decode(errors="replace")
        kind = lib.dynconv_status_string(status).decode()
        raise DynconvError(status, f"libdynconv: {kind}: {msg}")


def dtype_code(dtype: torch.dtype) -> int:
    try:
        return _TORCH_DTYPES[dtype]
    except KeyError:
        raise TypeError(f"dynamic convolution supports bfloat16 and float32 tensors, got {dtype}") from None


def on_device(fn):
    """Runs an autograd forward/backward with its first tensor's device current:
    the library launches on the current device, the stream comes from the tensor."""

    @functools.wraps(fn)
    def wrapper(ctx, first, *args):
        with device_of(first):
            return fn(ctx, first, *args)

    return wrapper


class _NoSecondDerivative(torch.autograd.Function):
    """Gradients as they are; differentiating them is an error."""

    @staticmethod
    def forward(ctx, *grads):
        return tuple(g.view_as(g) for g in grads)

    @staticmethod
    def backward(ctx, *_):
        raise RuntimeError("this operator's gradients cannot be differentiated again (create_graph=True)")


def differentiable_once(backward):
    """Decorator of a Function's backward whose kernels autograd does not see.  Under create_graph=True
    its gradients would come back as constants and a penalty on them would be left out without a word;
    here differentiating them raises.  (torch's once_differentiable does so only where the upstream gradient
    asks for a gradient itself, but these depend on the saved inputs too.)"""

    @functools.wraps(backward)
    def wrapper(ctx, *upstream):
        if not torch.is_grad_enabled():
            return backward(ctx, *upstream)
        with torch.no_grad():
            grads = backward(ctx, *upstream)
        there = [i for i, g in enumerate(grads) if g is not None]
        marked = _NoSecondDerivative.apply(*(grads[i].requires_grad_() for i in there))
        out = [None] * len(grads)
        for i, g in zip(there, marked):
            out[i] = g
        return tuple(out)

    return wrapper


_is_tracing = torch._C._is_tracing if hasattr(torch._C, "_is_tracing") else torch.jit.is_tracing
_says_level = hasattr(forward_ad, "_current_level")


def watched() -> bool:
    """Whether somebody watches a call who asks for no gradient: inside a level of forward-mode differentiation,
    whose tangents a direct call of the library would drop, or under torch.jit.trace, which would record the
    allocation of the outputs alone.  Such calls go through their autograd Function, which refuses tangents and is
    recorded as a whole, or are refused."""
    return not _says_level or forward_ad._current_level >= 0 or _is_tracing()


_same_device = contextlib.nullcontext()
# the bindings under torch.cuda.current_device / current_stream, without the Python objects, for
# calls whose kernels take a few microseconds
current_device = torch._C._cuda_getDevice if hasattr(torch._C, "_cuda_getDevice") else torch.cuda.current_device
raw_stream_of = torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream") else None


def device_of(t: torch.Tensor):
    """Context in which t's device is current (free when it already is)."""
    if t.get_device() == current_device():
        return _same_device
    return torch.cuda.device(t.device)


def raw_stream(t: torch.Tensor) -> int:
    """The current stream of t's device as an address."""
    return raw_stream_of(t.get_device())


def ptr(t: torch.Tensor | None):
    return None if t is None else ctypes.c_void_p(t.data_ptr())


def stream_of(t: torch.Tensor):
    return ctypes.c_void_p(torch.cuda.current_stream(t.device).cuda_stream)


def check_device(t: torch.Tensor) -> None:
    """Synchronise the current stream and raise if a device-side bounded wait gave up."""
    check(load().dynconv_check_device(stream_of(t)))


_sync_checks = os.environ.get("DYNCONV_SYNC_CHECK", "0") not in ("", "0")


def set_sync_checks(enabled: bool) -> None:
    """Debug mode (also DYNCONV_SYNC_CHECK=1 in the environment): every forward and
    backward call synchronises its stream and raises DynconvError(DYNCONV_ERR_TIMEOUT)
    at the call whose kernel gave up a bounded wait.  Off by default: the normal path
    never synchronises, and a timed-out kernel is reported by the next check_device()."""
    global _sync_checks
    _sync_checks = bool(enabled)


def after_call(t: torch.Tensor) -> None:
    """Called by the ops after their launches; checks the device only in debug mode
    (and never while the stream is being captured into a CUDA graph)."""
    if _sync_checks and not torch.cuda.is_current_stream_capturing():
        check_device(t)
