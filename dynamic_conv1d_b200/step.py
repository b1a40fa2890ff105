"""The dynamic convolutions for one token at a time, on a cache of each sequence's last
W-1 inputs (libdynconv's ``dynconv_lr_step`` / ``dynconv_hw_step``).

A prompt runs through the whole-sequence ops; ``convolution_cache(x, W)`` keeps its last
W-1 inputs, and each step takes one token per sequence, updating the cache in place:

    y = lowrank_dynamic_convolution(x, z, U, static_w, residual=True)      # the prompt
    cache = convolution_cache(x, W)
    y_t = lowrank_dynamic_convolution_step(x_t, z_t, U, cache, static_w, residual=True)

The steps have no gradient (generating text needs none) and refuse inputs that ask for one.  They
count as updates in place of the cache: a backward that kept it before a step raises.
"""
from __future__ import annotations

import torch
from torch.autograd.graph import increment_version

from . import _lib


def _refuse_gradient():
    raise RuntimeError("a single-token step has no gradient: call it under torch.no_grad()")


def _refuse_watched(*tensors):
    """For a call that is watched (``_lib.watched``): it may go on where no tensor has a tangent and no trace is taken."""
    if any(t is not None and torch.autograd.forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        _refuse_gradient()
    if torch.jit.is_tracing():
        raise RuntimeError("a single-token step cannot be traced: the trace would not hold what the step updates")


def _slots(slots: torch.Tensor, B: int, dev: int):
    """(pointer, bytes of an index) of a slot table on device `dev`."""
    assert slots.get_device() == dev and slots.is_contiguous() and slots.shape == (B,)
    assert slots.dtype in (torch.int32, torch.int64), "slots must be int32 or int64"
    return slots.data_ptr(), slots.element_size()


def convolution_cache(x: torch.Tensor, W: int) -> torch.Tensor:
    """The cache of the single-token steps after a prompt: the last W-1 inputs of
    x [B, T, C], oldest first, with zeros where T < W-1.  A fresh tensor [B, W-1, C]."""
    B, T, C = x.shape
    cache = x.new_zeros(B, W - 1, C)
    n = min(T, W - 1)
    if n > 0:
        cache[:, W - 1 - n:] = x[:, T - n:].detach()
    return cache


def lowrank_dynamic_convolution_grouped_step(
    x: torch.Tensor,
    z: torch.Tensor,
    U: torch.Tensor,
    cache: torch.Tensor,
    static_w: torch.Tensor | None = None,
    residual: bool = False,
    slots: torch.Tensor | None = None,
) -> torch.Tensor:
    """One token of G low-rank convolutions (``lowrank_dynamic_convolution_grouped``).

    Args:
        x:        [B, G*D] the sequences' inputs (bfloat16 or float32, CUDA, contiguous).
        z:        [B, G*R], U: [G, R, W*D], static_w: [G, W, D] or None.
        cache:    [n, W-1, G*D] in x's dtype, oldest input first; updated in place.
        residual: add x to the output.
        slots:    [B] int32 or int64, each sequence's row of the cache, none twice; rows
                  outside 0..n-1 touch no cache and give zeros.  None: row b (n >= B).

    Returns:
        y: [B, G*D].
    """
    assert U.dim() == 3
    G, R, WD = U.shape
    return _lowrank_step(x, z, U, cache, static_w, residual, slots, R, WD, G)


def lowrank_dynamic_convolution_step(
    x: torch.Tensor,
    z: torch.Tensor,
    U: torch.Tensor,
    cache: torch.Tensor,
    static_w: torch.Tensor | None = None,
    residual: bool = False,
    slots: torch.Tensor | None = None,
) -> torch.Tensor:
    """One token of ``lowrank_dynamic_convolution``: x [B, D], z [B, R], U [R, W*D],
    static_w [W, D], cache [n, W-1, D].  See ``lowrank_dynamic_convolution_grouped_step``."""
    assert U.dim() == 2
    R, WD = U.shape
    return _lowrank_step(x, z, U, cache, static_w, residual, slots, R, WD, 1)


def _check_cache(cache, dev, dtype, B, W, C, slots):
    """Rows of the cache."""
    assert cache.get_device() == dev and cache.is_contiguous() and cache.dtype == dtype and cache.dim() == 3
    n, rows, channels = cache.shape
    assert rows == W - 1 and channels == C, f"cache must be [n, {W - 1}, {C}]"
    assert slots is not None or n >= B
    return n


def _lowrank_step(x, z, U, cache, static_w, residual, slots, R, WD, G):
    dev = x.get_device()  # (-1 on the CPU)
    assert dev >= 0 and x.is_contiguous() and x.dim() == 2
    assert z.get_device() == dev and z.is_contiguous()
    assert U.get_device() == dev and U.is_contiguous()
    B, C = x.shape
    D = C // G
    assert D * G == C and z.shape == (B, G * R)
    W = WD // D
    assert W * D == WD, "U must be [G, R, W*D]"
    dtype = x.dtype
    n = _check_cache(cache, dev, dtype, B, W, C, slots)
    if static_w is not None:
        assert static_w.get_device() == dev and static_w.is_contiguous()
        assert static_w.shape == ((W, D) if U.dim() == 2 else (G, W, D))
        if static_w.dtype != dtype:
            static_w = static_w.to(dtype)
    if torch.is_grad_enabled() and (x.requires_grad or z.requires_grad or U.requires_grad or cache.requires_grad
                                    or (static_w is not None and static_w.requires_grad)):
        _refuse_gradient()
    if _lib.watched():
        _refuse_watched(x, z, U, cache, static_w)
    code = _lib.dtype_code(dtype)
    # parameters of another dtype are cast for the call, as by the whole-sequence op
    if z.dtype != dtype:
        z = z.to(dtype)
    if U.dtype != dtype:
        U = U.to(dtype)
    sp, sb = (None, 0) if slots is None else _slots(slots, B, dev)
    y = torch.empty_like(x)
    with _lib.device_of(x):
        status = _lib.load().dynconv_lr_step(
            x.data_ptr(), z.data_ptr(), U.data_ptr(), None if static_w is None else static_w.data_ptr(),
            cache.data_ptr(), y.data_ptr(), sp, sb, B, n, D, R, W, G, code, 1 if residual else 0, _lib.raw_stream(x))
        if status:
            _lib.check(status)
        _lib.after_call(y)
    increment_version(cache)
    return y


def headwise_dynamic_convolution_step(
    x: torch.Tensor,
    weight: torch.Tensor,
    cache: torch.Tensor,
    static_w: torch.Tensor | None = None,
    residual: bool = False,
    slots: torch.Tensor | None = None,
) -> torch.Tensor:
    """One token of ``headwise_dynamic_convolution``: x [B, D], weight [B, H, W],
    static_w [W, D], cache [n, W-1, D] (updated in place), slots as for
    ``lowrank_dynamic_convolution_grouped_step``.  Returns y [B, D]."""
    dev = x.get_device()
    assert dev >= 0 and x.is_contiguous() and x.dim() == 2
    assert weight.get_device() == dev and weight.dim() == 3 and weight.shape[0] == x.shape[0]
    B, D = x.shape
    H, W = weight.shape[1:]
    assert D % H == 0, f"D={D} must be divisible by H={H}"
    dtype = x.dtype
    n = _check_cache(cache, dev, dtype, B, W, D, slots)
    if static_w is not None:
        assert static_w.get_device() == dev and static_w.is_contiguous()
        assert static_w.dtype == dtype
        assert static_w.shape == (W, D)
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or cache.requires_grad
                                    or (static_w is not None and static_w.requires_grad)):
        _refuse_gradient()
    if _lib.watched():
        _refuse_watched(x, weight, cache, static_w)
    code = _lib.dtype_code(dtype)
    if weight.dtype != dtype or not weight.is_contiguous():
        weight = weight.to(dtype=dtype).contiguous()
    sp, sb = (None, 0) if slots is None else _slots(slots, B, dev)
    y = torch.empty_like(x)
    with _lib.device_of(x):
        status = _lib.load().dynconv_hw_step(
            x.data_ptr(), weight.data_ptr(), None if static_w is None else static_w.data_ptr(),
            cache.data_ptr(), y.data_ptr(), sp, sb, B, n, D, H, W, code, 1 if residual else 0, _lib.raw_stream(x))
        if status:
            _lib.check(status)
        _lib.after_call(y)
    increment_version(cache)
    return y
