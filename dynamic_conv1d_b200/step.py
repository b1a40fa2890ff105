"""The dynamic convolutions for one token at a time, on a cache of each sequence's last
W-1 inputs (libdynconv's ``dynconv_lr_step`` / ``dynconv_hw_step``).

A prompt runs through the whole-sequence ops; ``convolution_cache(x, W)`` keeps its last
W-1 inputs, and each step takes one token per sequence, updating the cache in place:

    y = lowrank_dynamic_convolution(x, z, U, static_w, residual=True)      # the prompt
    cache = convolution_cache(x, W)
    y_t = lowrank_dynamic_convolution_step(x_t, z_t, U, cache, static_w, residual=True)

The steps have no gradient (generating text needs none) and refuse inputs that ask for one.
"""
from __future__ import annotations

import torch

from . import _lib


def _no_grad_wanted(*tensors) -> None:
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError("a single-token step has no gradient: call it under torch.no_grad()")


def _slots(slots: torch.Tensor | None, B: int):
    """(pointer, bytes of an index) of a slot table."""
    if slots is None:
        return None, 0
    assert slots.is_cuda and slots.is_contiguous() and slots.shape == (B,)
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
    assert x.is_cuda and x.is_contiguous() and x.dim() == 2
    assert z.is_cuda and z.is_contiguous() and z.dim() == 2 and z.shape[0] == x.shape[0]
    assert U.is_cuda and U.is_contiguous() and U.dim() == 3
    B, C = x.shape
    G, R, WD = U.shape
    assert C % G == 0 and z.shape[1] == G * R
    D = C // G
    assert WD % D == 0, "U must be [G, R, W*D]"
    return _lowrank_step(x, z, U, cache, static_w, residual, slots, B, D, R, WD // D, G)


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
    assert x.is_cuda and x.is_contiguous() and x.dim() == 2
    assert z.is_cuda and z.is_contiguous() and z.dim() == 2 and z.shape[0] == x.shape[0]
    assert U.is_cuda and U.is_contiguous() and U.dim() == 2
    B, D = x.shape
    R, WD = U.shape
    assert z.shape[1] == R
    assert WD % D == 0, "U must be [R, W*D]"
    return _lowrank_step(x, z, U, cache, static_w, residual, slots, B, D, R, WD // D, 1)


def _check_cache(x, cache, W, slots):
    assert cache.is_cuda and cache.is_contiguous() and cache.dtype == x.dtype
    assert cache.dim() == 3 and cache.shape[1:] == (W - 1, x.shape[1])
    assert slots is not None or cache.shape[0] >= x.shape[0]


def _lowrank_step(x, z, U, cache, static_w, residual, slots, B, D, R, W, G):
    _check_cache(x, cache, W, slots)
    if static_w is not None:
        assert static_w.is_cuda and static_w.is_contiguous()
        assert static_w.shape == ((W, D) if U.dim() == 2 else (G, W, D))
    _no_grad_wanted(x, z, U, static_w)
    code = _lib.dtype_code(x.dtype)
    # parameters of another dtype are cast for the call, as by the whole-sequence op
    if z.dtype != x.dtype:
        z = z.to(x.dtype)
    if U.dtype != x.dtype:
        U = U.to(x.dtype)
    if static_w is not None and static_w.dtype != x.dtype:
        static_w = static_w.to(x.dtype)
    sp, sb = _slots(slots, B)
    y = torch.empty_like(x)
    with _lib.device_of(x):
        _lib.check(
            _lib.load().dynconv_lr_step(
                x.data_ptr(), z.data_ptr(), U.data_ptr(), None if static_w is None else static_w.data_ptr(),
                cache.data_ptr(), y.data_ptr(), sp, sb, B, cache.shape[0], D, R, W, G, code, int(bool(residual)),
                _lib.raw_stream(x),
            )
        )
        _lib.after_call(y)
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
    assert x.is_cuda and x.is_contiguous() and x.dim() == 2
    assert weight.is_cuda and weight.dim() == 3 and weight.shape[0] == x.shape[0]
    B, D = x.shape
    H, W = weight.shape[1:]
    assert D % H == 0, f"D={D} must be divisible by H={H}"
    _check_cache(x, cache, W, slots)
    if static_w is not None:
        assert static_w.is_cuda and static_w.is_contiguous()
        assert static_w.dtype == x.dtype
        assert static_w.shape == (W, D)
    _no_grad_wanted(x, weight, static_w)
    code = _lib.dtype_code(x.dtype)
    weight = weight.to(dtype=x.dtype).contiguous()
    sp, sb = _slots(slots, B)
    y = torch.empty_like(x)
    with _lib.device_of(x):
        _lib.check(
            _lib.load().dynconv_hw_step(
                x.data_ptr(), weight.data_ptr(), None if static_w is None else static_w.data_ptr(),
                cache.data_ptr(), y.data_ptr(), sp, sb, B, cache.shape[0], D, H, W, code, int(bool(residual)),
                _lib.raw_stream(x),
            )
        )
        _lib.after_call(y)
    return y
