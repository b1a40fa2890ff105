"""Root-mean-square norms fused with what stands next to them in a layer (libdynconv's
``dynconv_gated_norm_*`` and ``dynconv_residual_norm_*``).

``gated_rms_norm`` normalises rows under a gate, one row per head; without weight and gate it is
the normalisation of queries and keys.  ``residual_rms_norm`` adds a block's output to the residual
stream and gives the next block its norm.  Sums are float32; the sums over rows behind the gradients
of weights are added in a fixed order.  Weights may be float32 beside bfloat16 rows, and so are their gradients then.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from .linear_attention import _ptr

_Strides4 = ctypes.c_int64 * 4


def _rows(t: torch.Tensor):
    """t [..., D] as rows (n, g) with one stride each, dense in D: (t, N, G, outer, inner).  Copied
    where its leading dimensions do not fold into two."""
    D = t.shape[-1]
    if t.is_contiguous():
        n = t.numel() // D if D else 0
        return t, n, 1, D, 0
    if t.stride(-1) == 1 or D == 1:
        # fold from the right: dimensions whose strides continue one another
        dims = [(n, s) for n, s in zip(t.shape[:-1], t.stride()[:-1]) if n != 1]
        folded = []
        for n, s in reversed(dims):
            if folded and s == folded[-1][0] * folded[-1][1]:
                folded[-1] = (folded[-1][0] * n, folded[-1][1])
            else:
                folded.append((n, s))
        if len(folded) <= 2 and t.numel():
            folded += [(1, 0)] * (2 - len(folded))
            (g, inner), (n, outer) = folded
            return t, n, g, outer, inner
    t = t.contiguous()
    return t, t.numel() // D if D else 0, 1, D, 0


def _pair(x, gate):
    """x and gate over the same split of their rows: (x, gate, N, G, strides)."""
    if x.is_contiguous() and (gate is None or gate.is_contiguous()):
        D = x.shape[-1]
        return x, gate, x.numel() // D if D else 0, 1, _Strides4(D, 0, D, 0)
    x, n, g, xo, xi = _rows(x)
    if gate is None:
        return x, None, n, g, _Strides4(xo, xi, 0, 0)
    gate, m, h, go, gi = _rows(gate)
    if g != h:  # one of them is a single run of rows: cut it like the other
        if g == 1:
            n, g, xo, xi = m, h, xo * h, xo
        elif h == 1:
            go, gi = go * g, go
        else:
            x, gate = x.contiguous(), gate.contiguous()
            n, g, xo, xi, go, gi = n * g, 1, x.shape[-1], 0, x.shape[-1], 0
    return x, gate, n, g, _Strides4(xo, xi, go, gi)


def _sum_workspace(lib, like, D, sums):
    n = lib.dynconv_norm_workspace_bytes(D) * sums
    return (torch.empty(n, device=like.device, dtype=torch.uint8), n) if n else (None, 0)


def _code(like, weight):
    code = _lib.dtype_code(like.dtype)
    return code if weight is None or weight.dtype == like.dtype else code + _lib.WEIGHTS_F32


def _gated_forward(x, weight, gate, eps, scale):
    x, gate, n, g, strides = _pair(x, gate)
    lib = _lib.load()
    code = _code(x, weight)
    with _lib.device_of(x):
        y = x.new_empty(x.shape)
        status = lib.dynconv_gated_norm_fwd(x.data_ptr(), _ptr(weight), _ptr(gate), y.data_ptr(), strides, n, g, x.shape[-1],
                                            eps, scale, code, _lib.raw_stream(x))
        if status:
            _lib.check(status)
        _lib.after_call(y)
    return y


class _GatedRmsNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, gate, eps, scale):
        ctx.save_for_backward(x, weight, gate)
        ctx.args = (eps, scale)
        return _gated_forward(x, weight, gate, eps, scale)

    @staticmethod
    @_lib.differentiable_once
    def backward(ctx, dy):
        x, weight, gate = ctx.saved_tensors
        eps, scale = ctx.args
        x, gate, n, g, strides = _pair(x, gate)
        lib = _lib.load()
        code = _code(x, weight)
        with _lib.device_of(x):
            dy = dy.contiguous()
            want_x, want_w, want_g = ctx.needs_input_grad[:3]
            dx = x.new_empty(x.shape) if want_x else None
            dg = x.new_empty(x.shape) if want_g else None
            dw = torch.empty_like(weight) if want_w else None
            ws, nbytes = _sum_workspace(lib, x, x.shape[-1], 1) if want_w else (None, 0)
            status = lib.dynconv_gated_norm_bwd(
                x.data_ptr(), _ptr(weight), _ptr(gate), dy.data_ptr(), _ptr(dx), _ptr(dw), _ptr(dg), strides, _ptr(ws), nbytes,
                n, g, x.shape[-1], eps, scale, code, _lib.raw_stream(x))
            if status:
                _lib.check(status)
            _lib.after_call(x)
        return dx, dw, dg, None, None


def _check_weight(weight, x, name="weight"):
    assert weight.get_device() == x.get_device() and weight.is_contiguous() and weight.shape == x.shape[-1:], f"{name} must be [{x.shape[-1]}]"
    return weight if weight.dtype == x.dtype else weight.float()


def gated_rms_norm(
    x: torch.Tensor,
    weight: torch.Tensor | None = None,
    gate: torch.Tensor | None = None,
    eps: float = 1e-6,
    scale: float = 1.0,
) -> torch.Tensor:
    """scale * x * rsqrt(mean(x^2) + eps) * weight * silu(gate), over the last dimension.

    Args:
        x:      [..., D] (bfloat16 or float32, CUDA), D <= 16384; views of a fused projection are read in place.
        weight: [D] or None, in x's dtype or float32 (its gradient likewise); cast to float32 when it has another one.
        gate:   of x's shape and dtype, or None.
        scale:  a number; D**-0.5 without weight and gate gives rows of length one.

    Returns:
        a tensor of x's shape, contiguous.  Differentiable (once) in x, weight and gate.
    """
    assert x.is_cuda and x.dim() >= 1
    if weight is not None:
        weight = _check_weight(weight, x)
    if gate is not None:
        assert gate.get_device() == x.get_device() and gate.shape == x.shape and gate.dtype == x.dtype
    eps, scale = float(eps), float(scale)
    if (torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad)
                                     or (gate is not None and gate.requires_grad))) or _lib.watched():
        return _GatedRmsNormFn.apply(x, weight, gate, eps, scale)
    return _gated_forward(x, weight, gate, eps, scale)


def _residual_forward(x, residual, weight, scale, factor, eps):
    lib = _lib.load()
    code = _code(x, weight)
    D = x.shape[-1]
    with _lib.device_of(x):
        y, h = torch.empty_like(x), torch.empty_like(x)
        status = lib.dynconv_residual_norm_fwd(
            x.data_ptr(), residual.data_ptr(), weight.data_ptr(), _ptr(scale), factor, y.data_ptr(), h.data_ptr(),
            x.numel() // D if D else 0, D, eps, code, _lib.raw_stream(x))
        if status:
            _lib.check(status)
        _lib.after_call(y)
    return y, h


class _ResidualRmsNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, scale, factor, eps):
        y, h = _residual_forward(x, residual, weight, scale, factor, eps)
        # (x is kept for the gradient of a scale per channel alone)
        ctx.save_for_backward(h, x if scale is not None and scale.requires_grad else None, weight, scale)
        ctx.args = (factor, eps)
        ctx.set_materialize_grads(False)
        return y, h

    @staticmethod
    @_lib.differentiable_once
    def backward(ctx, dy, dh):
        h, x, weight, scale = ctx.saved_tensors
        factor, eps = ctx.args
        D = h.shape[-1]
        lib = _lib.load()
        code = _code(h, weight)
        with _lib.device_of(h):
            dy = None if dy is None else dy.contiguous()
            dh = None if dh is None else dh.contiguous()
            want_x, want_r, want_w, want_s = ctx.needs_input_grad[:4]
            dx = torch.empty_like(h) if want_x else None
            dr = torch.empty_like(h) if want_r else None
            dw = torch.empty_like(weight) if want_w else None
            ds = torch.empty_like(scale) if want_s else None
            ws, nbytes = _sum_workspace(lib, h, D, int(want_w) + int(want_s))
            status = lib.dynconv_residual_norm_bwd(
                h.data_ptr(), _ptr(x), weight.data_ptr(), _ptr(scale), factor, _ptr(dy), _ptr(dh), _ptr(dx), _ptr(dr), _ptr(dw),
                _ptr(ds), _ptr(ws), nbytes, h.numel() // D if D else 0, D, eps, code,
                _lib.raw_stream(h))
            if status:
                _lib.check(status)
            _lib.after_call(h)
        return dx, dr, dw, ds, None, None


def residual_rms_norm(
    x: torch.Tensor,
    residual: torch.Tensor,
    weight: torch.Tensor,
    scale: torch.Tensor | float = 1.0,
    eps: float = 1e-6,
) -> tuple[torch.Tensor, torch.Tensor]:
    """The residual stream after a block, and its norm for the next one:

        h = residual + scale * x,   y = h * rsqrt(mean(h^2) + eps) * weight

    Args:
        x, residual: [..., D] (bfloat16 or float32, CUDA, contiguous), D <= 16384.
        weight:      [D]; scale: a number, or [D].  In x's dtype or float32 (their gradients likewise); cast to
                     float32 when one has another, or when the other is float32.

    Returns:
        (y, h), both of x's shape; y is the norm of the sum before it is rounded to x's dtype.
        Differentiable (once) in x, residual, weight and scale.
    """
    assert x.is_cuda and x.is_contiguous() and x.dim() >= 1
    assert residual.get_device() == x.get_device() and residual.is_contiguous() and residual.shape == x.shape
    assert residual.dtype == x.dtype
    weight = _check_weight(weight, x)
    factor = 1.0
    if isinstance(scale, torch.Tensor):
        scale = _check_weight(scale, x, "scale")
        if scale.dtype != weight.dtype:
            weight, scale = weight.float(), scale.float()
    else:
        scale, factor = None, float(scale)
    args = (x, residual, weight, scale)
    if (torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in args)) or _lib.watched():
        return _ResidualRmsNormFn.apply(*args, factor, float(eps))
    return _residual_forward(*args, factor, float(eps))
