"""Linear attention with one decay factor for each head, over libdynconv's
``dynconv_la_fwd`` / ``dynconv_la_bwd`` / ``dynconv_la_step``:

    S_t = exp(log_decay[h]) * S_{t-1} + k_t v_t^T          (dk x dv, float32)
    o_t = scale * q_t S_t

A prompt or a training batch runs in chunks of tokens (products within a chunk under a mask
of decays, a state handed from chunk to chunk); generating text runs the recurrence one
token at a time on a state kept by the caller.
"""
from __future__ import annotations

import ctypes

import torch
from torch.autograd.graph import increment_version

from . import _lib
from .step import _refuse_gradient, _refuse_watched, _slots

_Strides = {n: ctypes.c_int64 * n for n in (6, 12, 21)}


def _dense(t: torch.Tensor) -> torch.Tensor:
    """The kernels read any strides of batch, time and head, and a dense last dimension."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _strides(*tensors):
    s = []
    for t in tensors:
        s += t.stride()[:3]
    return _Strides[len(s)](*s)


def _ptr(t):
    return None if t is None else t.data_ptr()


def _workspace(lib, like, sizes, code, backward):
    n = lib.dynconv_la_workspace_bytes(*sizes, code, backward)
    return (torch.empty(n, device=like.device, dtype=torch.uint8), n) if n else (None, 0)


def _fwd(like, addresses, strides, sizes, log_decay, s0, o, s1, scale):
    """addresses of q, k, v, o; strides of their batch, time and head; sizes B, T, H, dk, dv."""
    lib = _lib.load()
    code = _lib.dtype_code(like.dtype)
    ws, n = _workspace(lib, like, sizes, code, 0)
    q, k, v = addresses
    status = lib.dynconv_la_fwd(q, k, v, log_decay.data_ptr(), _ptr(s0), o.data_ptr(), _ptr(s1), strides, _ptr(ws), n,
                                *sizes, scale, code, _lib.raw_stream(like))
    if status:
        _lib.check(status)
    _lib.after_call(o)


def _bwd(like, addresses, strides, sizes, log_decay, s0, ds1, ds0, scale):
    """addresses of q, k, v, do, dq, dk, dv; strides likewise."""
    lib = _lib.load()
    code = _lib.dtype_code(like.dtype)
    if ds1 is not None:
        ds1 = ds1.to(torch.float32).contiguous()
    q, k, v, do, dq, dk_, dv_ = addresses
    with _lib.device_of(like):
        ws, n = _workspace(lib, like, sizes, code, 1)
        status = lib.dynconv_la_bwd(q, k, v, log_decay.data_ptr(), _ptr(s0), do, _ptr(ds1), dq, dk_, dv_, _ptr(ds0),
                                    strides, _ptr(ws), n, *sizes, scale, code, _lib.raw_stream(like))
        if status:
            _lib.check(status)
        _lib.after_call(like)


class _DecayLinearAttentionFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, log_decay, initial_state, scale, want_state):
        q, k, v = _dense(q), _dense(k), _dense(v)
        B, T, H, dk = q.shape
        dv = v.shape[-1]
        with _lib.device_of(q):
            o = torch.empty((B, T, H, dv), device=q.device, dtype=q.dtype)
            s1 = torch.empty((B, H, dk, dv), device=q.device, dtype=torch.float32) if want_state else None
            _fwd(q, (q.data_ptr(), k.data_ptr(), v.data_ptr()), _strides(q, k, v, o), (B, T, H, dk, dv), log_decay,
                 initial_state, o, s1, scale)
        ctx.save_for_backward(q, k, v, log_decay, initial_state)
        ctx.scale = scale
        ctx.set_materialize_grads(False)
        return o, s1

    @staticmethod
    @_lib.differentiable_once
    def backward(ctx, do, ds1):
        q, k, v, log_decay, s0 = ctx.saved_tensors
        B, T, H, dk = q.shape
        do = torch.zeros(v.shape, device=v.device, dtype=v.dtype) if do is None else _dense(do.to(v.dtype))
        dq, dk_, dv_ = (torch.empty(t.shape, device=t.device, dtype=t.dtype) for t in (q, k, v))
        ds0 = torch.empty_like(s0) if s0 is not None and ctx.needs_input_grad[4] else None
        tensors = (q, k, v, do, dq, dk_, dv_)
        _bwd(q, [t.data_ptr() for t in tensors], _strides(*tensors), (B, T, H, dk, v.shape[-1]), log_decay, s0, ds1, ds0,
             ctx.scale)
        return dq, dk_, dv_, None, ds0, None, None


class _FusedDecayLinearAttentionFn(torch.autograd.Function):
    """On the thirds of one [B, T, 3*H*d] buffer, its gradient written as one buffer too."""

    @staticmethod
    def forward(ctx, qkv, log_decay, initial_state, scale, want_state):
        B, T, C = qkv.shape
        H = log_decay.shape[0]
        d = C // (3 * H)
        third = (T * C, C, d)  # strides of q, k and v in the buffer
        own = (T * H * d, H * d, d)
        at, step = qkv.data_ptr(), H * d * qkv.element_size()
        with _lib.device_of(qkv):
            o = torch.empty((B, T, H * d), device=qkv.device, dtype=qkv.dtype)
            s1 = torch.empty((B, H, d, d), device=qkv.device, dtype=torch.float32) if want_state else None
            _fwd(qkv, (at, at + step, at + 2 * step), _Strides[12](*third, *third, *third, *own), (B, T, H, d, d),
                 log_decay, initial_state, o, s1, scale)
        ctx.save_for_backward(qkv, log_decay, initial_state)
        ctx.scale = scale
        ctx.set_materialize_grads(False)
        return o, s1

    @staticmethod
    @_lib.differentiable_once
    def backward(ctx, do, ds1):
        qkv, log_decay, s0 = ctx.saved_tensors
        B, T, C = qkv.shape
        H = log_decay.shape[0]
        d = C // (3 * H)
        if do is None:
            do = torch.zeros((B, T, H * d), device=qkv.device, dtype=qkv.dtype)
        do = do.to(qkv.dtype).contiguous()
        dqkv = torch.empty_like(qkv)
        ds0 = torch.empty_like(s0) if s0 is not None and ctx.needs_input_grad[2] else None
        third, own = (T * C, C, d), (T * H * d, H * d, d)
        at, to, step = qkv.data_ptr(), dqkv.data_ptr(), H * d * qkv.element_size()
        _bwd(qkv, (at, at + step, at + 2 * step, do.data_ptr(), to, to + step, to + 2 * step),
             _Strides[21](*third, *third, *third, *own, *third, *third, *third), (B, T, H, d, d), log_decay, s0, ds1, ds0,
             ctx.scale)
        return dqkv, None, ds0, None, None


def _check_decay(log_decay, dev, H):
    assert log_decay.get_device() == dev and log_decay.is_contiguous() and log_decay.dtype == torch.float32
    assert log_decay.shape == (H,)
    assert not log_decay.requires_grad, "the decay is a constant of each head: it has no gradient"


def _check_state(state, dev, rows, H, dk, dv):
    """Rows of a state."""
    assert state.get_device() == dev and state.is_contiguous() and state.dtype == torch.float32 and state.dim() == 4
    n, h, a, b = state.shape
    assert h == H and a == dk and b == dv, f"state must be [n, {H}, {dk}, {dv}]"
    assert rows is None or n == rows
    return n


def decay_linear_attention(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    log_decay: torch.Tensor,
    initial_state: torch.Tensor | None = None,
    scale: float | None = None,
    return_state: bool = False,
):
    """Causal linear attention with a decay for each head.

    Args:
        q, k:          [B, T, H, dk] (bfloat16 or float32, CUDA; any strides of batch, time and
                       head, so views of a fused projection are read in place).
        v:             [B, T, H, dv].  dk, dv <= 256; multiples of 8 up to 128 run on the
                       tensor cores in bfloat16.
        log_decay:     [H] float32, the logarithm of each head's decay per token, <= 0.
        initial_state: [B, H, dk, dv] float32, the state before the first token (None: zero).
        scale:         factor of the queries; dk**-0.5 by default.
        return_state:  also return the state after the last token, [B, H, dk, dv] float32.

    Returns:
        o [B, T, H, dv], or (o, state).  Differentiable (once) in q, k, v and initial_state.
    """
    dev = q.get_device()  # (-1 on the CPU)
    assert dev >= 0 and k.get_device() == dev and v.get_device() == dev
    assert q.dim() == 4 and k.shape == q.shape and v.shape[:3] == q.shape[:3] and v.dim() == 4
    assert q.dtype == k.dtype == v.dtype
    _, _, H, dk = q.shape
    _check_decay(log_decay, dev, H)
    if initial_state is not None:
        _check_state(initial_state, dev, q.shape[0], H, dk, v.shape[-1])
    scale = dk**-0.5 if scale is None else float(scale)
    o, s1 = _DecayLinearAttentionFn.apply(q, k, v, log_decay, initial_state, scale, bool(return_state))
    return (o, s1) if return_state else o


def decay_linear_attention_fused(
    qkv: torch.Tensor,
    log_decay: torch.Tensor,
    initial_state: torch.Tensor | None = None,
    scale: float | None = None,
    return_state: bool = False,
):
    """``decay_linear_attention`` on the fused queries, keys and values qkv [B, T, 3*H*d], as
    ``QKVLowRankDynamicShortConvolution.forward_fused`` returns them, with H = len(log_decay).
    Returns o [B, T, H*d] (or (o, state)); the gradient comes back as one [B, T, 3*H*d]
    tensor, with no split or concatenation on either way."""
    dev = qkv.get_device()
    assert dev >= 0 and qkv.is_contiguous() and qkv.dim() == 3
    H = log_decay.shape[0]
    assert qkv.shape[-1] % (3 * H) == 0, "qkv must be [B, T, 3*H*d]"
    d = qkv.shape[-1] // (3 * H)
    _check_decay(log_decay, dev, H)
    if initial_state is not None:
        _check_state(initial_state, dev, qkv.shape[0], H, d, d)
    scale = d**-0.5 if scale is None else float(scale)
    o, s1 = _FusedDecayLinearAttentionFn.apply(qkv, log_decay, initial_state, scale, bool(return_state))
    return (o, s1) if return_state else o


def decay_linear_attention_step(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    state: torch.Tensor,
    log_decay: torch.Tensor,
    scale: float | None = None,
    slots: torch.Tensor | None = None,
) -> torch.Tensor:
    """One token for each of B sequences.

    Args:
        q, k:  [B, H, dk], v: [B, H, dv] (bfloat16 or float32; views of a fused row will do).
        state: [n, H, dk, dv] float32, contiguous; updated in place.
        slots: [B] int32 or int64, each sequence's row of the state, none twice; rows outside
               0..n-1 touch no state and give zeros.  None: row b (n >= B).

    Returns:
        o: [B, H, dv].  Has no gradient.
    """
    dev = q.get_device()
    assert dev >= 0 and k.get_device() == dev and v.get_device() == dev
    assert q.dim() == 3 and k.shape == q.shape and v.dim() == 3 and v.shape[:2] == q.shape[:2]
    assert q.dtype == k.dtype == v.dtype
    B, H, dk = q.shape
    dv = v.shape[-1]
    _check_decay(log_decay, dev, H)
    n = _check_state(state, dev, None, H, dk, dv)
    assert slots is not None or n >= B
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or state.requires_grad):
        _refuse_gradient()
    if _lib.watched():
        _refuse_watched(q, k, v, state)
    code = _lib.dtype_code(q.dtype)
    (qb, qh, qd), (kb, kh, kd), (vb, vh, vd) = q.stride(), k.stride(), v.stride()
    if (qd != 1 and dk > 1) or (kd != 1 and dk > 1) or (vd != 1 and dv > 1):
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
        (qb, qh, _), (kb, kh, _), (vb, vh, _) = q.stride(), k.stride(), v.stride()
    sp, sb = (None, 0) if slots is None else _slots(slots, B, dev)
    o = torch.empty((B, H, dv), device=q.device, dtype=q.dtype)
    with _lib.device_of(q):
        status = _lib.load().dynconv_la_step(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), state.data_ptr(), log_decay.data_ptr(), o.data_ptr(), sp, sb,
            _Strides[6](qb, qh, kb, kh, vb, vh), B, n, H, dk, dv, dk**-0.5 if scale is None else float(scale), code,
            _lib.raw_stream(q))
        if status:
            _lib.check(status)
        _lib.after_call(o)
    increment_version(state)  # (a backward that kept the state before this step raises)
    return o
