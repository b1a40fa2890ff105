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

from . import _lib
from .step import _no_grad_wanted, _slots

_Strides = {n: ctypes.c_int64 * n for n in (6, 12, 21)}


def _dense(t: torch.Tensor) -> torch.Tensor:
    """The kernels read any strides of batch, time and head, and a dense last dimension."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _strides(*tensors):
    s = []
    for t in tensors:
        s += t.stride()[:3]
    return _Strides[len(s)](*s)


def _workspace(lib, q, dv, backward):
    B, T, H, dk = q.shape
    n = lib.dynconv_la_workspace_bytes(B, T, H, dk, dv, _lib.dtype_code(q.dtype), backward)
    return torch.empty(n, device=q.device, dtype=torch.uint8) if n else None


def _fwd(q, k, v, log_decay, s0, o, s1, scale):
    lib = _lib.load()
    B, T, H, dk = q.shape
    dv = v.shape[-1]
    ws = _workspace(lib, q, dv, 0)
    _lib.check(
        lib.dynconv_la_fwd(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), log_decay.data_ptr(), None if s0 is None else s0.data_ptr(),
            o.data_ptr(), None if s1 is None else s1.data_ptr(), _strides(q, k, v, o),
            None if ws is None else ws.data_ptr(), 0 if ws is None else ws.numel(),
            B, T, H, dk, dv, scale, _lib.dtype_code(q.dtype), _lib.raw_stream(q),
        )
    )
    _lib.after_call(o)


def _bwd(q, k, v, log_decay, s0, do, ds1, dq, dk_, dv_, ds0, scale):
    lib = _lib.load()
    B, T, H, dk = q.shape
    dv = v.shape[-1]
    if ds1 is not None:
        ds1 = ds1.to(torch.float32).contiguous()
    with _lib.device_of(q):
        ws = _workspace(lib, q, dv, 1)
        _lib.check(
            lib.dynconv_la_bwd(
                q.data_ptr(), k.data_ptr(), v.data_ptr(), log_decay.data_ptr(), None if s0 is None else s0.data_ptr(),
                do.data_ptr(), None if ds1 is None else ds1.data_ptr(), dq.data_ptr(), dk_.data_ptr(), dv_.data_ptr(),
                None if ds0 is None else ds0.data_ptr(), _strides(q, k, v, do, dq, dk_, dv_),
                None if ws is None else ws.data_ptr(), 0 if ws is None else ws.numel(),
                B, T, H, dk, dv, scale, _lib.dtype_code(q.dtype), _lib.raw_stream(q),
            )
        )
        _lib.after_call(dq)


class _DecayLinearAttentionFn(torch.autograd.Function):
    @staticmethod
    @_lib.on_device
    def forward(ctx, q, k, v, log_decay, initial_state, scale, want_state):
        q, k, v = _dense(q), _dense(k), _dense(v)
        B, T, H, dk = q.shape
        dv = v.shape[-1]
        o = torch.empty((B, T, H, dv), device=q.device, dtype=q.dtype)
        s1 = torch.empty((B, H, dk, dv), device=q.device, dtype=torch.float32) if want_state else None
        _fwd(q, k, v, log_decay, initial_state, o, s1, scale)
        ctx.save_for_backward(q, k, v, log_decay, initial_state)
        ctx.scale = scale
        ctx.set_materialize_grads(False)
        return o, s1

    @staticmethod
    def backward(ctx, do, ds1):
        q, k, v, log_decay, s0 = ctx.saved_tensors
        do = torch.zeros(v.shape, device=v.device, dtype=v.dtype) if do is None else _dense(do.to(v.dtype))
        dq, dk_, dv_ = (torch.empty(t.shape, device=t.device, dtype=t.dtype) for t in (q, k, v))
        ds0 = torch.empty_like(s0) if s0 is not None and ctx.needs_input_grad[4] else None
        _bwd(q, k, v, log_decay, s0, do, ds1, dq, dk_, dv_, ds0, ctx.scale)
        return dq, dk_, dv_, None, ds0, None, None


class _FusedDecayLinearAttentionFn(torch.autograd.Function):
    """On the thirds of one [B, T, 3*H*d] buffer, its gradient written as one buffer too."""

    @staticmethod
    @_lib.on_device
    def forward(ctx, qkv, log_decay, initial_state, scale, want_state):
        B, T, C = qkv.shape
        H = log_decay.shape[0]
        d = C // (3 * H)
        q, k, v = qkv.view(B, T, 3, H, d).unbind(2)
        o = torch.empty((B, T, H * d), device=qkv.device, dtype=qkv.dtype)
        s1 = torch.empty((B, H, d, d), device=qkv.device, dtype=torch.float32) if want_state else None
        _fwd(q, k, v, log_decay, initial_state, o.view(B, T, H, d), s1, scale)
        ctx.save_for_backward(qkv, log_decay, initial_state)
        ctx.scale = scale
        ctx.set_materialize_grads(False)
        return o, s1

    @staticmethod
    def backward(ctx, do, ds1):
        qkv, log_decay, s0 = ctx.saved_tensors
        B, T, C = qkv.shape
        H = log_decay.shape[0]
        d = C // (3 * H)
        shape = (B, T, 3, H, d)
        if do is None:
            do = torch.zeros((B, T, H * d), device=qkv.device, dtype=qkv.dtype)
        do = do.to(qkv.dtype).contiguous().view(B, T, H, d)
        dqkv = torch.empty_like(qkv)
        ds0 = torch.empty_like(s0) if s0 is not None and ctx.needs_input_grad[2] else None
        _bwd(*qkv.view(shape).unbind(2), log_decay, s0, do, ds1, *dqkv.view(shape).unbind(2), ds0,
             ctx.scale)
        return dqkv, None, ds0, None, None


def _check_decay(log_decay, H):
    assert log_decay.is_cuda and log_decay.is_contiguous() and log_decay.dtype == torch.float32
    assert log_decay.shape == (H,)
    assert not log_decay.requires_grad, "the decay is a constant of each head: it has no gradient"


def _check_state(state, rows, H, dk, dv):
    assert state.is_cuda and state.is_contiguous() and state.dtype == torch.float32
    assert state.dim() == 4 and state.shape[1:] == (H, dk, dv)
    assert rows is None or state.shape[0] == rows


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
        o [B, T, H, dv], or (o, state).  Differentiable in q, k, v and initial_state.
    """
    assert q.is_cuda and k.is_cuda and v.is_cuda
    assert q.dim() == 4 and k.shape == q.shape and v.shape[:3] == q.shape[:3] and v.dim() == 4
    assert q.dtype == k.dtype == v.dtype
    _, _, H, dk = q.shape
    _check_decay(log_decay, H)
    if initial_state is not None:
        _check_state(initial_state, q.shape[0], H, dk, v.shape[-1])
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
    assert qkv.is_cuda and qkv.is_contiguous() and qkv.dim() == 3
    H = log_decay.shape[0]
    assert qkv.shape[-1] % (3 * H) == 0, "qkv must be [B, T, 3*H*d]"
    d = qkv.shape[-1] // (3 * H)
    _check_decay(log_decay, H)
    if initial_state is not None:
        _check_state(initial_state, qkv.shape[0], H, d, d)
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
    assert q.is_cuda and k.is_cuda and v.is_cuda
    assert q.dim() == 3 and k.shape == q.shape and v.dim() == 3 and v.shape[:2] == q.shape[:2]
    assert q.dtype == k.dtype == v.dtype
    B, H, dk = q.shape
    dv = v.shape[-1]
    _check_decay(log_decay, H)
    _check_state(state, None, H, dk, dv)
    assert slots is not None or state.shape[0] >= B
    _no_grad_wanted(q, k, v, state)
    code = _lib.dtype_code(q.dtype)
    q, k, v = _dense(q), _dense(k), _dense(v)
    sp, sb = _slots(slots, B)
    o = torch.empty((B, H, dv), device=q.device, dtype=q.dtype)
    with _lib.device_of(q):
        _lib.check(
            _lib.load().dynconv_la_step(
                q.data_ptr(), k.data_ptr(), v.data_ptr(), state.data_ptr(), log_decay.data_ptr(), o.data_ptr(), sp, sb,
                _Strides[6](*q.stride()[:2], *k.stride()[:2], *v.stride()[:2]), B, state.shape[0], H, dk, dv,
                dk**-0.5 if scale is None else float(scale), code, _lib.raw_stream(q),
            )
        )
        _lib.after_call(o)
    return o
