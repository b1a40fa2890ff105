"""The gated delta rule, over libdynconv's ``dynconv_delta_fwd`` / ``dynconv_delta_bwd`` /
``dynconv_delta_step``:

    S_t = a_t S_{t-1} + k_t u_t^T,   a_t = exp(log_decay_t)                (dk x dv, float32)
    u_t = beta_t (v_t - a_t S_{t-1}^T k_t)
    o_t = scale * q_t S_t

What the state holds for a token's key is replaced by the token's value, by the share beta_t, and
everything fades by the token's own decay.  A prompt or a training batch runs in chunks of tokens
(a triangular system within a chunk, the state handed from chunk to chunk); generating text runs
the recurrence one token at a time on a state kept by the caller.
"""
from __future__ import annotations

import ctypes

import torch
from torch.autograd.graph import increment_version

from . import _lib
from .linear_attention import _check_state, _dense, _ptr
from .step import _refuse_gradient, _refuse_watched, _slots

_Strides = {n: ctypes.c_int64 * n for n in (10, 18, 30)}


def _strides(*tensors):
    s = []
    for t in tensors:
        s += _row_strides(t)
    return _Strides[len(s)](*s)


def _rows(t: torch.Tensor) -> torch.Tensor:
    """t as the kernels read it: dense in the last dimension and, where its width allows, every row at a
    positive multiple of 16 bytes."""
    t = _dense(t)
    per = 16 // t.element_size()
    if t.shape[-1] % per == 0 and (t.data_ptr() % 16 or any(n > 1 and (s <= 0 or s % per) for n, s in zip(t.shape[:3], t.stride()[:3]))):
        t = t.clone(memory_format=torch.contiguous_format)
    return t


def _row_strides(t: torch.Tensor):
    """Strides of batch, time and head; those of dimensions of one count for nothing, and zero is aligned."""
    return [s if n > 1 else 0 for n, s in zip(t.shape[:3], t.stride()[:3])]


def _workspace(lib, like, B, T, H, dk, dv, code, backward):
    n = lib.dynconv_delta_workspace_bytes(B, T, H, dk, dv, code, backward)
    return torch.empty(n, device=like.device, dtype=torch.uint8)


def _code(q, log_decay):
    code = _lib.dtype_code(q.dtype)
    return code if log_decay.dtype == q.dtype else code + _lib.GATES_F32


def _forward(q, k, v, log_decay, beta, initial_state, scale, want_state, keep):
    q, k, v = _rows(q), _rows(k), _rows(v)
    B, T, H, dk = q.shape
    dv = v.shape[-1]
    if scale is None:
        scale = dk**-0.5
    lib = _lib.load()
    code = _code(q, log_decay)
    with _lib.device_of(q):
        o = torch.empty((B, T, H, dv), device=q.device, dtype=q.dtype)
        s1 = torch.empty((B, H, dk, dv), device=q.device, dtype=torch.float32) if want_state else None
        kept, n = None, 0
        if keep:
            n = lib.dynconv_delta_kept_bytes(B, T, H, dk, dv, code)
            kept = torch.empty(n, device=q.device, dtype=torch.uint8)
        ws = _workspace(lib, q, B, T, H, dk, dv, code, 0)
        status = lib.dynconv_delta_fwd(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), log_decay.data_ptr(), beta.data_ptr(), _ptr(initial_state), o.data_ptr(),
            _ptr(s1), _ptr(kept), n, _strides(q, k, v, log_decay, beta, o), ws.data_ptr(), ws.numel(),
            B, T, H, dk, dv, scale, code, _lib.raw_stream(q))
        if status:
            _lib.check(status)
        _lib.after_call(o)
    return o, s1, q, k, kept, scale


class _GatedDeltaRuleFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, log_decay, beta, initial_state, scale, want_state):
        o, s1, q, k, kept, scale = _forward(q, k, v, log_decay, beta, initial_state, scale, want_state, True)
        ctx.save_for_backward(q, k, log_decay, beta, kept)
        ctx.args = (scale, v.shape[-1], initial_state is not None)
        ctx.set_materialize_grads(False)
        return o, s1

    @staticmethod
    @_lib.differentiable_once
    def backward(ctx, do, ds1):
        q, k, log_decay, beta, kept = ctx.saved_tensors
        scale, dv, has_state = ctx.args
        B, T, H, dk = q.shape
        lib = _lib.load()
        code = _code(q, log_decay)
        with _lib.device_of(q):
            do = torch.zeros((B, T, H, dv), device=q.device, dtype=q.dtype) if do is None else _rows(do.to(q.dtype))
            if ds1 is not None:
                ds1 = ds1.to(torch.float32).contiguous()
            new = lambda like, *shape: torch.empty(shape, device=q.device, dtype=like.dtype)  # noqa: E731
            dq, dk_, dv_ = new(q, B, T, H, dk), new(q, B, T, H, dk), new(q, B, T, H, dv)
            dg, db = new(log_decay, B, T, H), new(beta, B, T, H)
            ds0 = None
            if has_state and ctx.needs_input_grad[5]:
                ds0 = torch.empty((B, H, dk, dv), device=q.device, dtype=torch.float32)
            ws = _workspace(lib, q, B, T, H, dk, dv, code, 1)
            status = lib.dynconv_delta_bwd(
                q.data_ptr(), k.data_ptr(), log_decay.data_ptr(), beta.data_ptr(), kept.data_ptr(), kept.numel(), do.data_ptr(),
                _ptr(ds1), dq.data_ptr(), dk_.data_ptr(), dv_.data_ptr(), dg.data_ptr(), db.data_ptr(), _ptr(ds0),
                _strides(q, k, log_decay, beta, do, dq, dk_, dv_, dg, db), ws.data_ptr(), ws.numel(), B, T, H, dk, dv, scale,
                code, _lib.raw_stream(q))
            if status:
                _lib.check(status)
            _lib.after_call(dq)
        return dq, dk_, dv_, dg, db, ds0, None, None


def _check_gates(log_decay, beta, like, shape):
    dev, dtype = like.get_device(), log_decay.dtype
    assert log_decay.get_device() == dev and beta.get_device() == dev
    assert dtype == beta.dtype and (dtype == like.dtype or dtype == torch.float32)
    assert log_decay.shape == shape and beta.shape == shape, f"log_decay and beta must be {list(shape)}"


def gated_delta_rule(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    log_decay: torch.Tensor,
    beta: torch.Tensor,
    initial_state: torch.Tensor | None = None,
    scale: float | None = None,
    return_state: bool = False,
):
    """The gated delta rule over whole sequences.

    Args:
        q, k:          [B, T, H, dk] (bfloat16 or float32, CUDA; any strides of batch, time and
                       head, so views of a fused projection are read in place).  dk <= 128.  Keys
                       are meant to have a length of at most one (``gated_rms_norm`` gives them it).
                       B * H <= 65535.
        v:             [B, T, H, dv], dv <= 256.
        log_decay:     [B, T, H] in q's dtype or float32, the logarithm of each token's decay, <= 0.
        beta:          [B, T, H] in log_decay's dtype, the share of the value that is replaced.
        initial_state: [B, H, dk, dv] float32, the state before the first token (None: zero).
        scale:         factor of the queries; dk**-0.5 by default.
        return_state:  also return the state after the last token, [B, H, dk, dv] float32.

    Returns:
        o [B, T, H, dv], or (o, state).  Differentiable (once) in all tensors.  What is not finite in
        one token reaches no earlier token's output; from it on the head's are NaN (from a value: at
        least its own columns'; a query is its own token's alone).
        With gradients the call keeps the state at every 64th token (float32: 32nd) in that type's digits and
        four bytes (float32: six) for each number of v.
    """
    dev = q.get_device()  # (-1 on the CPU)
    assert dev >= 0 and k.get_device() == dev and v.get_device() == dev
    assert q.dim() == 4 and k.shape == q.shape and v.shape[:3] == q.shape[:3] and v.dim() == 4
    assert q.dtype == k.dtype == v.dtype
    B, T, H, dk = q.shape
    _check_gates(log_decay, beta, q, (B, T, H))
    if initial_state is not None:
        _check_state(initial_state, dev, B, H, dk, v.shape[-1])
    scale = None if scale is None else float(scale)
    args = (q, k, v, log_decay, beta, initial_state)
    if (torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in args)) or _lib.watched():
        o, s1 = _GatedDeltaRuleFn.apply(*args, scale, bool(return_state))
    else:
        o, s1 = _forward(*args, scale, return_state, False)[:2]
    return (o, s1) if return_state else o


def gated_delta_rule_step(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    state: torch.Tensor,
    log_decay: torch.Tensor,
    beta: torch.Tensor,
    scale: float | None = None,
    slots: torch.Tensor | None = None,
) -> torch.Tensor:
    """One token for each of B sequences.

    Args:
        q, k:            [B, H, dk], v: [B, H, dv] (bfloat16 or float32; views of a fused row will do).
                         B and H up to 65535 each.
        state:           [n, H, dk, dv] float32, contiguous; updated in place.
        log_decay, beta: [B, H], both in q's dtype or both float32.
        slots:           [B] int32 or int64, each sequence's row of the state, none twice; rows
                         outside 0..n-1 touch no state and give zeros.  None: row b (n >= B).

    Returns:
        o: [B, H, dv].  Has no gradient.
    """
    dev = q.get_device()
    assert dev >= 0 and k.get_device() == dev and v.get_device() == dev
    assert q.dim() == 3 and k.shape == q.shape and v.dim() == 3 and v.shape[:2] == q.shape[:2]
    assert q.dtype == k.dtype == v.dtype
    B, H, dk = q.shape
    dv = v.shape[-1]
    _check_gates(log_decay, beta, q, (B, H))
    n = _check_state(state, dev, None, H, dk, dv)
    assert slots is not None or n >= B
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or state.requires_grad
                                    or log_decay.requires_grad or beta.requires_grad):
        _refuse_gradient()
    if _lib.watched():
        _refuse_watched(q, k, v, state, log_decay, beta)
    code = _code(q, log_decay)
    q, k, v = _dense(q), _dense(k), _dense(v)
    sp, sb = (None, 0) if slots is None else _slots(slots, B, dev)
    (qb, qh, _), (kb, kh, _), (vb, vh, _) = q.stride(), k.stride(), v.stride()
    strides = _Strides[10](qb, qh, kb, kh, vb, vh, *log_decay.stride(), *beta.stride())
    with _lib.device_of(q):
        o = v.new_empty((B, H, dv))
        status = _lib.load().dynconv_delta_step(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), log_decay.data_ptr(), beta.data_ptr(), state.data_ptr(), o.data_ptr(), sp, sb,
            strides, B, n, H, dk, dv, dk**-0.5 if scale is None else float(scale), code, _lib.raw_stream(q))
        if status:
            _lib.check(status)
        _lib.after_call(o)
    increment_version(state)  # (a backward that kept the state before this step raises)
    return o
