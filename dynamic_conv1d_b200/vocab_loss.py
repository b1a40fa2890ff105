"""Softmax cross entropy over a large vocabulary, in pieces of it, without keeping the
logits (libdynconv's ``dynconv_vocab_loss_fwd`` / ``dynconv_vocab_loss_bwd``).

The forward reads the hidden states and the vocabulary's weight once and keeps two float32
per token (the logarithm of the sum of exponentials, and the token's loss).  The backward computes the logits
again, one piece of the vocabulary at a time, into a buffer that holds that piece's
gradient only.  float32 tensors are multiplied as three bfloat16 parts each, to float32
accuracy.
"""
from __future__ import annotations

import torch

from . import _lib

_REDUCTIONS = {"none": 0, "sum": 1, "mean": 2}
_KEEP_ROWS = 4  # added to the reduction for the library


def _aligned(t):
    """t at a 16-byte boundary, where its rows of bfloat16 are whole multiples of 16 bytes (the
    library then reads them in place)."""
    return t.clone() if t.dtype == torch.bfloat16 and t.shape[1] % 8 == 0 and t.data_ptr() % 16 else t


class _LinearCrossEntropyFn(torch.autograd.Function):
    @staticmethod
    @_lib.on_device
    def forward(ctx, hidden, weight, target, ignore_index, reduction):
        N, D = hidden.shape
        V = weight.shape[0]
        lib = _lib.load()
        code = _lib.dtype_code(hidden.dtype)
        hidden, w = _aligned(hidden), _aligned(weight if weight.dtype == hidden.dtype else weight.to(hidden.dtype))
        loss = torch.empty((N,) if reduction == 0 else (), device=hidden.device, dtype=torch.float32)
        kept = torch.empty(2 * N + 2, device=hidden.device, dtype=torch.float32)  # stats, lse, the rows' losses
        n = lib.dynconv_vocab_loss_fwd_workspace_bytes(N, D, V, code)
        ws = torch.empty(max(n, 1), device=hidden.device, dtype=torch.uint8)
        _lib.check(
            lib.dynconv_vocab_loss_fwd(
                hidden.data_ptr(), w.data_ptr(), target.data_ptr(), loss.data_ptr(), kept.data_ptr() + 8,
                kept.data_ptr(), ws.data_ptr(), ws.numel(), N, D, V, ignore_index, reduction + _KEEP_ROWS,
                code, _lib.raw_stream(hidden),
            )
        )
        _lib.after_call(loss)
        ctx.save_for_backward(hidden, w, target, kept)
        ctx.args = (ignore_index, reduction, weight.dtype)
        return loss

    @staticmethod
    @_lib.differentiable_once
    @_lib.on_device
    def backward(ctx, dloss):
        hidden, w, target, kept = ctx.saved_tensors
        ignore_index, reduction, weight_dtype = ctx.args
        N, D = hidden.shape
        V = w.shape[0]
        lib = _lib.load()
        code = _lib.dtype_code(hidden.dtype)
        dloss = dloss.to(torch.float32).contiguous()
        dh = torch.empty_like(hidden) if ctx.needs_input_grad[0] else None
        dw = torch.empty_like(w) if ctx.needs_input_grad[1] else None
        n = lib.dynconv_vocab_loss_bwd_workspace_bytes(N, D, V, code, int(dh is not None), int(dw is not None))
        ws = torch.empty(max(n, 1), device=hidden.device, dtype=torch.uint8)
        _lib.check(
            lib.dynconv_vocab_loss_bwd(
                hidden.data_ptr(), w.data_ptr(), target.data_ptr(), kept.data_ptr() + 8, kept.data_ptr(),
                dloss.data_ptr(), None if dh is None else dh.data_ptr(), None if dw is None else dw.data_ptr(),
                ws.data_ptr(), ws.numel(), N, D, V, ignore_index, reduction + _KEEP_ROWS, code, _lib.raw_stream(hidden),
            )
        )
        _lib.after_call(hidden)
        if dw is not None and dw.dtype != weight_dtype:
            dw = dw.to(weight_dtype)
        return dh, dw, None, None, None


def linear_cross_entropy(
    hidden: torch.Tensor,
    weight: torch.Tensor,
    target: torch.Tensor,
    ignore_index: int = -100,
    reduction: str = "mean",
) -> torch.Tensor:
    """Cross entropy of ``hidden @ weight.T`` against ``target``, without the logits in memory.

    Args:
        hidden:       [..., D] (bfloat16 or float32, CUDA, contiguous).
        weight:       [V, D], contiguous; cast to hidden's dtype when it has another one (its
                      gradient is then rounded to that dtype before it is cast back).
        target:       [...] int64, the index of each row's word.  Rows whose target is
                      ``ignore_index`` count for nothing, whatever they hold.  Any other target
                      outside 0..V-1 makes the loss NaN (and gives that row no gradient).
        reduction:    "mean" over the rows that count (NaN when none does), "sum", or "none".

    Returns:
        the loss in float32: a scalar, or of target's shape for "none".  Differentiable (once) in
        hidden and weight.  Under ``data_parallel()`` both the mean and weight's gradient
        are this rank's own, as for any other parameter of the model around the ops.
    """
    assert hidden.is_cuda and hidden.is_contiguous()
    assert weight.device == hidden.device and weight.is_contiguous() and weight.dim() == 2
    assert weight.shape[1] == hidden.shape[-1]
    assert target.device == hidden.device and target.dtype == torch.int64 and target.shape == hidden.shape[:-1]
    assert reduction in _REDUCTIONS, f"reduction must be one of {tuple(_REDUCTIONS)}"
    if hidden.dim() != 2:  # (a view is one more node of the graph)
        hidden = hidden.view(-1, hidden.shape[-1])
    loss = _LinearCrossEntropyFn.apply(
        hidden, weight, target.reshape(-1).contiguous(), int(ignore_index), _REDUCTIONS[reduction])
    return loss.view(target.shape) if reduction == "none" else loss
