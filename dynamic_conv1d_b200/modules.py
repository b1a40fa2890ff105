"""nn.Module wrappers of the low-rank dynamic convolution, as in the reference's
README (README.md:57-84: ``LowRankDynamicShortConvolution``; README.md:86-105:
one module each for the queries, keys and values of an attention layer).

``LowRankDynamicShortConvolution`` has the reference module's parameters, their
initialisation and its error: ``proj_in`` (d_model -> R, no bias) produces z from
the pre-norm input, ``proj_out`` is U (zeros, [R, W*d_model]), and
``proj_out_bias`` is static_w ([W, d_model], uniform in +-1/sqrt(W)), folded into
the kernels as rank R -- so R+1 must be a power of two.

``QKVLowRankDynamicShortConvolution`` holds the three modules' parameters,
computes the three z projections as one GEMM (the three proj_in weights stacked,
one read of the pre-norm activations instead of three) and the three
convolutions as one grouped kernel launch per direction.

``ConvolvedLinearAttention`` is an attention layer on top of it: the three convolved
streams mixed by linear attention with a decay for each head, for training and prompts,
and its single-token form for generating text.  ``ConvolvedGatedDelta`` is its sibling on the gated
delta rule, with learned decays and a gated norm, and ``ResidualRMSNorm`` stands between two blocks.

proj_in is an ordinary GEMM (cuBLAS through ``torch.nn.functional.linear``): z
needs a dot product over all d_model channels for each token, while a
convolution tile sees 128 of them, so it is not fused into the convolution
kernels."""
from __future__ import annotations

import math
from dataclasses import dataclass

import torch
from torch import nn

from .gated_delta import gated_delta_rule, gated_delta_rule_step
from .linear_attention import decay_linear_attention_fused, decay_linear_attention_step
from .lowrank import lowrank_dynamic_convolution, lowrank_dynamic_convolution_grouped
from .norm import gated_rms_norm, residual_rms_norm
from .step import convolution_cache, lowrank_dynamic_convolution_grouped_step


def _check_rank(R: int) -> None:
    if ((R + 1) & R) != 0:
        raise ValueError("R+1 must be a power of two")


class LowRankDynamicShortConvolution(nn.Module):
    """Low-rank dynamic short convolution with its static (bias) filter.

    forward(x, pre_z): x [B, T, d_model] is convolved, pre_z [B, T, d_model] (the
    pre-norm activations) produces the rank-R mixing coefficients z.
    """

    def __init__(self, d_model: int, R: int, W: int):
        super().__init__()
        _check_rank(R)
        self.d_model, self.R, self.W = d_model, R, W
        self.proj_in = nn.Linear(d_model, R, bias=False)
        self.proj_out = nn.Parameter(torch.zeros(R, W * d_model))
        self.proj_out_bias = nn.Parameter(torch.empty(W, d_model))
        nn.init.uniform_(self.proj_out_bias, -1.0 / math.sqrt(W), +1.0 / math.sqrt(W))

    def forward(self, x: torch.Tensor, pre_z: torch.Tensor) -> torch.Tensor:
        z = self.proj_in(pre_z)
        return lowrank_dynamic_convolution(
            x=x.contiguous(),
            z=z.contiguous(),
            U=self.proj_out,
            static_w=self.proj_out_bias,
            residual=True,
        )


class QKVLowRankDynamicShortConvolution(nn.Module):
    """The query, key and value convolutions of one attention layer.

    Parameters are those of three ``LowRankDynamicShortConvolution`` modules
    (``q``, ``k``, ``v``).  The three proj_in GEMMs run as one over the stacked
    weights, and the three convolutions as one grouped launch per direction
    (``lowrank_dynamic_convolution_grouped``), with one all-reduce of the stacked
    dU / static_w gradients under ``data_parallel()``.

    ``forward_fused(qkv, pre_z)`` takes the fused projection output [B, T, 3*d_model]
    as it comes out of the QKV GEMM and returns the three results in the same
    layout, with no split or copy.  ``forward(q, k, v, pre_z)`` takes the three
    tensors (concatenated once, as the reference's ``.contiguous()`` calls copy
    them) and returns three [B, T, d_model] views.
    """

    def __init__(self, d_model: int, R: int, W: int):
        super().__init__()
        self.q = LowRankDynamicShortConvolution(d_model, R, W)
        self.k = LowRankDynamicShortConvolution(d_model, R, W)
        self.v = LowRankDynamicShortConvolution(d_model, R, W)

    def stacked(self):
        """The three modules' parameters as the fused calls take them: proj_in [3R, d_model],
        U [3, R, W*d_model], static_w [3, W, d_model].  A program that generates text keeps
        the result for its ``step`` calls."""
        mods = (self.q, self.k, self.v)
        return (torch.cat([m.proj_in.weight for m in mods], dim=0), torch.stack([m.proj_out for m in mods]),
                torch.stack([m.proj_out_bias for m in mods]))

    def forward_fused(self, qkv: torch.Tensor, pre_z: torch.Tensor) -> torch.Tensor:
        w_in, U, sw = self.stacked()
        z_all = torch.nn.functional.linear(pre_z, w_in)  # [B, T, 3R]
        return lowrank_dynamic_convolution_grouped(qkv.contiguous(), z_all.contiguous(), U, sw, residual=True)

    def step(self, qkv: torch.Tensor, pre_z: torch.Tensor, cache: torch.Tensor, stacked=None,
             slots: torch.Tensor | None = None) -> torch.Tensor:
        """One token: qkv [B, 3*d_model] and pre_z [B, d_model], on a cache [n, W-1, 3*d_model]
        updated in place (``convolution_cache(qkv, W)`` after a prompt); stacked as from
        ``stacked()``, slots as for ``lowrank_dynamic_convolution_grouped_step``."""
        w_in, U, sw = self.stacked() if stacked is None else stacked
        z_all = torch.nn.functional.linear(pre_z, w_in)
        return lowrank_dynamic_convolution_grouped_step(qkv.contiguous(), z_all.contiguous(), U, cache, sw, residual=True,
                                                        slots=slots)

    def forward(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, pre_z: torch.Tensor):
        y = self.forward_fused(torch.cat([q, k, v], dim=-1), pre_z)
        return y.split(self.q.d_model, dim=-1)


@dataclass
class LayerCache:
    """What one ``ConvolvedLinearAttention`` or ``ConvolvedGatedDelta`` layer keeps of its sequences between tokens."""

    conv: torch.Tensor  # [n, W-1, 3*d_model]: the last inputs of the convolutions
    state: torch.Tensor  # [n, H, d, d] float32: the attention's state
    stacked: tuple  # the convolutions' parameters, laid out once


class ConvolvedLinearAttention(nn.Module):
    """An attention layer on convolved queries, keys and values: one fused projection, the
    grouped low-rank dynamic convolution of its three thirds, linear attention whose state
    decays by a factor of its own in each head, and an output projection.

    The decays are constants: 1 - 2^-5 in the first head to 1 - 2^-12 in the last, a memory of
    about 32 to 4096 tokens.  ``forward`` takes pre-norm activations [B, T, d_model].
    ``prompt`` does the same for sequences that will be continued and returns their
    ``LayerCache``; ``step`` takes one token of each, [B, d_model].  Nothing in between is
    split, concatenated or copied.
    """

    def __init__(self, d_model: int, n_heads: int, R: int = 15, W: int = 4):
        super().__init__()
        if d_model % n_heads != 0:
            raise ValueError("d_model must be divisible by n_heads")
        self.d_model, self.n_heads, self.W = d_model, n_heads, W
        self.qkv = nn.Linear(d_model, 3 * d_model, bias=False)
        self.conv = QKVLowRankDynamicShortConvolution(d_model, R, W)
        self.out = nn.Linear(d_model, d_model, bias=False)
        self._log_decay = None

    @property
    def log_decay(self) -> torch.Tensor:
        """[n_heads] float32 on the parameters' device whatever their type: not a buffer, which .to(dtype)
        would round.  Made where it is first used, from the number of heads alone: on the CPU, so that
        every device has the same bits, and outside inference mode, whose tensors no backward may keep."""
        device = self.qkv.weight.device
        if self._log_decay is None or self._log_decay.device != device:
            with torch.inference_mode(False):
                e = torch.linspace(5, 12, self.n_heads, dtype=torch.float64, device="cpu")
                self._log_decay = torch.log1p(-torch.exp2(-e)).float().to(device)
        return self._log_decay

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        y = self.conv.forward_fused(self.qkv(x), x)
        return self.out(decay_linear_attention_fused(y, self.log_decay))

    def prompt(self, x: torch.Tensor) -> tuple[torch.Tensor, LayerCache]:
        qkv = self.qkv(x)
        y = self.conv.forward_fused(qkv, x)
        o, state = decay_linear_attention_fused(y, self.log_decay, return_state=True)
        return self.out(o), LayerCache(convolution_cache(qkv, self.W), state, self.conv.stacked())

    def step(self, x: torch.Tensor, cache: LayerCache, slots: torch.Tensor | None = None) -> torch.Tensor:
        B, H = x.shape[0], self.n_heads
        y = self.conv.step(self.qkv(x), x, cache.conv, cache.stacked, slots)
        q, k, v = y.view(B, 3, H, self.d_model // H).unbind(1)
        o = decay_linear_attention_step(q, k, v, cache.state, self.log_decay, slots=slots)
        return self.out(o.view(B, self.d_model))


class ConvolvedGatedDelta(nn.Module):
    """A layer on the gated delta rule: one fused projection of queries, keys and values, the grouped
    low-rank dynamic convolution of its three thirds, queries and keys of length one, the rule with
    decays and rates that come from the input, a norm of each head's output under a gate, and an
    output projection.

    The decay of head h is exp(-exp(A_log[h]) softplus(a + dt_bias[h])), its rate sigmoid(b), with a and b
    linear in the input.  ``forward``, ``prompt`` and ``step`` are those of ``ConvolvedLinearAttention``.
    A head has at most 128 channels.
    """

    def __init__(self, d_model: int, n_heads: int, R: int = 15, W: int = 4):
        super().__init__()
        if d_model % n_heads != 0:
            raise ValueError("d_model must be divisible by n_heads")
        if d_model // n_heads > 128:
            raise ValueError("a head must have at most 128 channels")
        self.d_model, self.n_heads, self.d_head, self.W = d_model, n_heads, d_model // n_heads, W
        self.qkv = nn.Linear(d_model, 3 * d_model, bias=False)
        self.conv = QKVLowRankDynamicShortConvolution(d_model, R, W)
        self.gates = nn.Linear(d_model, 2 * n_heads, bias=False)
        # decay rates of 1 to 16 over the heads, steps of about 0.001 to 0.1
        self.A_log = nn.Parameter(torch.linspace(1, 16, n_heads).log())
        steps = torch.exp(torch.rand(n_heads) * math.log(100.0) + math.log(1e-3))
        self.dt_bias = nn.Parameter(steps + torch.log(-torch.expm1(-steps)))  # (softplus gives the steps)
        self.gate = nn.Linear(d_model, d_model, bias=False)
        self.norm = nn.Parameter(torch.ones(self.d_head))
        self.out = nn.Linear(d_model, d_model, bias=False)

    def _gates(self, x: torch.Tensor):
        """log decays and rates, [..., n_heads] float32 (a long memory's decay is lost between two numbers of bf16)."""
        a, b = self.gates(x).split(self.n_heads, -1)
        g = -torch.exp(self.A_log.float()) * torch.nn.functional.softplus(a.float() + self.dt_bias.float())
        return g, torch.sigmoid(b.float())

    def _heads(self, y: torch.Tensor):
        """Queries and keys of length one, and values, [..., n_heads, d_head], of the convolved [..., 3*d_model]."""
        qk, v = y.split([2 * self.d_model, self.d_model], -1)
        qk = gated_rms_norm(qk.unflatten(-1, (2 * self.n_heads, self.d_head)), scale=self.d_head**-0.5)
        q, k = qk.split(self.n_heads, -2)
        return q, k, v.unflatten(-1, (self.n_heads, self.d_head))

    def _finish(self, o: torch.Tensor, x: torch.Tensor) -> torch.Tensor:
        return self.out(gated_rms_norm(o, self.norm, self.gate(x).view(o.shape)).flatten(-2))

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return self._finish(gated_delta_rule(*self._heads(self.conv.forward_fused(self.qkv(x), x)), *self._gates(x)), x)

    def prompt(self, x: torch.Tensor) -> tuple[torch.Tensor, LayerCache]:
        qkv = self.qkv(x)
        o, state = gated_delta_rule(*self._heads(self.conv.forward_fused(qkv, x)), *self._gates(x), return_state=True)
        return self._finish(o, x), LayerCache(convolution_cache(qkv, self.W), state, self.conv.stacked())

    def step(self, x: torch.Tensor, cache: LayerCache, slots: torch.Tensor | None = None) -> torch.Tensor:
        q, k, v = self._heads(self.conv.step(self.qkv(x), x, cache.conv, cache.stacked, slots))
        o = gated_delta_rule_step(q, k, v, cache.state, *self._gates(x), slots=slots)
        return self._finish(o, x)


class ResidualRMSNorm(nn.Module):
    """Between two blocks: adds the one's output to the residual stream, times a learned scale per channel
    where ``layer_scale`` is given (its initial value), and normalises the sum for the other.
    forward(x, residual) returns (normalised, residual stream)."""

    def __init__(self, d_model: int, layer_scale: float | None = None, eps: float = 1e-6):
        super().__init__()
        self.weight = nn.Parameter(torch.ones(d_model))
        self.scale = None if layer_scale is None else nn.Parameter(torch.full((d_model,), float(layer_scale)))
        self.eps = eps

    def forward(self, x: torch.Tensor, residual: torch.Tensor):
        return residual_rms_norm(x, residual, self.weight, 1.0 if self.scale is None else self.scale, self.eps)
