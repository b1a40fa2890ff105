"""GPU: the attention layer built on the convolutions and linear attention, and the example
model that trains and generates with it.

The layer in bf16 against the same layer from elementary operations in 64 bits: five bf16
results feed one another (projection, convolution, attention, output projection and the
attention's two rounded operands), each off by less than 2^-9 of its values in the root mean
square; 2^-6 bounds their sum with room for the projections' amplification."""
from __future__ import annotations

import importlib.util
import os

import pytest
import torch

from conftest import ROOT
from dynamic_conv1d_b200 import ConvolvedLinearAttention, check_device

pytestmark = pytest.mark.gpu


def rel(a, b):
    a, b = a.detach().double(), b.detach().double()
    return (torch.linalg.vector_norm(a - b) / torch.linalg.vector_norm(b)).item()


def layer(d_model=256, heads=4, R=15, W=4):
    torch.manual_seed(0)
    m = ConvolvedLinearAttention(d_model, heads, R, W).cuda()
    for c in (m.conv.q, m.conv.k, m.conv.v):
        torch.nn.init.normal_(c.proj_out, std=0.3)
    return m.to(torch.bfloat16)


def definition(m, x):
    B, T, D = x.shape
    H, W = m.n_heads, m.W
    f = lambda p: p.detach().double()  # noqa: E731
    qkv = x @ f(m.qkv.weight).T
    parts = []
    for i, c in enumerate((m.conv.q, m.conv.k, m.conv.v)):
        u = qkv[..., i * D:(i + 1) * D]
        w = ((x @ f(c.proj_in.weight).T) @ f(c.proj_out)).view(B, T, W, D) + f(c.proj_out_bias)
        y = u.clone()
        for k in range(W):
            y = y + w[:, :, k] * torch.nn.functional.pad(u, (0, 0, k, 0))[:, :T]
        parts.append(y.view(B, T, H, D // H))
    q, k, v = parts
    g = torch.exp(m.log_decay.double())[:, None, None]
    S = torch.zeros(B, H, D // H, D // H, device=x.device, dtype=torch.float64)
    out = []
    for t in range(T):
        S = S * g + k[:, t, :, :, None] * v[:, t, :, None, :]
        out.append((q[:, t, :, None, :] @ S).squeeze(-2) * (D // H) ** -0.5)
    return torch.stack(out, 1).reshape(B, T, D) @ f(m.out.weight).T


@pytest.mark.parametrize("d_model,heads,W", [(256, 4, 4), (128, 2, 3), (96, 3, 2)])
def test_layer_against_its_definition(d_model, heads, W):
    m = layer(d_model, heads, W=W)
    x = torch.randn(2, 75, d_model, device="cuda").bfloat16()
    y = m(x)
    check_device(y)
    assert rel(y, definition(m, x.double())) <= 2.0**-6
    assert m.log_decay.dtype == torch.float32
    y.float().square().mean().backward()
    assert all(p.grad is not None and p.grad.isfinite().all() for p in m.parameters())


@pytest.mark.parametrize("T", [1, 2, 30, 130])
def test_prompt_and_steps(T):
    m = layer()
    x = torch.randn(3, T + 5, 256, device="cuda").bfloat16()
    with torch.no_grad():
        whole = m(x)
        y, cache = m.prompt(x[:, :T])
        rest = [m.step(x[:, t], cache) for t in range(T, T + 5)]
    assert rel(torch.cat([y, torch.stack(rest, 1)], 1), whole) <= 2.0**-6


def test_slots():
    m = layer()
    x = torch.randn(4, 9, 256, device="cuda").bfloat16()
    with torch.no_grad():
        _, cache = m.prompt(x[:, :8])
        want = m.step(x[:, 8], cache)
        _, pool = m.prompt(x[:, :8].flip(0))
        got = m.step(x[:, 8], pool, slots=torch.tensor([3, 2, 1, 0], device="cuda"))
    assert torch.equal(got, want)


def test_example_learns_and_generates(capsys):
    spec = importlib.util.spec_from_file_location("linear_attention_lm", os.path.join(ROOT, "examples", "linear_attention_lm.py"))
    lm = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(lm)
    first, last, right = lm.main(["--steps", "200"])
    assert first > 5.0  # about log(500): the model starts ignorant
    assert last < 1.5 and right > 0.8


def test_training_after_evaluation_in_inference_mode():
    """The layer's first use on a device may be under inference mode."""
    x = torch.randn(2, 40, 256, device="cuda").bfloat16()
    m = layer()
    want = layer()(x)
    with torch.inference_mode():
        y, cache = m.prompt(x)
        m.step(x[:, 0], cache)
    assert torch.equal(y, want)
    m(x).float().square().mean().backward()
    assert all(p.grad is not None and p.grad.isfinite().all() for p in m.parameters())
