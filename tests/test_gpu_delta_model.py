"""GPU: the layer on the gated delta rule as a model uses it, convolutions, norms, rule and gates together, and the example
that trains and generates with it.

The layer in bf16 against the same layer from elementary operations in 64 bits: eight bf16 results feed one another
(projection, convolution, lengths, gates, rule, gate, norm, output projection), each off by less than 2^-9 of its values
in the root mean square, the rule's with two rounded operands: 2^-6 bounds their sum of ten.  The log decays' own rounding
moves a state by 2^-9 of its decay's logarithm."""
from __future__ import annotations

import importlib.util
import os

import pytest
import torch

from conftest import ROOT
from dynamic_conv1d_b200 import ConvolvedGatedDelta, ResidualRMSNorm, check_device

pytestmark = pytest.mark.gpu


def rel(a, b):
    a, b = a.detach().double(), b.detach().double()
    return (torch.linalg.vector_norm(a - b) / torch.linalg.vector_norm(b)).item()


def layer(d_model=256, heads=4, R=15, W=4, dtype=torch.bfloat16):
    torch.manual_seed(0)
    m = ConvolvedGatedDelta(d_model, heads, R, W).cuda()
    for c in (m.conv.q, m.conv.k, m.conv.v):
        torch.nn.init.normal_(c.proj_out, std=0.3)
    return m.to(dtype)


def definition(m, x, p):
    """The layer in the type of x from its parameters p (name -> tensor), token by token."""
    B, T, D = x.shape
    H, d, W = m.n_heads, m.d_head, m.W
    qkv = x @ p["qkv.weight"].T
    parts = []
    for i, c in enumerate("qkv"):
        u = qkv[..., i * D:(i + 1) * D]
        w = ((x @ p[f"conv.{c}.proj_in.weight"].T) @ p[f"conv.{c}.proj_out"]).view(B, T, W, D) + p[f"conv.{c}.proj_out_bias"]
        y = u.clone()
        for k in range(W):
            y = y + w[:, :, k] * torch.nn.functional.pad(u, (0, 0, k, 0))[:, :T]
        parts.append(y.view(B, T, H, d))
    q, k, v = parts
    q, k = (t * torch.rsqrt(t.square().mean(-1, keepdim=True) + 1e-6) * d**-0.5 for t in (q, k))
    a, b = (x @ p["gates.weight"].T).split(H, -1)
    g = -torch.exp(p["A_log"]) * torch.nn.functional.softplus(a + p["dt_bias"])
    beta = torch.sigmoid(b)
    S = torch.zeros(B, H, d, d, device=x.device, dtype=x.dtype)
    out = []
    for t in range(T):
        S = S * torch.exp(g[:, t])[..., None, None]
        u = beta[:, t, :, None] * (v[:, t] - (k[:, t, :, None, :] @ S).squeeze(-2))
        S = S + k[:, t, :, :, None] * u[..., None, :]
        out.append((q[:, t, :, None, :] @ S).squeeze(-2) * d**-0.5)
    o = torch.stack(out, 1)
    z = (x @ p["gate.weight"].T).view(B, T, H, d)
    o = o * torch.rsqrt(o.square().mean(-1, keepdim=True) + 1e-6) * p["norm"] * torch.nn.functional.silu(z)
    return o.reshape(B, T, D) @ p["out.weight"].T


@pytest.mark.parametrize("d_model,heads,W", [(256, 4, 4), (128, 2, 3), (96, 3, 2)])
def test_layer_against_its_definition(d_model, heads, W):
    m = layer(d_model, heads, W=W)
    x = torch.randn(2, 150, d_model, device="cuda", dtype=torch.bfloat16)
    y = m(x)
    check_device(y)
    assert rel(y, definition(m, x.double(), {n: t.detach().double() for n, t in m.named_parameters()})) <= 2.0**-6


def test_gradients_against_the_definition():
    """In fp32, so that every parameter's gradient can be held to the formulas': 1e-4 for chains of ten sums of at most 512 products of
    2^-24 each (3e-4 if all were to add up), with the decays' derivative among them."""
    m = layer(64, 2, dtype=torch.float32)
    x = torch.randn(2, 70, 64, device="cuda")
    dy = torch.randn(2, 70, 64, device="cuda")
    xo = x.clone().requires_grad_()
    torch.backends.cuda.matmul.allow_tf32 = False
    m(xo).backward(dy)
    p = {n: t.detach().double().requires_grad_() for n, t in m.named_parameters()}
    xr = x.double().requires_grad_()
    definition(m, xr, p).backward(dy.double())
    assert rel(xo.grad, xr.grad) <= 1e-4
    for n, t in m.named_parameters():
        assert rel(t.grad, p[n].grad) <= 1e-4, n


@pytest.mark.parametrize("T", [2, 64, 100])
def test_prompt_and_steps(T):
    m = layer()
    x = torch.randn(3, T + 6, 256, device="cuda", dtype=torch.bfloat16)
    with torch.no_grad():
        whole = m(x)
        y, cache = m.prompt(x[:, :T])
        steps = torch.stack([m.step(x[:, t], cache) for t in range(T, T + 6)], 1)
    assert rel(y, whole[:, :T]) <= 2.0**-6 and rel(steps, whole[:, T:]) <= 2.0**-6


def test_slots():
    m = layer()
    x = torch.randn(3, 20, 256, device="cuda", dtype=torch.bfloat16)
    with torch.no_grad():
        _, cache = m.prompt(x[:, :-1])
        own = m.step(x[:, -1], cache)
        _, cache = m.prompt(x[:, :-1])
        pool = type(cache)(torch.zeros(5, *cache.conv.shape[1:], device="cuda", dtype=torch.bfloat16),
                           torch.zeros(5, *cache.state.shape[1:], device="cuda"), cache.stacked)
        rows = torch.tensor([4, 0, 2], device="cuda", dtype=torch.int32)
        pool.conv[rows.long()], pool.state[rows.long()] = cache.conv, cache.state
        assert torch.equal(m.step(x[:, -1], pool, slots=rows), own)


def test_padded_batch():
    """What stands behind the end of a sequence, even what is not finite, does not reach its tokens."""
    m = layer()
    x = torch.randn(2, 90, 256, device="cuda", dtype=torch.bfloat16)
    with torch.no_grad():
        want = m(x[:, :70].contiguous())
        x[:, 70:] = float("nan")
        got = m(x)
    assert rel(got[:, :70], want) <= 2.0**-6


def test_residual_norm_module():
    m = ResidualRMSNorm(128, layer_scale=0.1).cuda().bfloat16()
    x, r = (torch.randn(5, 7, 128, device="cuda", dtype=torch.bfloat16, requires_grad=True) for _ in range(2))
    y, h = m(x, r)
    want = r.double() + 0.1 * x.double()
    assert rel(h, want) <= 2.0**-8
    assert rel(y, want * torch.rsqrt(want.square().mean(-1, keepdim=True) + 1e-6)) <= 2.0**-7
    (y.sum() + h.sum()).backward()
    assert all(t.grad is not None and t.grad.isfinite().all() for t in (x, r, m.weight, m.scale))
    assert ResidualRMSNorm(128).scale is None


def test_example_runs(capsys):
    path = os.path.join(ROOT, "examples", "linear_attention_lm.py")
    spec = importlib.util.spec_from_file_location("linear_attention_lm", path)
    lm = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(lm)
    model = lm.LanguageModel(50, 64, 2, 2, layer="delta").cuda().bfloat16()
    loss = model.loss(torch.randint(0, 50, (4, 33), device="cuda"))
    loss.backward()
    assert loss.isfinite()
    for n, p in model.named_parameters():
        assert p.grad is not None and p.grad.isfinite().all(), n
    first, last, _ = lm.main(["--steps", "3", "--generate", "4", "--layer", "delta"])
    assert first > 0 and last > 0
    assert "loss" in capsys.readouterr().out
