"""GPU: float32 norm weights beside bfloat16 tensors.  They are read as they are, and their gradients come back in float32.

Tolerances.  An output in bf16 is rounded once, by at most 2^-8 of its value, after float32 arithmetic that is off by
less than 2^-16 (a hundred additions of 2^-24, the gate's quick exponential of 2^-21).  Gradients of weights are float32
sums: 128 * 2^-24 relative to the definition at the residual stream that the call returned."""
from __future__ import annotations

import pytest
import torch

from dynamic_conv1d_b200 import ResidualRMSNorm, gated_rms_norm, residual_rms_norm
from test_gpu_norm import gated, rel, residual, rnd

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
STEP, SUM_TOL = 2.0**-9, 128 * 2.0**-24


def weights(D, seed):
    """float32 numbers next to the middle between two of bf16: 2^-8 is lost where they are rounded."""
    return 1 + 2.0**-8 * (1 - 2.0**-6) + 2.0**-7 * rnd(D, seed=seed).round()


def once_rounded(y, ref, terms=0.0):
    """terms: the size of what may have cancelled in the result, in float32."""
    return bool(((y.detach().double() - ref.detach()).abs() <= (2.0**-8 + 2.0**-16) * ref.detach().abs() + 2.0**-22 * terms).all())


@pytest.mark.parametrize("D", [1, 7, 32, 99, 128, 512, 513, 1000, 2048, 2050, 4097, 16384])
@pytest.mark.parametrize("with_z", [True, False])
def test_gated(D, with_z):
    N = 70 if D < 3000 else 5
    x, w, dy = rnd(N, 3, D, dtype=BF16, seed=1), weights(D, 2), rnd(N, 3, D, dtype=BF16, seed=4)
    z = rnd(N, 3, D, dtype=BF16, seed=3) if with_z else None
    leaves = [x, w, z] if with_z else [x, w]
    own, ref = [t.detach().clone().requires_grad_() for t in leaves], [t.detach().double().requires_grad_() for t in leaves]
    y, ry = gated_rms_norm(*own, eps=0.5, scale=0.7), gated(ref[0], ref[1], ref[2] if with_z else None, 0.5, 0.7)
    assert y.dtype == BF16 and once_rounded(y, ry)
    y.backward(dy)
    ry.backward(dy.double())
    assert own[1].grad.dtype == F32 and rel(own[1].grad, ref[1].grad) <= SUM_TOL
    for a, b in zip(own, ref):
        assert rel(a.grad, b.grad) <= 2 * STEP


@pytest.mark.parametrize("D", [1, 7, 32, 99, 128, 512, 513, 1000, 2048, 2050, 4097, 16384])
@pytest.mark.parametrize("scale", ["channels", "bf16 channels", 0.5])
def test_residual(D, scale):
    N = 210 if D < 3000 else 7
    x, r, dy, dh = (rnd(N, D, dtype=BF16, seed=i) for i in range(4))
    w, s = weights(D, 5), weights(D, 7) / 2
    if scale == "bf16 channels":
        s = s.bfloat16()
    leaves = (x, r, w) if scale == 0.5 else (x, r, w, s)
    own, ref = [t.detach().clone().requires_grad_() for t in leaves], [t.detach().double().requires_grad_() for t in leaves]
    at = lambda t: scale if scale == 0.5 else t[3]  # noqa: E731
    y, h = residual_rms_norm(*own[:3], at(own))
    ry, rh = residual(*ref[:3], at(ref), 1e-6)
    with torch.no_grad():
        terms = (at(ref) * ref[0]).abs() + ref[1].abs()
        assert once_rounded(h, rh, terms)
        assert once_rounded(y, ry, terms * torch.rsqrt(rh.square().mean(-1, keepdim=True) + 1e-6) * ref[2].abs())
    torch.autograd.backward([y, h], [dy, dh])
    hd, wd = h.detach().double(), w.double()
    n = torch.rsqrt(hd.square().mean(-1, keepdim=True) + 1e-6)
    g = dy.double() * wd
    t = dh.double() + n * (g - hd * n.square() * (g * hd).mean(-1, keepdim=True))
    assert own[2].grad.dtype == F32 and rel(own[2].grad, (dy.double() * hd * n).sum(0)) <= SUM_TOL
    assert rel(own[1].grad, t) <= 2 * STEP and rel(own[0].grad, t * (scale if scale == 0.5 else s.double())) <= 2 * STEP
    if scale == "channels":
        assert own[3].grad.dtype == F32 and rel(own[3].grad, (t * x.double()).sum(0)) <= SUM_TOL
    elif scale == "bf16 channels":
        assert own[3].grad.dtype == BF16 and rel(own[3].grad, (t * x.double()).sum(0)) <= 2 * STEP


def test_weights_off_16_bytes_and_casts():
    """A float32 weight at any address; one of another type is cast to float32; bf16 beside bf16 stays as it was."""
    x, r, w = rnd(9, 64, dtype=BF16), rnd(9, 64, dtype=BF16, seed=1), weights(64, 2)
    odd = torch.cat([w[:1], w])[1:]
    assert odd.data_ptr() % 16
    assert rel(gated_rms_norm(x, odd), gated(x.double(), w.double(), None, 1e-6, 1.0)) <= 2 * STEP
    want = gated_rms_norm(x, w)
    assert torch.equal(gated_rms_norm(x, w.double()), want)
    half = (1 + rnd(64, seed=3) / 4).half()
    assert torch.equal(gated_rms_norm(x, half), gated_rms_norm(x, half.float()))
    assert torch.equal(residual_rms_norm(x, r, w, w.double())[0], residual_rms_norm(x, r, w, w)[0])
    w32 = w.bfloat16().float()
    assert torch.equal(gated_rms_norm(x.float(), w.bfloat16()), gated_rms_norm(x.float(), w32))
    assert torch.equal(gated_rms_norm(x, w.bfloat16()), gated_rms_norm(x, w32))
    a = w.detach().requires_grad_()
    gated_rms_norm(x[:0], a).sum().backward()  # (no row)
    assert a.grad.dtype == F32 and not a.grad.any()


def test_module():
    norm = ResidualRMSNorm(128, layer_scale=0.1).cuda()
    x = rnd(5, 128, dtype=BF16)
    y, h = norm(x, x)
    (y.float().sum() + h.float().sum()).backward()
    assert y.dtype == BF16 and norm.weight.grad.dtype == F32 and norm.scale.grad.isfinite().all()
