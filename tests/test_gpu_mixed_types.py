"""GPU: float32 gates and norm weights beside bfloat16 tensors.  They are read as they are, and their gradients come back
in float32.

Tolerances.  An output in bf16 is rounded once, by at most 2^-8 of its value, after float32 arithmetic that is off by
less than 2^-16 (a hundred additions of 2^-24, the gate's quick exponential of 2^-21).  Gradients of weights are float32
sums: 128 * 2^-24 relative to the definition at the residual stream that the call returned.  The rule's: those of
``test_gpu_gated_delta``; its states are held to float32 whatever the tensors' type."""
from __future__ import annotations

import pytest
import torch

from dynamic_conv1d_b200 import ConvolvedGatedDelta, ResidualRMSNorm, check_device, gated_delta_rule, gated_delta_rule_step
from dynamic_conv1d_b200 import gated_rms_norm, residual_rms_norm
from test_gpu_gated_delta import F32_TOL, NAMES, STEP, inputs, recurrence, rel, tol
from test_gpu_norm import gated, residual, rnd

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
SUM_TOL = 128 * 2.0**-24


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


@pytest.mark.parametrize("N,D", [(80003, 64), (30001, 128), (9001, 520), (5003, 1024), (2502, 2048), (1203, 4096), (907, 8192), (331, 16384)])
def test_rows_in_turn(N, D):
    """So many rows that a CTA takes several, and its places in shared memory are used several times over.  Sums of up to
    80003 products, over at most 34 rows of a thread and 592 CTAs: under 256 additions of 2^-24 in a row."""
    x, z, dy, dh = (rnd(N, D, dtype=BF16, seed=i) for i in range(4))
    w, s = weights(D, 5), weights(D, 7) / 2
    wide = torch.cat([x, z], -1)  # (rows of two tensors side by side)
    own, ref = [t.detach().requires_grad_() for t in (wide, w)], [t.detach().double().requires_grad_() for t in (x, w, z)]
    gated_rms_norm(own[0][:, :D], own[1], own[0][:, D:]).backward(dy)
    gated(*ref, 1e-6, 1.0).backward(dy.double())
    for a, b in ((own[0].grad[:, :D], ref[0].grad), (own[0].grad[:, D:], ref[2].grad)):
        assert rel(a, b) <= 2 * STEP
    assert rel(own[1].grad, ref[1].grad) <= 256 * 2.0**-24
    own = [t.detach().requires_grad_() for t in (x, z, w, s)]
    y, h = residual_rms_norm(*own)
    torch.autograd.backward([y, h], [dy, dh])
    hd, wd = h.detach().double(), w.double()
    n = torch.rsqrt(hd.square().mean(-1, keepdim=True) + 1e-6)
    g = dy.double() * wd
    t = dh.double() + n * (g - hd * n.square() * (g * hd).mean(-1, keepdim=True))
    assert rel(own[1].grad, t) <= 2 * STEP and rel(own[0].grad, t * s.double()) <= 2 * STEP
    assert rel(own[2].grad, (dy.double() * hd * n).sum(0)) <= 256 * 2.0**-24
    assert rel(own[3].grad, (t * x.double()).sum(0)) <= 256 * 2.0**-24


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


@pytest.mark.parametrize("dk,dv,T", [(64, 64, 1), (64, 64, 63), (128, 128, 200), (13, 7, 130), (32, 96, 1200)])
@pytest.mark.parametrize("states", [True, False])
def test_rule(dk, dv, T, states):
    """Gates in float32, views of a wider tensor among them."""
    ts, S0, do, dS = inputs(2, T, 3, dk, dv, BF16, seed=T, decay=0.02)
    gates = torch.cat([-0.02 * torch.nn.functional.softplus(rnd(2, T, 3, seed=1)), torch.sigmoid(rnd(2, T, 3, seed=2))], -1)
    own = [t.detach().requires_grad_() for t in (*ts[:3], gates)]
    s_own = S0.detach().requires_grad_() if states else None
    out = gated_delta_rule(*own[:3], *own[3].split(3, -1), initial_state=s_own, return_state=states)
    o, S = out if states else (out, None)
    torch.autograd.backward([o, S] if states else [o], [do, dS] if states else [do])
    ref = [t.detach().double().requires_grad_() for t in (*ts[:3], gates)]
    s_ref = (S0 if states else torch.zeros_like(S0)).double().requires_grad_()
    ro, rS = recurrence(*ref[:3], *ref[3].split(3, -1), s_ref, dk**-0.5)
    torch.autograd.backward([ro, rS] if states else [ro], [do.double(), dS.double()] if states else [do.double()])
    check_device(o)
    assert rel(o, ro) <= tol("o", BF16)
    if states:
        assert rel(S, rS) <= F32_TOL and rel(s_own.grad, s_ref.grad) <= F32_TOL
    for n, a, b in zip(NAMES, own[:3], ref):
        assert rel(a.grad, b.grad) <= tol("d" + n, BF16), n
    assert own[3].grad.dtype == F32
    for n, a, b in zip(("dlog_decay", "dbeta"), own[3].grad.split(3, -1), ref[3].grad.split(3, -1)):
        assert rel(a, b) <= tol(n, BF16), n


def test_rule_gates_that_bf16_holds():
    """Gates that both types hold give the same bits."""
    ts, S0, do, _ = inputs(2, 150, 4, 128, 128, BF16, seed=3)
    grads = []
    for gate in (BF16, F32):
        own = [t.detach().to(gate if i > 2 else BF16).requires_grad_() for i, t in enumerate(ts)]
        o, S = gated_delta_rule(*own, initial_state=S0, return_state=True)
        o.backward(do)
        grads.append([o, S, *(t.grad.bfloat16() for t in own)])
    assert all(torch.equal(a, b) for a, b in zip(*grads))


@pytest.mark.parametrize("dk,dv", [(128, 128), (64, 64), (37, 51)])
def test_step(dk, dv):
    ts, S0, _, _ = inputs(5, 40, 3, dk, dv, BF16, seed=dk)
    g, beta = -0.02 * torch.nn.functional.softplus(rnd(5, 40, 3, seed=1)), torch.sigmoid(rnd(5, 40, 3, seed=2))
    S = S0.clone()
    got = torch.stack([gated_delta_rule_step(*(x[:, t] for x in ts[:3]), S, g[:, t], beta[:, t]) for t in range(40)], 1)
    ro, rS = recurrence(*(t.double() for t in (*ts[:3], g, beta)), S0.double(), dk**-0.5)
    assert rel(got, ro) <= 2 * STEP and rel(S, rS) <= F32_TOL


def test_gates_of_two_types_are_refused():
    ts, S0, _, _ = inputs(1, 4, 2, 16, 16, BF16)
    for g, b in ((ts[3].float(), ts[4]), (ts[3], ts[4].float()), (ts[3].double(), ts[4].double()), (ts[3].half(), ts[4].half())):
        with pytest.raises(AssertionError):
            gated_delta_rule(*ts[:3], g, b)
        with pytest.raises(AssertionError):
            gated_delta_rule_step(*(t[:, 0] for t in ts[:3]), S0.clone(), g[:, 0], b[:, 0])


def test_layer():
    """The layer hands its decays on in float32, and float32 norm weights serve a bf16 model."""
    torch.manual_seed(0)
    m = ConvolvedGatedDelta(128, 2).cuda().bfloat16()
    m.A_log.data, m.dt_bias.data, m.norm.data = m.A_log.data.float(), m.dt_bias.data.float(), m.norm.data.float()
    x = torch.randn(2, 50, 128, device="cuda", dtype=BF16)
    g, beta = m._gates(x)
    a, b = m.gates(x).double().split(2, -1)
    want = -torch.exp(m.A_log.double()) * torch.nn.functional.softplus(a + m.dt_bias.double())
    assert g.dtype == beta.dtype == F32
    # (float32 exponentials, logarithms and a product, a few 2^-24 each; of a decay's logarithm near -1e-3 to -1)
    assert rel(g, want) <= 2.0**-20 and rel(beta, torch.sigmoid(b)) <= 2.0**-20
    m(x).float().square().mean().backward()
    assert all(p.grad is not None and p.grad.dtype == p.dtype and p.grad.isfinite().all() for p in m.parameters())
