"""GPU: the gated delta rule and the norms where other tests say little: batches of steps beyond 65535 heads, few columns of
many chains, gradients of views, gradients along their own direction, one channel."""
from __future__ import annotations

import pytest
import torch

from dynamic_conv1d_b200 import check_device, gated_delta_rule, gated_delta_rule_step, gated_rms_norm
from test_gpu_gated_delta import BF16, F32, F32_TOL, STEP, check, inputs, recurrence, rel
from test_gpu_norm import TOL, gated, rnd

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_step_of_more_heads_than_a_grid_dimension(dtype):
    """2048 sequences of 33 heads: 67584 states."""
    ts, S0, _, _ = inputs(2048, 1, 33, 8, 12, dtype, seed=1)
    ts, S = [t[:, 0] for t in ts], S0.clone()
    o = gated_delta_rule_step(*ts[:3], S, *ts[3:])
    ro, rS = recurrence(*(t[:, None].double() for t in ts), S0.double(), 8**-0.5)
    check_device(o)
    assert rel(o, ro[:, 0]) <= (2 * STEP if dtype == BF16 else F32_TOL) and rel(S, rS) <= F32_TOL


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("dk,dv", [(64, 16), (128, 16), (128, 32), (64, 48)])
def test_few_columns_of_many_chains(dtype, dk, dv):
    """Fewer slices of 16 columns than the teams that so many chains would have."""
    check(*inputs(4, 130, 50, dk, dv, dtype, seed=dv), states=dv != 32)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("dk,dv", [(64, 64), (128, 48), (13, 7)])
def test_gradients_of_views(dtype, dk, dv):
    """Tensors laid out otherwise have the gradients of dense ones, bit for bit, upstream gradients laid out otherwise too."""
    ts, S0, do, _ = inputs(2, 100, 4, dk, dv, dtype, seed=dk)

    def run(make, up):
        own = [t.detach().clone().requires_grad_() for t in ts]
        o = gated_delta_rule(*make(own), initial_state=S0)
        return [o.detach(), *torch.autograd.grad(o, own, up)]

    def fused(own):
        q, k, v, g, b = torch.cat([t.flatten(2) for t in own], -1).split([4 * dk, 4 * dk, 4 * dv, 4, 4], -1)
        return (*(t.unflatten(-1, (4, -1)) for t in (q, k, v)), g, b)

    heads_first = lambda own: [t.transpose(1, 2).contiguous().transpose(1, 2) for t in own]  # noqa: E731
    odd = lambda own: [torch.cat([t.flatten()[:1], t.flatten()])[1:].view(t.shape) for t in own]  # noqa: E731
    strided = lambda own: [torch.stack([t, t.detach()], -1)[..., 0] for t in own]  # noqa: E731
    want = run(lambda own: own, do)
    ups = [do, do.transpose(1, 2).contiguous().transpose(1, 2), torch.stack([do, do], -1)[..., 0],
           torch.cat([do.flatten()[:1], do.flatten()])[1:].view(do.shape)]
    for make in (fused, heads_first, odd, strided):
        for up in ups:
            assert all(torch.equal(a, b) for a, b in zip(run(make, up), want))
    one = do[:, :1, :1].expand(do.shape)
    assert all(torch.equal(a, b) for a, b in zip(run(fused, one), run(lambda own: own, one.contiguous())))


@pytest.mark.parametrize("which", range(6))
def test_gradients_along_themselves(which):
    """The slope of the definition along the kernels' gradient is that gradient's own length: a gradient off by a share of its
    size shows as that share.  In 64 bits a difference over 2e-4 of the tensor's size is off by some 1e-8 of the slope."""
    ts, S0, do, _ = inputs(1, 150, 2, 32, 32, F32, seed=12)
    own = [t.detach().requires_grad_() for t in (*ts, S0)]
    gated_delta_rule(*own[:5], initial_state=own[5]).backward(do)
    grad = own[which].grad.double()
    step = grad * (1e-4 * own[which].detach().double().norm() / grad.norm())
    f = lambda x: (recurrence(*x, 32**-0.5)[0] * do.double()).sum()  # noqa: E731
    with torch.no_grad():
        moved = [[t.double() + s * step if i == which else t.double() for i, t in enumerate((*ts, S0))] for s in (1, -1)]
        slope = ((f(moved[0]) - f(moved[1])) / 2).item()
    want = (grad * step).sum().item()
    assert want > 0 and abs(slope - want) <= 2 * F32_TOL * want


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_one_channel(dtype):
    """With eps of the size of x^2 the gradient of one channel is no difference of equal terms: (|x| <= 4) a sixteenth of them
    at least, so sixteen times a few roundings of 2^-24 before the result's own."""
    x, w, z, dy = (rnd(50, 3, 1, dtype=dtype, seed=i).clamp(-4, 4) if i != 1 else rnd(1, dtype=dtype, seed=1) for i in range(4))
    own, ref = [t.detach().clone().requires_grad_() for t in (x, w, z)], [t.detach().double().requires_grad_() for t in (x, w, z)]
    y, ry = gated_rms_norm(*own, eps=1.0, scale=0.7), gated(*ref, 1.0, 0.7)
    y.backward(dy)
    ry.backward(dy.double())
    assert rel(y, ry) <= TOL[dtype]
    for a, b in zip(own, ref):
        assert rel(a.grad, b.grad) <= TOL[dtype]
