"""GPU: calls of the gated delta rule, the norms and the single-token steps that autograd watches without asking for a
gradient: inputs with a tangent (forward-mode differentiation) and calls under ``torch.jit.trace``."""
from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

from dynamic_conv1d_b200 import (
    decay_linear_attention_step,
    gated_delta_rule,
    gated_delta_rule_step,
    gated_rms_norm,
    headwise_dynamic_convolution_step,
    lowrank_dynamic_convolution_grouped_step,
    lowrank_dynamic_convolution_step,
    residual_rms_norm,
)

pytestmark = [pytest.mark.gpu, pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning")]


def rnd(*shape, seed=0):
    return torch.randn(*shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed))


def rule_inputs(T=70, seed=0):
    q, k = (torch.nn.functional.normalize(rnd(2, T, 3, 32, seed=seed + i), dim=-1) for i in range(2))
    return [q, k, rnd(2, T, 3, 16, seed=seed + 2), -torch.rand(2, T, 3, device="cuda"), torch.rand(2, T, 3, device="cuda")]


# name -> (call, inputs of `n` rows or tokens)
CALLS = {
    "rule": (lambda q, k, v, g, b: gated_delta_rule(q, k, v, g, b), lambda n, s: rule_inputs(n, s)),
    "rule_state": (lambda q, k, v, g, b, S: gated_delta_rule(q, k, v, g, b, S, 0.5, True),
                   lambda n, s: [*rule_inputs(n, s), rnd(2, 3, 32, 16, seed=s + 9)]),
    "length": (lambda x: gated_rms_norm(x, scale=0.25), lambda n, s: [rnd(n, 3, 48, seed=s)]),
    "gated": (lambda x, w, z: gated_rms_norm(x, w, z), lambda n, s: [rnd(n, 3, 48, seed=s), rnd(48, seed=s + 1), rnd(n, 3, 48, seed=s + 2)]),
    "residual": (lambda x, r, w, s: residual_rms_norm(x, r, w, s),
                 lambda n, s: [rnd(n, 96, seed=s), rnd(n, 96, seed=s + 1), rnd(96, seed=s + 2), rnd(96, seed=s + 3)]),
    "residual_factor": (lambda x, r, w: residual_rms_norm(x, r, w, 0.5),
                        lambda n, s: [rnd(n, 96, seed=s), rnd(n, 96, seed=s + 1), rnd(96, seed=s + 2)]),
}
STEPS = {
    "delta": (lambda q, k, v, S, g, b: gated_delta_rule_step(q, k, v, S, g, b),
              lambda: [rnd(2, 3, 32), rnd(2, 3, 32), rnd(2, 3, 16), rnd(2, 3, 32, 16), -torch.rand(2, 3, device="cuda"), torch.rand(2, 3, device="cuda")]),
    "attention": (lambda q, k, v, S: decay_linear_attention_step(q, k, v, S, torch.full((3,), -0.1, device="cuda")),
                  lambda: [rnd(2, 3, 32), rnd(2, 3, 32), rnd(2, 3, 16), rnd(2, 3, 32, 16)]),
    "lowrank": (lambda x, z, U, c, w: lowrank_dynamic_convolution_step(x, z, U, c, w),
                lambda: [rnd(2, 64), rnd(2, 7), rnd(7, 256), rnd(2, 3, 64), rnd(4, 64)]),
    "grouped": (lambda x, z, U, c: lowrank_dynamic_convolution_grouped_step(x, z, U, c),
                lambda: [rnd(2, 128), rnd(2, 14), rnd(2, 7, 256), rnd(2, 3, 128)]),
    "headwise": (lambda x, w, c, s: headwise_dynamic_convolution_step(x, w, c, s),
                 lambda: [rnd(2, 64), rnd(2, 8, 4), rnd(2, 3, 64), rnd(4, 64)]),
}


def outputs(y):
    return y if isinstance(y, tuple) else (y,)


@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("name", CALLS)
def test_a_tangent_is_refused(name, grad):
    """The operators have no forward-mode derivative: a tangent is an error, never a derivative of zero."""
    call, make = CALLS[name]
    args = make(20, 0)
    with torch.set_grad_enabled(grad), forward_ad.dual_level():
        for i in range(len(args)):
            dual = [forward_ad.make_dual(t, torch.ones_like(t)) if j == i else t for j, t in enumerate(args)]
            with pytest.raises(NotImplementedError, match="jvp"):
                call(*dual)
        assert all(torch.equal(a, b) for a, b in zip(outputs(call(*args)), outputs(call(*args))))  # (none has a tangent)


@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("name", CALLS)
def test_traced(name, grad):
    """A traced call runs the operator again, on inputs of other values and lengths, and has its gradients."""
    call, make = CALLS[name]
    with torch.set_grad_enabled(grad):
        traced = torch.jit.trace(call, make(20, 0), check_trace=False)
    for n in (20, 33):
        args = make(n, 50)
        got, want = outputs(traced(*args)), outputs(call(*args))
        assert len(got) == len(want) and all(torch.equal(a, b) for a, b in zip(got, want))
    a, b = ([t.detach().clone().requires_grad_() for t in args] for _ in range(2))
    for f, leaves in ((traced, a), (call, b)):
        sum(y.sum() for y in outputs(f(*leaves))).backward()
    assert all(torch.equal(x.grad, y.grad) for x, y in zip(a, b))


@pytest.mark.parametrize("name", STEPS)
def test_steps_refuse_both(name):
    """A step has neither a derivative of either kind nor a record of what it updates."""
    call, make = STEPS[name]
    args = make()
    before = [t.clone() for t in args]
    with torch.no_grad(), forward_ad.dual_level():
        for i in range(len(args)):
            dual = [forward_ad.make_dual(t, torch.ones_like(t)) if j == i else t for j, t in enumerate(args)]
            with pytest.raises(RuntimeError, match="no gradient"):
                call(*dual)
    with torch.no_grad(), pytest.raises(RuntimeError, match="trace"):
        torch.jit.trace(call, args, check_trace=False)
    assert all(torch.equal(a, b) for a, b in zip(args, before))  # (nothing ran)
    with forward_ad.dual_level():  # (a level in which no input has a tangent is no concern of theirs)
        y = call(*args)
    assert y.isfinite().all()
