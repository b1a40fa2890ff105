"""GPU: the gated delta rule against the recurrence in 64 bits.

Tolerances are relative 2-norms, set from the roundings the operator makes:
  bf16: a rounding to eight bits is off by at most 2^-8 of a value and by less than 2^-9 of it in the root
        mean square; outputs are rounded once, after products in which one operand (the scores, or the
        state) was: 3 * 2^-9.  Gradients of q, k and v: one more rounding, of the gradient of the state: 4 * 2^-9;
        the gradient of the log decays is a sum of four such terms of either sign: 8 * 2^-9;
  fp32: sums of up to 512 products, each addition at most 2^-24: 512 * 2^-24 = 3.1e-5 is the bound if all were to
        add up;
  states (always fp32, from bf16 or fp32 inputs): the same fp32 bound.
"""
from __future__ import annotations

import pytest
import torch

from dynamic_conv1d_b200 import DynconvError, check_device, gated_delta_rule, gated_delta_rule_step

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
STEP, F32_TOL = 2.0**-9, 512 * 2.0**-24
NAMES = ("q", "k", "v", "log_decay", "beta")


def tol(name, dtype):
    if dtype == F32 or name in ("state", "dstate"):
        return F32_TOL
    return {"o": 3, "dlog_decay": 8}.get(name, 4) * STEP


def rel(a, b):
    a, b = a.detach().double(), b.detach().float().double()
    n, d = torch.linalg.vector_norm(b), torch.linalg.vector_norm(a - b)
    return (d / n if n > 0 else d).item()


def recurrence(q, k, v, g, beta, S, scale):
    """The definition, token by token; differentiable, in the tensors' type (64 bits here)."""
    out = []
    for t in range(q.shape[1]):
        P = S * torch.exp(g[:, t])[..., None, None]
        u = beta[:, t, :, None] * (v[:, t] - (k[:, t, :, None, :] @ P).squeeze(-2))
        S = P + k[:, t, :, :, None] * u[..., None, :]
        out.append(scale * (q[:, t, :, None, :] @ S).squeeze(-2))
    return torch.stack(out, 1), S


def inputs(B, T, H, dk, dv, dtype, seed=0, decay=0.1):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, device="cuda", generator=gen)  # noqa: E731
    unit = lambda *s: torch.nn.functional.normalize(r(*s) + 0.3, dim=-1)  # noqa: E731
    q, k, v = unit(B, T, H, dk), unit(B, T, H, dk), r(B, T, H, dv)
    g, beta = -decay * torch.nn.functional.softplus(r(B, T, H)), torch.sigmoid(r(B, T, H))
    return [t.to(dtype) for t in (q, k, v, g, beta)], r(B, H, dk, dv), r(B, T, H, dv).to(dtype), r(B, H, dk, dv)


def check(ts, S0, do, dS, scale=None, states=True):
    """Outputs and all gradients of one call; states: with an initial and a final state."""
    dtype, sc = ts[0].dtype, ts[0].shape[-1] ** -0.5 if scale is None else scale
    own = [t.detach().requires_grad_() for t in ts]
    s_own = S0.detach().requires_grad_() if states else None
    out = gated_delta_rule(*own, initial_state=s_own, scale=scale, return_state=states)
    o, S = out if states else (out, None)
    torch.autograd.backward([o, S] if states else [o], [do, dS] if states else [do])
    ref = [t.detach().double().requires_grad_() for t in ts]
    s_ref = (S0 if states else torch.zeros_like(S0)).double().requires_grad_()
    ro, rS = recurrence(*ref, s_ref, sc)
    torch.autograd.backward([ro, rS] if states else [ro], [do.double(), dS.double()] if states else [do.double()])
    check_device(o)
    err = {"o": rel(o, ro)}
    if states:
        err["state"], err["dstate"] = rel(S, rS), rel(s_own.grad, s_ref.grad)
    err.update({"d" + n: rel(a.grad, b.grad) for n, a, b in zip(NAMES, own, ref)})
    bad = {n: (e, tol(n, dtype)) for n, e in err.items() if not e <= tol(n, dtype)}
    assert not bad, bad
    return o


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("T", [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 200])
def test_lengths(dtype, T):
    check(*inputs(2, T, 3, 64, 64, dtype, seed=T))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("dk,dv", [(128, 128), (64, 128), (128, 64), (32, 96), (80, 72), (16, 16), (8, 8), (1, 1), (13, 7),
                                   (65, 33), (100, 256), (128, 250), (127, 129)])
def test_widths(dtype, dk, dv):
    check(*inputs(2, 100, 2, dk, dv, dtype, seed=dk + dv))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("B,H", [(1, 1), (1, 20), (3, 50), (2, 100)])
def test_teams_and_stages(dtype, B, H):
    """Few and many chains: four warps for a slice of the state or two, one slice for a CTA to four."""
    check(*inputs(B, 140, H, 128, 128, dtype, seed=B + H), states=H != 50)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("decay", [0.0, 1e-4, 3.0, 60.0])
def test_decays(dtype, decay):
    check(*inputs(2, 150, 3, 64, 64, dtype, seed=5, decay=decay))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_forgetting_at_once(dtype):
    """A log decay of minus infinity starts anew; far ones of the same chunk keep their digits."""
    ts, S0, do, dS = inputs(1, 150, 2, 64, 64, dtype, seed=6)
    with torch.no_grad():
        ts[3][:, [0, 40, 41, 100]] = -torch.inf
    o, S = gated_delta_rule(*ts, initial_state=S0, return_state=True)
    ro, rS = recurrence(*(t.double() for t in ts), S0.double(), 64**-0.5)
    assert rel(o, ro) <= tol("o", dtype) and rel(S, rS) <= F32_TOL
    with torch.no_grad():
        ts[3][:, [0, 40, 41, 100]] = -1e4
    check(ts, S0, do, dS)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_rates_of_zero_and_one(dtype):
    """Padding tokens have a rate of zero: no update, and still the gradient of the rate."""
    ts, S0, do, dS = inputs(2, 90, 2, 64, 32, dtype, seed=7)
    with torch.no_grad():
        ts[4][:, ::3] = 0.0
        ts[4][:, 1::3] = 1.0
    check(ts, S0, do, dS)


def test_long():
    ts, S0, do, dS = inputs(1, 1500, 2, 128, 128, BF16, seed=8, decay=0.01)
    check(ts, S0, do, dS)
    check(*inputs(1, 700, 2, 128, 128, F32, seed=8, decay=0.01))


def test_scale_and_defaults():
    ts, S0, do, dS = inputs(2, 70, 2, 64, 64, BF16, seed=9)
    check(ts, S0, do, dS, scale=0.3)
    check(ts, S0, do, dS, states=False)
    a = gated_delta_rule(*ts)
    b = gated_delta_rule(*ts, scale=64**-0.5, return_state=True)[0]
    assert rel(a, b) <= 3 * STEP


@pytest.mark.parametrize("which", ["o", "state"])
def test_one_of_the_gradients(which):
    ts, S0, do, dS = inputs(2, 80, 2, 64, 64, F32, seed=10)
    own, ref = ([t.detach().to(d).requires_grad_() for t in (*ts, S0)] for d in (F32, torch.float64))
    o, S = gated_delta_rule(*own[:5], initial_state=own[5], return_state=True)
    ro, rS = recurrence(*ref, 64**-0.5)
    up = do if which == "o" else dS
    (o if which == "o" else S).backward(up)
    (ro if which == "o" else rS).backward(up.double())
    for a, b in zip(own, ref):
        g = torch.zeros_like(a) if a.grad is None else a.grad
        assert rel(g, torch.zeros_like(b) if b.grad is None else b.grad) <= F32_TOL


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_layouts(dtype):
    """Views of one projection, heads before tokens, rows off 16 bytes, shared heads (stride zero)."""
    ts, S0, do, dS = inputs(2, 100, 4, 64, 64, dtype, seed=11)
    want = gated_delta_rule(*ts, initial_state=S0)
    fused = torch.cat([t.flatten(2) for t in ts], -1)
    q, k, v, g, b = fused.split([256, 256, 256, 4, 4], -1)
    q, k, v = (t.unflatten(-1, (4, 64)) for t in (q, k, v))
    assert torch.equal(gated_delta_rule(q, k, v, g, b, initial_state=S0), want)
    heads_first = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in ts]
    assert torch.equal(gated_delta_rule(*heads_first, initial_state=S0), want)
    odd = [torch.cat([t.flatten()[:1], t.flatten()])[1:].view(t.shape) for t in ts]
    assert odd[0].data_ptr() % 16
    assert torch.equal(gated_delta_rule(*odd, initial_state=S0), want)
    strided = [torch.stack([t, t], -1)[..., 0] for t in ts]
    assert torch.equal(gated_delta_rule(*strided, initial_state=S0), want)
    one = ts[1][:, :, :1].detach().requires_grad_()
    o = gated_delta_rule(ts[0], one.expand(-1, -1, 4, -1), *ts[2:])
    o.backward(do)
    ref = ts[1][:, :, :1].double().requires_grad_()
    ro, _ = recurrence(ts[0].double(), ref.expand(-1, -1, 4, -1), *(t.double() for t in ts[2:]), torch.zeros_like(S0).double(), 1 / 8)
    ro.backward(do.double())
    assert rel(o, ro) <= tol("o", dtype) and rel(one.grad, ref.grad) <= 2 * tol("dk", dtype)


@pytest.mark.parametrize("which", range(5))
def test_gradient_against_differences(which):
    ts, S0, do, _ = inputs(1, 50, 1, 32, 32, F32, seed=12)
    own = [t.detach().requires_grad_() for t in ts]
    f = lambda x: (gated_delta_rule(*x, initial_state=S0).double() * do.double()).sum().item()  # noqa: E731
    gated_delta_rule(*own, initial_state=S0).backward(do)
    step = torch.randn_like(ts[which]) * (0.2 if which < 3 else 0.02)
    with torch.no_grad():
        moved = [[t + s * step if i == which else t for i, t in enumerate(ts)] for s in (0.05, -0.05)]
        slope = (f(moved[0]) - f(moved[1])) / 0.1
    want = (own[which].grad.double() * step.double()).sum().item()
    # central differences: the third derivative's share of a step of 0.05 is under a hundredth of the scale
    scale = (own[which].grad.double().norm() * step.double().norm()).item()
    assert abs(slope - want) <= 1e-2 * scale


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_empty(dtype):
    for B, T in ((0, 5), (2, 0)):
        ts, S0, _, _ = inputs(B, T, 2, 16, 16, dtype)
        own = [t.requires_grad_() for t in (*ts, S0)]
        o, S = gated_delta_rule(*own[:5], initial_state=own[5], return_state=True)
        assert o.shape == (B, T, 2, 16) and torch.equal(S, S0)
        (o.sum() + 2 * S.sum()).backward()
        assert torch.equal(own[5].grad, torch.full_like(S0, 2.0))
        assert all(t.grad.shape == t.shape for t in ts)
    assert not gated_delta_rule(*(inputs(2, 0, 2, 16, 16, dtype)[0]), return_state=True)[1].any()


def test_same_bits_again():
    ts, S0, do, dS = inputs(2, 300, 8, 128, 128, BF16, seed=13)
    runs = []
    for _ in range(2):
        own = [t.detach().requires_grad_() for t in ts]
        o, S = gated_delta_rule(*own, initial_state=S0, return_state=True)
        torch.autograd.backward([o, S], [do, dS])
        runs.append([o, S, *(t.grad for t in own)])
    assert all(torch.equal(a, b) for a, b in zip(*runs))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("t,which", [(0, 1), (70, 1), (70, 2), (95, 0), (63, 3), (77, 4), (64, 2)])
def test_what_is_not_finite_reaches_no_earlier_token(dtype, bad, t, which):
    if which == 3 and bad == -float("inf"):
        pytest.skip("a log decay of minus infinity is a number like others")
    ts, S0, _, _ = inputs(2, 150, 3, 64, 64, dtype, seed=14)
    want = gated_delta_rule(*ts, initial_state=S0)
    with torch.no_grad():
        ts[which][1, t, 2, ...] = bad
        o, S = gated_delta_rule(*ts, initial_state=S0, return_state=True)
    here = torch.ones(2, 150, 3, dtype=torch.bool, device="cuda")
    here[1, t:, 2] = False
    assert rel(o[here], want[here]) <= 3 * STEP
    if which == 0:  # a query is its own token's alone
        here[1, t + 1:, 2] = True
        assert rel(o[here], want[here]) <= 3 * STEP and o[1, t, 2].isnan().all() and S.isfinite().all()
    else:
        assert o[1, t:, 2].isnan().any(-1).all()
        clean = torch.ones(2, 3, dtype=torch.bool, device="cuda")
        clean[1, 2] = False
        assert S[clean].isfinite().all() and S[1, 2].isnan().any()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("t", [0, 63, 64, 90])
def test_gradients_that_are_not_finite_reach_no_later_token(dtype, t):
    ts, S0, do, _ = inputs(2, 150, 3, 64, 64, dtype, seed=15)
    grads = []
    for bad in (False, True):
        own = [x.detach().requires_grad_() for x in ts]
        up = do.clone()
        if bad:
            up[1, t, 2, 5] = float("nan")
        gated_delta_rule(*own, initial_state=S0).backward(up)
        grads.append([x.grad for x in own])
    here = torch.ones(2, 150, 3, dtype=torch.bool, device="cuda")
    here[1, :t + 1, 2] = False
    for n, a, b in zip(NAMES, *grads):
        assert rel(b[here], a[here]) <= tol("d" + n, dtype), n
        assert b[1, t, 2].isnan().any() or n == "beta", n


# --------------------------------------------------------------------------------- steps


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("B,H,dk,dv", [(1, 1, 1, 1), (1, 16, 128, 128), (5, 3, 64, 96), (2, 2, 37, 51), (70, 4, 128, 256), (3, 2, 100, 30)])
def test_step(dtype, B, H, dk, dv):
    ts, S0, _, _ = inputs(B, 3, H, dk, dv, dtype, seed=dk)
    S = S0.clone()
    got = torch.stack([gated_delta_rule_step(*(x[:, t] for x in ts[:3]), S, *(x[:, t] for x in ts[3:])) for t in range(3)], 1)
    ro, rS = recurrence(*(t.double() for t in ts), S0.double(), dk**-0.5)
    # (one rounding: 2^-8 of a value at most, whose root mean square says little of three values)
    assert rel(got, ro) <= (2 * STEP if dtype == BF16 else F32_TOL) and rel(S, rS) <= F32_TOL


@pytest.mark.parametrize("index", [torch.int32, torch.int64])
def test_step_slots(index):
    B, n = 6, 9
    ts, _, _, _ = inputs(B, 1, 2, 64, 64, BF16, seed=16)
    ts = [t[:, 0] for t in ts]
    pool = torch.randn(n, 2, 64, 64, device="cuda")
    slots = torch.tensor([7, -1, 0, 9, 3, 1 << 20], device="cuda", dtype=index)
    with torch.no_grad():
        ts[2][1] = float("nan")  # a padding row may hold anything
    before, live = pool.clone(), [0, 2, 4]
    o = gated_delta_rule_step(*ts[:3], pool, *ts[3:], slots=slots)
    rows = slots[live].long()
    own = before[rows].contiguous()
    want = gated_delta_rule_step(*(t[live] for t in ts[:3]), own, *(t[live] for t in ts[3:]))
    assert torch.equal(o[live], want) and torch.equal(pool[rows], own)
    assert not o[[1, 3, 5]].any()
    rest = torch.ones(n, dtype=torch.bool, device="cuda")
    rest[rows] = False
    assert torch.equal(pool[rest], before[rest])


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("T", [1, 64, 100])
def test_prompt_then_steps(dtype, T):
    ts, S0, _, _ = inputs(2, T + 5, 3, 64, 64, dtype, seed=17)
    whole, S_whole = gated_delta_rule(*ts, initial_state=S0, return_state=True)
    _, S = gated_delta_rule(*(t[:, :T] for t in ts), initial_state=S0, return_state=True)
    o = torch.stack([gated_delta_rule_step(*(x[:, t] for x in ts[:3]), S, *(x[:, t] for x in ts[3:])) for t in range(T, T + 5)], 1)
    assert rel(o, whole[:, T:]) <= (4 * STEP if dtype == BF16 else F32_TOL) and rel(S, S_whole) <= F32_TOL


def test_other_stream_and_graph():
    """A training step and a token's step captured on a stream of their own, and replayed on new inputs."""
    ts, S0, do, _ = inputs(2, 130, 4, 64, 64, BF16, seed=18)
    new, _, new_do, _ = inputs(2, 130, 4, 64, 64, BF16, seed=19)

    def train(x, up):
        own = [t.detach().requires_grad_() for t in x]
        o = gated_delta_rule(*own)
        return [o.detach(), *torch.autograd.grad(o, own, up)]

    want, want_step = train(new, new_do), S0.clone()
    step = lambda x, S: gated_delta_rule_step(*(t[:, 0] for t in x[:3]), S, *(t[:, 0] for t in x[3:]))  # noqa: E731
    want_o = step(new, want_step)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        train(ts, do)
        state = S0.clone()
        step(ts, state)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = train(ts, do)
        got_o = step(ts, state)
    for a, b in zip((*ts, do, state), (*new, new_do, S0)):
        a.copy_(b)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert torch.equal(got_o, want_o) and torch.equal(state, want_step)


def test_refusals():
    ts, S0, _, _ = inputs(2, 8, 2, 16, 16, BF16)
    q, k, v, g, b = ts
    for args in ((q.cpu(), k, v, g, b), (q, k[:, :4], v, g, b), (q, k.float(), v, g, b), (q, k, v, g[..., None], b),
                 (q, k, v, g.float(), b), (q, k, v, g, b[:, :4]), (q[0], k[0], v[0], g[0], b[0])):
        with pytest.raises(AssertionError):
            gated_delta_rule(*args)
    with pytest.raises(AssertionError):
        gated_delta_rule(*ts, initial_state=S0[:1])
    with pytest.raises(AssertionError):
        gated_delta_rule(*ts, initial_state=S0.bfloat16())
    with pytest.raises(TypeError):
        gated_delta_rule(*(t.half() for t in ts))
    big = inputs(1, 4, 1, 129, 16, BF16)[0]
    with pytest.raises(DynconvError):
        gated_delta_rule(*big)
    with pytest.raises(DynconvError):
        gated_delta_rule(*inputs(1, 4, 1, 16, 257, BF16)[0])
    one = [t[:, 0] for t in ts]
    with pytest.raises(AssertionError):
        gated_delta_rule_step(*one[:3], S0[:1], *one[3:])
    with pytest.raises(AssertionError):
        gated_delta_rule_step(*one[:3], S0, *one[3:], slots=torch.zeros(2, device="cuda"))
    with pytest.raises(RuntimeError):
        gated_delta_rule_step(one[0].clone().requires_grad_(), *one[1:3], S0, *one[3:])


def test_autograd_sees_updates_and_refuses_second_derivatives():
    ts, S0, _, _ = inputs(1, 6, 1, 16, 16, F32)
    S = S0.clone()
    w = torch.ones_like(S, requires_grad=True)
    y = (w * S).sum()
    gated_delta_rule_step(*(t[:, 0] for t in ts[:3]), S, *(t[:, 0] for t in ts[3:]))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    own = [t.requires_grad_() for t in ts]
    (dq,) = torch.autograd.grad(gated_delta_rule(*own).sum(), own[:1], create_graph=True)
    with pytest.raises(RuntimeError, match="cannot be differentiated again"):
        dq.sum().backward()
