"""GPU: linear attention with decay against the recurrence in 64 bits.

Tolerances are relative 2-norms, set from the roundings the operator makes:
  bf16: a rounding to eight bits is off by at most 2^-8 of a value and by less than 2^-9 of it
        in the root mean square; the result is rounded once, after products whose bf16
        operands (the scores and the state) were rounded once each: 3 * 2^-9;
  fp32: sums of up to 512 products, each addition at most 2^-24: 512 * 2^-24 = 3.1e-5 is the
        bound if all were to add up;
  states (always fp32, from bf16 or fp32 inputs): the same fp32 bound.
"""
from __future__ import annotations

import math

import pytest
import torch

from dynamic_conv1d_b200 import (
    check_device,
    decay_linear_attention,
    decay_linear_attention_fused,
    decay_linear_attention_step,
)

pytestmark = pytest.mark.gpu

BF16 = 3 * 2.0**-9
F32 = 512 * 2.0**-24
TOL = {torch.bfloat16: BF16, torch.float32: F32}


def rel(a, b):
    # what float32 cannot hold (a state decayed by exp(-300)) is zero in it
    a, b = a.detach().double(), b.detach().float().double()
    n = torch.linalg.vector_norm(b)
    d = torch.linalg.vector_norm(a - b)
    return (d / n if n > 0 else d).item()


def recurrence(q, k, v, log_decay, S, scale):
    """The definition, token by token, in the tensors' type (64 bits here)."""
    g = torch.exp(log_decay.double())[:, None, None]
    out = []
    for t in range(q.shape[1]):
        S = S * g + k[:, t, :, :, None] * v[:, t, :, None, :]
        out.append(scale * (q[:, t, :, None, :] @ S).squeeze(-2))
    return torch.stack(out, 1), S


def chunked(q, k, v, log_decay, S, scale, C=64):
    """The same sum, chunk by chunk (for long inputs): differentiable, in 64 bits."""
    lam = log_decay.double()[:, None, None]
    out = []
    for t0 in range(0, q.shape[1], C):
        qc, kc, vc = (x[:, t0:t0 + C].transpose(1, 2) for x in (q, k, v))
        L = qc.shape[2]
        i = torch.arange(L, device=q.device, dtype=torch.float64)
        m = torch.where(i[:, None] >= i, torch.exp(lam * (i[:, None] - i).clamp(min=0)), 0.0)
        o = ((qc @ kc.transpose(-1, -2)) * m) @ vc + torch.exp(lam * (i[:, None] + 1)) * (qc @ S)
        S = torch.exp(lam * L) * S + (kc * torch.exp(lam * (L - 1 - i[:, None]))).transpose(-1, -2) @ vc
        out.append(scale * o.transpose(1, 2))
    return torch.cat(out, 1), S


def inputs(B, T, H, dk, dv, dtype, seed=0, decay=None):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    q, k, v, do = (r(B, T, H, d).to(dtype) for d in (dk, dk, dv, dv))
    S0, dS = r(B, H, dk, dv), r(B, H, dk, dv)
    if decay is None:
        ld = torch.log1p(-torch.exp2(-torch.linspace(2, 9, H, device="cuda")))
    else:
        ld = torch.full((H,), decay, device="cuda")
    return q, k, v, do, S0, dS, ld.float()


def check(q, k, v, do, S0, dS, ld, scale=None, oracle=chunked):
    dtype = q.dtype
    sc = q.shape[-1] ** -0.5 if scale is None else scale
    own = [t.detach().requires_grad_() for t in (q, k, v, S0)]
    o, S = decay_linear_attention(own[0], own[1], own[2], ld, own[3], scale=scale, return_state=True)
    torch.autograd.backward([o, S], [do, dS])
    ref = [t.detach().double().requires_grad_() for t in (q, k, v, S0)]
    # the decay the kernels see is the float32 one
    ro, rS = oracle(ref[0], ref[1], ref[2], ld, ref[3], sc)
    torch.autograd.backward([ro, rS], [do.double(), dS.double()])
    check_device(o)
    err = {"o": (rel(o, ro), TOL[dtype]), "S": (rel(S, rS), F32)}
    for n, a, b in zip("qkv", own, ref):
        err["d" + n] = (rel(a.grad, b.grad), TOL[dtype])
    err["dS0"] = (rel(own[3].grad, ref[3].grad), F32)
    bad = {n: e for n, e in err.items() if not e[0] <= e[1]}
    assert not bad, bad
    return o, S


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T", [1, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 257, 500])
def test_lengths(dtype, T):
    check(*inputs(2, T, 3, 64, 64, dtype, seed=T), oracle=recurrence if T < 40 else chunked)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("dk,dv", [(128, 128), (64, 128), (128, 64), (32, 96), (96, 32), (80, 80), (40, 72), (8, 8), (16, 120),
                                   (13, 7), (1, 1), (130, 30), (256, 256), (64, 200)])
def test_widths(dtype, dk, dv):
    check(*inputs(2, 150, 2, dk, dv, dtype, seed=dk + dv))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("decay", [0.0, -1e-4, -0.1, -1.0, -20.0, -300.0, -math.inf])
def test_decays(dtype, decay):
    q, k, v, do, S0, dS, ld = inputs(1, 200, 2, 64, 64, dtype, decay=decay)
    check(q, k, v, do, S0, dS, ld.clamp(min=-1e3) if decay == -math.inf else ld)
    if decay == -math.inf:  # only the token itself is left, and no NaN
        o = decay_linear_attention(q, k, v, ld, S0)
        want = (q.double() * k.double()).sum(-1, keepdim=True) * v.double() * 64**-0.5
        assert rel(o, want) <= TOL[dtype]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T", [3000, 4099, 20000])
def test_long_few_heads(dtype, T):
    """Few heads and a long time axis: the chains are cut into segments."""
    check(*inputs(1, T, 1, 64, 64, dtype, seed=3))


@pytest.mark.parametrize("T", [1000, 2500])
def test_wide_segments(T):
    check(*inputs(1, T, 2, 128, 96, torch.bfloat16, seed=4))


def test_many_chains():
    check(*inputs(5, 70, 40, 64, 64, torch.bfloat16, seed=5))


def test_scale_and_defaults():
    q, k, v, do, S0, dS, ld = inputs(2, 100, 2, 64, 64, torch.bfloat16)
    check(q, k, v, do, S0, dS, ld, scale=0.3)
    check(q, k, v, do, S0, dS, ld, scale=0.0)
    o = decay_linear_attention(q, k, v, ld)
    ro, _ = chunked(q.double(), k.double(), v.double(), ld, torch.zeros_like(S0).double(), 64**-0.5)
    assert rel(o, ro) <= BF16


def test_gradient_of_the_output_alone():
    """No state in or out: the unused state's gradient is absent, not zero-filled by the caller."""
    q, k, v, do, S0, _, ld = inputs(2, 130, 2, 64, 64, torch.bfloat16)
    own = [t.requires_grad_() for t in (q, k, v)]
    torch.autograd.backward(decay_linear_attention(*own, ld), do)
    ref = [t.detach().double().requires_grad_() for t in own]
    o, _ = chunked(*ref, ld, torch.zeros_like(S0).double(), 64**-0.5)
    o.backward(do.double())
    for a, b in zip(own, ref):
        assert rel(a.grad, b.grad) <= BF16


def test_gradient_of_the_state_alone():
    q, k, v, _, S0, dS, ld = inputs(1, 130, 2, 64, 64, torch.bfloat16)
    own = [t.requires_grad_() for t in (q, k, v, S0)]
    _, S = decay_linear_attention(*own[:3], ld, own[3], return_state=True)
    S.backward(dS)
    ref = [t.detach().double().requires_grad_() for t in own]
    _, rS = chunked(*ref[:3], ld, ref[3], 1.0)
    rS.backward(dS.double())
    assert own[0].grad.count_nonzero() == 0
    for a, b, tol in zip(own[1:], ref[1:], (BF16, BF16, F32)):
        assert rel(a.grad, b.grad) <= tol


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T", [5, 300])
def test_layouts(dtype, T):
    """Heads before time, thirds of a fused projection, an offset view, a broadcast batch."""
    B, H, d = 3, 2, 64
    q, k, v, do, S0, dS, ld = inputs(B, T, H, d, d, dtype)
    want = decay_linear_attention(q, k, v, ld)
    head_first = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v)]
    assert torch.equal(decay_linear_attention(*head_first, ld), want)
    fused = torch.stack([q, k, v], 2).reshape(B, T, 3 * H * d)
    assert torch.equal(decay_linear_attention(*fused.view(B, T, 3, H, d).unbind(2), ld), want)
    assert torch.equal(decay_linear_attention_fused(fused, ld).view_as(want), want)
    odd = [torch.empty(B, T, H, d + 3, device="cuda", dtype=dtype) for _ in range(3)]
    for o_, t in zip(odd, (q, k, v)):
        o_[..., 1:d + 1] = t
    got = decay_linear_attention(*(o_[..., 1:d + 1] for o_ in odd), ld)
    assert rel(got, want) <= TOL[dtype]
    strided = torch.randn(B, T, H, 2 * d, device="cuda").to(dtype)[..., ::2]
    got = decay_linear_attention(strided, k, v, ld)
    assert torch.equal(got, decay_linear_attention(strided.contiguous(), k, v, ld))
    one = [t[:1].detach().requires_grad_() for t in (q, k, v)]
    wide = [t.expand(B, T, H, d) for t in one]
    torch.autograd.backward(decay_linear_attention(*wide, ld), do)
    ref = [t.detach().double().requires_grad_() for t in one]
    o, _ = chunked(*(t.expand(B, T, H, d) for t in ref), ld, torch.zeros_like(S0).double(), d**-0.5)
    o.backward(do.double())
    for a, b in zip(one, ref):
        assert rel(a.grad, b.grad) <= TOL[dtype]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_fused_gradient_is_one_buffer(dtype):
    B, T, H, d = 2, 200, 3, 64
    q, k, v, do, S0, dS, ld = inputs(B, T, H, d, d, dtype)
    x = torch.stack([q, k, v], 2).reshape(B, T, 3 * H * d).requires_grad_()
    s = S0.clone().requires_grad_()
    o, S = decay_linear_attention_fused(x, ld, initial_state=s, return_state=True)
    torch.autograd.backward([o, S], [do.reshape(B, T, H * d), dS])
    own = [t.requires_grad_() for t in (q, k, v, S0)]
    o2, S2 = decay_linear_attention(*own[:3], ld, own[3], return_state=True)
    torch.autograd.backward([o2, S2], [do, dS])
    assert torch.equal(o.view_as(o2), o2) and torch.equal(S, S2) and torch.equal(s.grad, S0.grad)
    assert torch.equal(x.grad.view(B, T, 3, H, d), torch.stack([t.grad for t in own[:3]], 2))


@pytest.mark.parametrize("which", [0, 1, 2, 3])
def test_gradient_against_differences(which):
    """The output is linear in each argument, so a central difference along any direction is
    the derivative itself, up to the fp32 rounding of the two outputs (2^-24 of sums of
    products of up to 512 terms, divided by the step of 1)."""
    q, k, v, do, S0, _, ld = inputs(1, 90, 2, 32, 48, torch.float32, seed=9)
    args = [q, k, v, S0]
    x = args[which].detach().requires_grad_()
    run = lambda a: decay_linear_attention(a[0], a[1], a[2], ld, a[3])  # noqa: E731
    run([x if i == which else t for i, t in enumerate(args)]).backward(do)
    e = torch.randn(x.shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    with torch.no_grad():
        hi = run([x + e if i == which else t for i, t in enumerate(args)]).double()
        lo = run([x - e if i == which else t for i, t in enumerate(args)]).double()
    dif = ((hi - lo) / 2 * do.double()).sum()
    ana = (x.grad.double() * e.double()).sum()
    size = ((hi - lo) / 2 * do.double()).abs().sum()
    assert (dif - ana).abs() <= F32 * size


def test_empty():
    q, k, v, do, S0, dS, ld = inputs(2, 4, 2, 64, 64, torch.bfloat16)
    e = [t[:, :0] for t in (q, k, v)]
    o, S = decay_linear_attention(*e, ld, S0, return_state=True)
    assert o.shape == (2, 0, 2, 64) and torch.equal(S, S0)
    _, S = decay_linear_attention(*e, ld, return_state=True)
    assert S.count_nonzero() == 0
    s = S0.clone().requires_grad_()
    decay_linear_attention(*e, ld, s, return_state=True)[1].backward(dS)
    assert torch.equal(s.grad, dS)
    assert decay_linear_attention(q[:0], k[:0], v[:0], ld).shape == (0, 4, 2, 64)


def test_same_bits_again():
    a = inputs(1, 3000, 2, 128, 128, torch.bfloat16)
    one, two = check(*a), check(*a)
    assert torch.equal(one[0], two[0]) and torch.equal(one[1], two[1])


def test_nan_stays_in_its_row_and_head():
    q, k, v, _, S0, _, ld = inputs(2, 300, 2, 64, 64, torch.bfloat16)
    want = decay_linear_attention(q, k, v, ld, S0)
    k = k.clone()
    k[1, 200, 1, 5] = float("nan")
    v = v.clone()
    v[0, 290, 0] = float("inf")
    got = decay_linear_attention(q, k, v, ld, S0)
    assert torch.equal(got[0, :, 1], want[0, :, 1]) and torch.equal(got[1, :, 0], want[1, :, 0])
    assert got[1, 200:, 1].isnan().all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("t", [0, 1, 130, 255, 299])
def test_later_tokens_stay_masked(dtype, bad, t):
    """What is not finite in one token's q, k or v reaches no earlier token (a prompt's padding may
    hold anything), and the gradients of a padded batch's own tokens stay finite."""
    q, k, v, do, S0, _, ld = inputs(1, 300, 2, 64, 64, dtype)
    want = decay_linear_attention(q, k, v, ld, S0)
    for x in (q, k, v):
        keep = x[0, t:, 1].clone()
        x[0, t:, 1] = bad
        got = decay_linear_attention(q, k, v, ld, S0)
        assert torch.equal(got[0, :t, 1], want[0, :t, 1]) and torch.equal(got[0, :, 0], want[0, :, 0])
        assert not got[0, t:, 1].isfinite().any()
        x[0, t:, 1] = keep
    # backwards in time: an upstream gradient that is not finite reaches no later token's dk, dv
    own = [x.detach().requires_grad_() for x in (q, k, v)]
    ref = torch.autograd.grad(decay_linear_attention(*own, ld, S0), own, do)
    do = do.clone()
    do[0, t, 0, 3] = bad
    got = torch.autograd.grad(decay_linear_attention(*own, ld, S0), own, do)
    for i, (g, r) in enumerate(zip(got, ref)):
        assert torch.equal(g[0, t + 1:, 0], r[0, t + 1:, 0]) and torch.equal(g[0, :, 1], r[0, :, 1])
        if i == 0:
            assert torch.equal(g[0, :t, 0], r[0, :t, 0])


# ------------------------------------------------------------------------------ steps


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B,H,dk,dv", [(1, 1, 1, 1), (1, 16, 128, 128), (3, 5, 64, 96), (2, 3, 13, 7), (4, 2, 256, 256),
                                       (70, 4, 128, 128), (2, 2, 200, 36), (300, 2, 32, 32)])
def test_step(dtype, B, H, dk, dv):
    q, k, v, _, S0, _, ld = inputs(B, 1, H, dk, dv, dtype, seed=B)
    S = S0.clone()
    o = decay_linear_attention_step(q[:, 0], k[:, 0], v[:, 0], S, ld)
    ro, rS = recurrence(q.double(), k.double(), v.double(), ld, S0.double(), dk**-0.5)
    check_device(o)
    assert rel(o, ro[:, 0]) <= TOL[dtype] and rel(S, rS) <= F32


@pytest.mark.parametrize("index", [torch.int32, torch.int64])
def test_step_slots(index):
    B, H, d, n = 6, 3, 64, 11
    q, k, v, _, _, _, ld = inputs(B, 1, H, d, d, torch.bfloat16)
    pool = torch.randn(n, H, d, d, device="cuda")
    slots = torch.tensor([7, -1, 0, 10, 11, 3], device="cuda", dtype=index)
    S = pool.clone()
    o = decay_linear_attention_step(q[:, 0], k[:, 0], v[:, 0], S, ld, slots=slots)
    live = [0, 2, 3, 5]
    rows = slots[live].long()
    ro, rS = recurrence(q[live].double(), k[live].double(), v[live].double(), ld, pool[rows].double(), d**-0.5)
    assert rel(o[live], ro[:, 0]) <= BF16 and rel(S[rows], rS) <= F32
    assert o[[1, 4]].count_nonzero() == 0
    rest = [i for i in range(n) if i not in rows.tolist()]
    assert torch.equal(S[rest], pool[rest])


def test_step_reads_views():
    B, H, d = 5, 2, 64
    row = torch.randn(B, 3, H, d, device="cuda").bfloat16()
    _, _, _, _, S0, _, ld = inputs(B, 1, H, d, d, torch.bfloat16)
    q, k, v = row.unbind(1)
    A, Bs = S0.clone(), S0.clone()
    assert torch.equal(decay_linear_attention_step(q, k, v, A, ld),
                       decay_linear_attention_step(q.contiguous(), k.contiguous(), v.contiguous(), Bs, ld))
    assert torch.equal(A, Bs)


def test_prompt_then_steps():
    """A prompt's state, continued token by token, gives what the whole sequence gives."""
    q, k, v, _, _, _, ld = inputs(2, 140, 3, 64, 64, torch.bfloat16)
    whole = decay_linear_attention(q, k, v, ld)
    o, S = decay_linear_attention(q[:, :133], k[:, :133], v[:, :133], ld, return_state=True)
    rest = [decay_linear_attention_step(q[:, t], k[:, t], v[:, t], S, ld) for t in range(133, 140)]
    assert rel(torch.cat([o, torch.stack(rest, 1)], 1), whole) <= 2 * BF16


def test_other_stream_and_graph():
    q, k, v, _, S0, _, ld = inputs(2, 300, 2, 64, 64, torch.bfloat16)
    want = decay_linear_attention(q, k, v, ld, S0)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        got = decay_linear_attention(q, k, v, ld, S0)
    torch.cuda.current_stream().wait_stream(st)
    assert torch.equal(got, want)
    S = S0.clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        o = decay_linear_attention(q, k, v, ld, S0)
        one = decay_linear_attention_step(q[:, 0], k[:, 0], v[:, 0], S, ld)
    q.copy_(torch.randn_like(q))
    S.copy_(S0)
    g.replay()
    assert torch.equal(o, decay_linear_attention(q, k, v, ld, S0))
    fresh = S0.clone()
    assert torch.equal(one, decay_linear_attention_step(q[:, 0], k[:, 0], v[:, 0], fresh, ld)) and torch.equal(S, fresh)


# --------------------------------------------------------------------------- refusals


def test_refusals():
    q, k, v, _, S0, _, ld = inputs(2, 8, 2, 64, 64, torch.bfloat16)
    for bad in (
        dict(q=q.half(), k=k.half(), v=v.half()),
        dict(k=k.float()),
        dict(k=k[:, :7]),
        dict(q=q.cpu()),
        dict(log_decay=ld.double()),
        dict(log_decay=ld[:1]),
        dict(log_decay=ld.clone().requires_grad_()),
        dict(initial_state=S0[:1]),
        dict(initial_state=S0.bfloat16()),
        dict(initial_state=S0.transpose(2, 3)),
        dict(q=torch.zeros(2, 8, 2, 257, device="cuda"), k=torch.zeros(2, 8, 2, 257, device="cuda"), v=v.float()),
    ):
        a = dict(q=q, k=k, v=v, log_decay=ld) | bad
        with pytest.raises((AssertionError, TypeError, RuntimeError)):
            decay_linear_attention(**a)
    with pytest.raises(AssertionError):
        decay_linear_attention_fused(torch.zeros(1, 2, 100, device="cuda"), ld)
    step = dict(q=q[:, 0], k=k[:, 0], v=v[:, 0], state=S0.clone(), log_decay=ld)
    for bad in (dict(state=S0[:1]), dict(state=S0.half()), dict(slots=torch.zeros(2, device="cuda")),
                dict(slots=torch.zeros(3, device="cuda", dtype=torch.int32)), dict(q=q[:, 0].clone().requires_grad_())):
        with pytest.raises((AssertionError, RuntimeError)):
            decay_linear_attention_step(**(step | bad))


# ------------------------------------------------------------------------------ autograd


def test_updates_in_place_are_seen_by_autograd():
    """A step on a state that a prompt's backward still needs is an error, not another gradient."""
    q, k, v, do, S0, _, ld = inputs(2, 20, 2, 64, 64, torch.bfloat16)
    S = S0.clone()
    o = decay_linear_attention(q.requires_grad_(), k, v, ld, S)
    with torch.no_grad():
        decay_linear_attention_step(q[:, 0], k[:, 0], v[:, 0], S, ld)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        o.backward(do)
    with torch.inference_mode():
        inside = S0.clone()
        decay_linear_attention_step(q[:, 0], k[:, 0], v[:, 0], inside, ld)
    assert torch.equal(inside, S)


def test_no_second_derivative():
    """The gradients are no functions of the inputs to autograd: differentiating them is an error, not a
    constant."""
    q, k, v, do, S0, _, ld = inputs(1, 40, 2, 64, 64, torch.float32)
    x = torch.stack([q, k, v], 2).reshape(1, 40, 3 * 2 * 64).requires_grad_()
    q.requires_grad_()
    for leaf, run in ((q, lambda: decay_linear_attention(q, k, v, ld, S0)), (x, lambda: decay_linear_attention_fused(x, ld))):
        o = run()
        (g,) = torch.autograd.grad(o, leaf, do.view_as(o), create_graph=True)
        with pytest.raises(RuntimeError, match="differentiated again"):
            (leaf.sum() + g.square().sum()).backward()
        (g1,) = torch.autograd.grad(run(), leaf, do.view_as(o))
        assert torch.equal(g, g1)
