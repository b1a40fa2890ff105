"""GPU: the gated norm and the residual norm against their definitions in 64 bits.

Tolerances are relative 2-norms: bf16 results are rounded once, by less than 2^-9 of a value in the root mean square
(bound: twice that, and three times where a gradient's sum holds the rounded residual stream); fp32 results come
from sums of up to 16384 numbers held by up to 1024 threads, 16 of each one after another, then in a tree or a
list of 32: under 64 additions of at most 2^-24, twice: 128 * 2^-24."""
from __future__ import annotations

import pytest
import torch

from dynamic_conv1d_b200 import DynconvError, gated_rms_norm, residual_rms_norm

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
TOL = {BF16: 2 * 2.0**-9, F32: 128 * 2.0**-24}
SUM_TOL = {BF16: 3 * 2.0**-9, F32: 128 * 2.0**-24}


def rel(a, b):
    a, b = a.detach().double(), b.detach().double()
    n, d = torch.linalg.vector_norm(b), torch.linalg.vector_norm(a - b)
    return (d / n if n > 0 else d).item()


def rnd(*shape, dtype=F32, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, device="cuda", generator=g).to(dtype)


def gated(x, w, z, eps, scale):
    y = scale * x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps)
    y = y if w is None else y * w
    return y if z is None else y * z * torch.sigmoid(z)


def residual(x, r, w, s, eps):
    h = r + s * x
    return h * torch.rsqrt(h.square().mean(-1, keepdim=True) + eps) * w, h


WIDTHS = [1, 2, 7, 8, 31, 32, 64, 99, 128, 256, 257, 511, 512, 513, 1000, 2048, 2050, 4096, 4097, 8192, 16384]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("D", WIDTHS)
def test_gated(dtype, D):
    N = 70 if D < 3000 else 5
    x, w, z, dy = rnd(N, 3, D, dtype=dtype, seed=1), 1 + rnd(D, dtype=dtype, seed=2) / 4, rnd(N, 3, D, dtype=dtype, seed=3), rnd(N, 3, D, dtype=dtype, seed=4)
    own, ref = [t.detach().requires_grad_() for t in (x, w, z)], [t.detach().double().requires_grad_() for t in (x, w, z)]
    y, ry = gated_rms_norm(*own, eps=1e-5, scale=0.7), gated(*ref, 1e-5, 0.7)
    y.backward(dy)
    ry.backward(dy.double())
    assert rel(y, ry) <= TOL[dtype]
    for n, a, b in zip("xwz", own, ref):
        # (one channel: dx is a difference of equal terms, zero but for eps)
        bound = 1.0 if n == "x" and D == 1 else TOL[dtype]
        assert rel(a.grad, b.grad) <= bound, n


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("D", WIDTHS)
@pytest.mark.parametrize("scale", ["channels", 0.5])
def test_residual(dtype, D, scale):
    N = 210 if D < 3000 else 7
    x, r, dy, dh = (rnd(N, D, dtype=dtype, seed=i) for i in range(4))
    w, s = 1 + rnd(D, dtype=dtype, seed=5) / 4, 0.5 + rnd(D, dtype=dtype, seed=6) / 8
    leaves = (x, r, w, s) if scale == "channels" else (x, r, w)
    own, ref = [t.detach().requires_grad_() for t in leaves], [t.detach().double().requires_grad_() for t in leaves]
    at = lambda t: t[3] if scale == "channels" else scale  # noqa: E731
    y, h = residual_rms_norm(*own[:3], at(own), eps=1e-6)
    ry, rh = residual(*ref[:3], at(ref), 1e-6)
    torch.autograd.backward([y, h], [dy, dh])
    torch.autograd.backward([ry, rh], [dy.double(), dh.double()])
    assert rel(y, ry) <= TOL[dtype] and rel(h, rh) <= TOL[dtype]
    for n, a, b in zip("xrws", own, ref):
        assert rel(a.grad, b.grad) <= SUM_TOL[dtype], n


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_many_rows(dtype):
    """More rows than threads of the card, a number that is no multiple of anything."""
    x, w, z, dy = rnd(40001, 2, 64, dtype=dtype), 1 + rnd(64, dtype=dtype, seed=1) / 4, rnd(40001, 2, 64, dtype=dtype, seed=2), rnd(40001, 2, 64, dtype=dtype, seed=3)
    own, ref = [t.detach().requires_grad_() for t in (x, w, z)], [t.detach().double().requires_grad_() for t in (x, w, z)]
    gated_rms_norm(*own).backward(dy)
    gated(*ref, 1e-6, 1.0).backward(dy.double())
    for a, b in zip(own, ref):
        # sums of 80002 products over at most 68 rows a thread, 32 threads and 600 CTAs: still under 128 additions in a row
        assert rel(a.grad, b.grad) <= (TOL[dtype] if dtype == BF16 else 256 * 2.0**-24)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("with_w,with_z", [(False, False), (True, False), (False, True)])
def test_optional_parts(dtype, with_w, with_z):
    x, dy = rnd(9, 5, 96, dtype=dtype), rnd(9, 5, 96, dtype=dtype, seed=1)
    w, z = (rnd(96, dtype=dtype, seed=2) if with_w else None), (rnd(9, 5, 96, dtype=dtype, seed=3) if with_z else None)
    own = [None if t is None else t.detach().requires_grad_() for t in (x, w, z)]
    ref = [None if t is None else t.detach().double().requires_grad_() for t in (x, w, z)]
    y, ry = gated_rms_norm(*own, scale=96**-0.5), gated(*ref, 1e-6, 96**-0.5)
    y.backward(dy)
    ry.backward(dy.double())
    assert rel(y, ry) <= TOL[dtype]
    for a, b in zip(own, ref):
        assert a is None or rel(a.grad, b.grad) <= TOL[dtype]
    if not with_w and not with_z:
        assert (y.double().square().sum(-1) - 1).abs().max() <= 2.0**-7


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_layouts(dtype):
    """Heads of a fused projection in place; a gate laid out otherwise; rows off 16 bytes; four dimensions."""
    big, z = rnd(3, 20, 6 * 64, dtype=dtype), rnd(3, 20, 2, 64, dtype=dtype, seed=1)
    x = big[..., 128:256].unflatten(-1, (2, 64))
    want = gated_rms_norm(x.contiguous(), gate=z)
    assert torch.equal(gated_rms_norm(x, gate=z), want)
    assert torch.equal(gated_rms_norm(x.contiguous(), gate=torch.cat([z, z], -1)[..., :64]), want)
    assert torch.equal(gated_rms_norm(x, gate=z.transpose(0, 1).contiguous().transpose(0, 1)), want)
    # rows off 16 bytes are read number by number, and their squares add up in another order
    odd = torch.cat([z.flatten()[:1], z.flatten()])[1:].view(z.shape)
    assert rel(gated_rms_norm(x, gate=odd), want) <= TOL[dtype]
    assert torch.equal(gated_rms_norm(x.transpose(1, 2), gate=z.transpose(1, 2)), want.transpose(1, 2))
    assert torch.equal(gated_rms_norm(x[0, 0, 0], gate=z[0, 0, 0]), want[0, 0, 0])
    one = rnd(64, dtype=dtype, seed=2).requires_grad_()
    gated_rms_norm(one.expand(10, 64)).sum().backward()
    ref = one.detach().double().requires_grad_()
    gated(ref.expand(10, 64), None, None, 1e-6, 1.0).sum().backward()
    assert rel(one.grad, ref.grad) <= 4 * TOL[dtype]


def test_missing_gradients_and_casts():
    x, r, w = rnd(6, 64, dtype=BF16), rnd(6, 64, dtype=BF16, seed=1), (1 + rnd(64, seed=2) / 4).requires_grad_()
    xg = x.clone().requires_grad_()
    y, h = residual_rms_norm(xg, r, w)
    y.sum().backward()  # h is not used
    assert w.grad.dtype == F32 and xg.grad.isfinite().all()
    xg.grad = None
    residual_rms_norm(xg, r, w)[1].sum().backward()  # y is not used
    assert torch.equal(xg.grad, torch.ones_like(x))
    g = gated_rms_norm(x, w.detach())
    assert g.dtype == BF16 and not g.requires_grad
    for t in (x, w):
        a = t.detach().clone().requires_grad_()
        args = (a, w.detach()) if t is x else (x, a)
        gated_rms_norm(*args).sum().backward()
        assert a.grad.shape == a.shape


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_empty_zero_and_not_finite_rows(dtype):
    w = torch.ones(32, device="cuda", dtype=dtype, requires_grad=True)
    s = torch.ones(32, device="cuda", dtype=dtype, requires_grad=True)
    y, h = residual_rms_norm(rnd(0, 32, dtype=dtype), rnd(0, 32, dtype=dtype), w, s)
    (y.sum() + h.sum() + gated_rms_norm(rnd(0, 4, 32, dtype=dtype), w).sum()).backward()
    assert y.shape == (0, 32) and not w.grad.any() and not s.grad.any()
    x = rnd(4, 32, dtype=dtype)
    x[1] = 0
    x[2, 3] = float("nan")
    x.requires_grad_()
    y = gated_rms_norm(x)
    y.sum().backward()
    for t in (y, x.grad):
        assert t[[0, 1, 3]].isfinite().all() and t[2].isnan().any()
    assert not y[1].any()


def test_same_bits_stream_and_graph():
    x, r, dy = (rnd(5000, 512, dtype=BF16, seed=i) for i in range(3))
    w, s = (torch.ones(512, device="cuda", dtype=BF16, requires_grad=True) for _ in range(2))

    def train():
        a, b = x.detach().requires_grad_(), r.detach().requires_grad_()
        y, h = residual_rms_norm(a, b, w, s)
        z = gated_rms_norm(y.view(5000, 8, 64), w[:64].contiguous(), h.view(5000, 8, 64))
        return [y.detach(), *torch.autograd.grad([z, h], [a, b, w, s], [dy.view(5000, 8, 64), dy])]

    want = train()
    assert all(torch.equal(a, b) for a, b in zip(train(), want))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        train()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = train()
    for t in got:
        t.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_refusals():
    x, w = rnd(4, 64), torch.ones(64, device="cuda")
    for bad in (lambda: gated_rms_norm(x.cpu()), lambda: gated_rms_norm(x, w[:32]), lambda: gated_rms_norm(x, gate=x.bfloat16()),
                lambda: gated_rms_norm(x, gate=x[:2]), lambda: residual_rms_norm(x, x[:2], w), lambda: residual_rms_norm(x[:, ::2], x[:, ::2], w[:32]),
                lambda: residual_rms_norm(x, x.bfloat16(), w), lambda: residual_rms_norm(x, x, w, w[:3])):
        with pytest.raises(AssertionError):
            bad()
    with pytest.raises(TypeError):
        gated_rms_norm(x.half())
    with pytest.raises(DynconvError):
        gated_rms_norm(rnd(2, 16385))
    a = x.clone().requires_grad_()
    (g,) = torch.autograd.grad(gated_rms_norm(a).sum(), a, create_graph=True)
    with pytest.raises(RuntimeError, match="cannot be differentiated again"):
        g.sum().backward()


@pytest.mark.parametrize("which", ["both", "y", "h"])
@pytest.mark.parametrize("N,D", [(48001, 64), (9001, 520), (5003, 1024), (2502, 2048), (1203, 4096), (907, 8192)])
def test_residual_rows_in_turn(N, D, which):
    """So many rows that a CTA's places in shared memory are used several times over, with one upstream gradient or both."""
    x, r, dy, dh = (rnd(N, D, dtype=BF16, seed=i) for i in range(4))
    w, s = 1 + rnd(D, dtype=BF16, seed=5) / 4, 0.5 + rnd(D, dtype=BF16, seed=6) / 8
    own, ref = [t.detach().requires_grad_() for t in (x, r, w, s)], [t.detach().double().requires_grad_() for t in (x, r, w, s)]
    y, h = residual_rms_norm(*own, eps=1e-6)
    ry, rh = residual(*ref, 1e-6)
    outs, ups = {"both": ([0, 1], (dy, dh)), "y": ([0], (dy,)), "h": ([1], (dh,))}[which]
    leaves = [i for i in range(4) if which != "h" or i != 2]  # (h does not depend on the weight)
    got = torch.autograd.grad([(y, h)[i] for i in outs], [own[i] for i in leaves], ups)
    want = torch.autograd.grad([(ry, rh)[i] for i in outs], [ref[i] for i in leaves], [u.double() for u in ups])
    for i, a, b in zip(leaves, got, want):
        # (a CTA adds 48001 / 9472 to 907 / 148 rows one after another, column sums of at most 592 follow: rounding to bf16 counts alone)
        assert rel(a, b) <= SUM_TOL[BF16], "xrws"[i]
