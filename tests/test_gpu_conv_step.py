"""GPU: the convolutions' single-token steps against their definition in 64 bits, and
against the whole-sequence operators.

Tolerances, value by value: a bf16 output is rounded once from its fp32 sum (half a unit in
the last of eight bits: 2^-8 of the value), an fp32 output likewise (2^-24); the sum has up
to W * (R + 1) = 512 products, each addition off by 2^-24 of the terms' absolute sum.
Where two bf16 results are compared, both roundings count.  The cache is moved, not
computed: equal bits."""
from __future__ import annotations

import pytest
import torch

from dynamic_conv1d_b200 import (
    check_device,
    convolution_cache,
    headwise_dynamic_convolution,
    headwise_dynamic_convolution_step,
    lowrank_dynamic_convolution,
    lowrank_dynamic_convolution_grouped_step,
    lowrank_dynamic_convolution_step,
)

pytestmark = pytest.mark.gpu

ROUND = {torch.bfloat16: 2.0**-8, torch.float32: 2.0**-24}
SUM = 512 * 2.0**-24
BOTH = [torch.bfloat16, torch.float32]


def rel(a, b):
    a, b = a.double(), b.double()
    n, d = torch.linalg.vector_norm(b), torch.linalg.vector_norm(a - b)
    return (d / n if n > 0 else d).item()


def near(y, want, terms):
    """y against its value in 64 bits, `terms` being the sum of the terms' absolute values."""
    return ((y.double() - want).abs() <= ROUND[y.dtype] * want.abs() + SUM * terms).all().item()


def lowrank_definition(x, z, U, cache, sw, residual):
    """[B, C], [B, G*R], [G, R, W*D], [B, W-1, C], [G, W, D] or None, all 64 bits."""
    B, C = x.shape
    G, R, WD = U.shape
    D = C // G
    W = WD // D
    w = torch.einsum("bgr,grn->bgn", z.view(B, G, R), U).view(B, G, W, D)
    if sw is not None:
        w = w + sw[None]
    w = w.transpose(1, 2).reshape(B, W, C)
    past = torch.cat([cache, x[:, None]], 1).flip(1)
    return (w * past).sum(1) + (x if residual else 0), torch.cat([cache, x[:, None]], 1)[:, 1:]


def make(B, G, D, R, W, dtype, n=None, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g).to(dtype)  # noqa: E731
    return r(B, G * D), r(B, G * R), r(G, R, W * D), r(n or B, W - 1, G * D), r(G, W, D)


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("static", [True, False])
@pytest.mark.parametrize("B,G,D,R,W", [(1, 1, 256, 15, 4), (1, 3, 2048, 15, 4), (2, 3, 100, 31, 3), (3, 1, 7, 1, 2), (4, 2, 33, 5, 8),
                                       (5, 1, 1, 3, 1), (8, 3, 512, 31, 4), (9, 1, 130, 64, 5), (257, 2, 64, 7, 6), (33, 16, 24, 64, 7)])
def test_lowrank(dtype, static, B, G, D, R, W):
    x, z, U, cache, sw = make(B, G, D, R, W, dtype, seed=B + W)
    sw = sw if static else None
    c = cache.clone()
    residual = bool(B % 2)
    y = lowrank_dynamic_convolution_grouped_step(x, z, U, c, sw, residual=residual)
    check_device(y)
    ref = [None if t is None else t.double() for t in (x, z, U, cache, sw)]
    ry, rc = lowrank_definition(*ref, residual)
    terms, _ = lowrank_definition(*(None if t is None else t.abs() for t in ref), residual)
    assert near(y, ry, terms)
    assert torch.equal(c.double(), rc)
    if G == 1:
        c = cache.clone()
        y1 = lowrank_dynamic_convolution_step(x, z, U[0], c, None if sw is None else sw[0], residual=residual)
        assert torch.equal(y1, y) and torch.equal(c.double(), rc)


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("static", [True, False])
@pytest.mark.parametrize("B,H,hs,W", [(1, 64, 32, 4), (1, 1, 1, 1), (2, 256, 1, 4), (3, 5, 7, 3), (64, 64, 32, 4), (2, 2, 128, 8), (700, 3, 2, 2),
                                      (2, 3, 5, 5), (2, 4, 6, 6), (2, 4, 2, 7)])
def test_headwise(dtype, static, B, H, hs, W):
    g = torch.Generator(device="cuda").manual_seed(B + H)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g).to(dtype)  # noqa: E731
    D = H * hs
    x, w, cache, sw = r(B, D), r(B, H, W), r(B, W - 1, D), r(W, D) if static else None
    c = cache.clone()
    y = headwise_dynamic_convolution_step(x, w, c, sw, residual=True)
    check_device(y)
    taps = w.double().transpose(1, 2).repeat_interleave(hs, 2)
    if static:
        taps = taps + sw.double()
    past = torch.cat([cache, x[:, None]], 1).double().flip(1)
    terms = ((w.double().abs().transpose(1, 2).repeat_interleave(hs, 2) + (sw.double().abs() if static else 0)) * past.abs()).sum(1)
    assert near(y, (taps * past).sum(1) + x.double(), terms + x.double().abs())
    assert torch.equal(c, torch.cat([cache, x[:, None]], 1)[:, 1:])


@pytest.mark.parametrize("W", [1, 2, 3, 4, 5, 6, 7, 8])
@pytest.mark.parametrize("R", [1, 15, 16, 31, 33, 47, 50, 64])
def test_lowrank_widths_and_ranks(W, R):
    """Every width with every number of 16-rank steps, whole octets of channels, rows beyond a block."""
    B, G, D = 70, 2, 40
    x, z, U, cache, sw = make(B, G, D, R, W, torch.bfloat16, seed=R + W)
    for s in (sw, None):
        c = cache.clone()
        y = lowrank_dynamic_convolution_grouped_step(x, z, U, c, s, residual=True)
        ref = [None if t is None else t.double() for t in (x, z, U, cache, s)]
        ry, rc = lowrank_definition(*ref, True)
        terms, _ = lowrank_definition(*(None if t is None else t.abs() for t in ref), True)
        assert near(y, ry, terms) and torch.equal(c.double(), rc)


@pytest.mark.parametrize("index", [torch.int32, torch.int64])
def test_slots(index):
    B, G, D, R, W, n = 6, 2, 64, 7, 4, 9
    x, z, U, pool, sw = make(B, G, D, R, W, torch.bfloat16, n=n)
    slots = torch.tensor([8, 3, -1, 0, 9, 5], device="cuda", dtype=index)
    c = pool.clone()
    y = lowrank_dynamic_convolution_grouped_step(x, z, U, c, sw, residual=True, slots=slots)
    live = [0, 1, 3, 5]
    rows = slots[live].long()
    ry, rc = lowrank_definition(x[live].double(), z[live].double(), U.double(), pool[rows].double(), sw.double(), True)
    terms, _ = lowrank_definition(*(t.double().abs() for t in (x[live], z[live], U, pool[rows], sw)), True)
    assert near(y[live], ry, terms) and torch.equal(c[rows].double(), rc)
    assert y[[2, 4]].count_nonzero() == 0
    rest = [i for i in range(n) if i not in rows.tolist()]
    assert torch.equal(c[rest], pool[rest])
    w = torch.randn(B, 4, W, device="cuda").bfloat16()
    c = pool.clone()
    y = headwise_dynamic_convolution_step(x, w, c, slots=slots)
    assert y[[2, 4]].count_nonzero() == 0 and y[live].count_nonzero() > 0 and torch.equal(c[rest], pool[rest])


@pytest.mark.parametrize("T", [1, 2, 3, 40])
def test_continues_a_prompt(T):
    """A prompt through the whole-sequence operators, then steps: what the longer sequence gives."""
    B, D, R, W, n = 2, 256, 15, 4, 6
    g = torch.Generator(device="cuda").manual_seed(T)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g).bfloat16()  # noqa: E731
    x, z, U, sw = r(B, T + n, D), r(B, T + n, R), r(R, W * D), r(W, D)
    w = r(B, T + n, 8, W)
    whole = lowrank_dynamic_convolution(x, z, U, sw, residual=True)
    whole_hw = headwise_dynamic_convolution(x, w, sw, residual=True)
    c = convolution_cache(x[:, :T], W)
    ch = convolution_cache(x[:, :T], W)
    assert c.shape == (B, W - 1, D)
    for t in range(T, T + n):
        xt = x[:, t].contiguous()
        y = lowrank_dynamic_convolution_step(xt, z[:, t].contiguous(), U, c, sw, residual=True)
        assert rel(y, whole[:, t]) <= 2.0**-7
        y = headwise_dynamic_convolution_step(xt, w[:, t], ch, sw, residual=True)
        assert rel(y, whole_hw[:, t]) <= 2.0**-7
    assert torch.equal(c, x[:, T + n - (W - 1):]) and torch.equal(ch, c)


def test_unaligned_and_empty():
    B, D, R, W = 3, 64, 7, 4
    x, z, U, cache, sw = make(B, 1, D, R, W, torch.bfloat16)
    shift = lambda t: torch.cat([t.new_zeros(1), t.flatten()])[1:].view(t.shape)  # noqa: E731
    c, cs = cache.clone(), shift(cache)
    y = lowrank_dynamic_convolution_step(x, z, U[0], c, sw[0])
    ys = lowrank_dynamic_convolution_step(shift(x), shift(z), shift(U[0]), cs, shift(sw[0]))
    assert rel(ys, y) <= 2.0**-7 and torch.equal(c, cs)
    assert lowrank_dynamic_convolution_step(x[:0], z[:0], U[0], c, sw[0]).shape == (0, D)


def test_graph():
    x, z, U, cache, sw = make(4, 3, 128, 15, 4, torch.bfloat16)
    c = cache.clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = lowrank_dynamic_convolution_grouped_step(x, z, U, c, sw, residual=True)
    c.copy_(cache)
    for _ in range(3):
        g.replay()
        cc = cache
        want = lowrank_dynamic_convolution_grouped_step(x, z, U, cc, sw, residual=True)
        assert torch.equal(y, want) and torch.equal(c, cc)


def test_refusals():
    x, z, U, cache, sw = make(2, 1, 64, 7, 4, torch.bfloat16)
    good = dict(x=x, z=z, U=U[0], cache=cache, static_w=sw[0])
    for bad in (dict(x=x.cpu()), dict(x=x.half()), dict(cache=cache.float()), dict(cache=cache[:, :2]), dict(cache=cache[:1]),
                dict(z=z[:1]), dict(U=U[0][:3]), dict(static_w=sw), dict(slots=torch.zeros(2, device="cuda")),
                dict(slots=torch.zeros(1, device="cuda", dtype=torch.int32)), dict(x=x.clone().requires_grad_())):
        with pytest.raises((AssertionError, TypeError, RuntimeError)):
            lowrank_dynamic_convolution_step(**(good | bad))
    with pytest.raises((AssertionError, RuntimeError)):  # nine taps
        x9, z9, U9, c9, s9 = make(1, 1, 8, 3, 9, torch.bfloat16)
        lowrank_dynamic_convolution_step(x9, z9, U9[0], c9, s9[0])
    with pytest.raises(AssertionError):
        headwise_dynamic_convolution_step(x, torch.zeros(2, 5, 4, device="cuda").bfloat16(), cache)


@pytest.mark.parametrize("dtype,B,D", [(torch.float32, 6, 64), (torch.float32, 70, 64), (torch.float32, 6, 33), (torch.bfloat16, 6, 33),
                                       (torch.bfloat16, 70, 33), (torch.bfloat16, 6, 64)])
def test_padding_rows_of_anything(dtype, B, D):
    """Rows whose slot lies outside the pool give zeros whatever their inputs hold, in every form of the
    step, and the other rows do not see them."""
    G, R, W, n = 2, 7, 4, 80
    x, z, U, pool, sw = make(B, G, D, R, W, dtype, n=n)
    slots = torch.arange(B, device="cuda", dtype=torch.int32)
    padding = [1, 4, B - 1]
    live = [i for i in range(B) if i not in padding]
    slots[padding] = torch.tensor([-1, n, -5], device="cuda", dtype=torch.int32)
    w = torch.randn(B, 4 if D % 4 == 0 else 3, W, device="cuda").to(dtype)
    D_hw = G * D
    want_pool, want_hw_pool = pool.clone(), pool.clone()
    want = lowrank_dynamic_convolution_grouped_step(x, z, U, want_pool, sw, residual=True, slots=slots)
    want_hw = headwise_dynamic_convolution_step(x, w, want_hw_pool, sw.reshape(W, D_hw), residual=True, slots=slots)
    for bad in (float("nan"), float("inf")):
        xb, zb, wb = x.clone(), z.clone(), w.clone()
        xb[padding], zb[padding], wb[padding] = bad, bad, bad
        c, ch = pool.clone(), pool.clone()
        y = lowrank_dynamic_convolution_grouped_step(xb, zb, U, c, sw, residual=True, slots=slots)
        yh = headwise_dynamic_convolution_step(xb, wb, ch, sw.reshape(W, D_hw), residual=True, slots=slots)
        for got, ref in ((y, want), (yh, want_hw)):
            assert got[padding].count_nonzero() == 0 and torch.equal(got[live], ref[live])
        assert torch.equal(c, want_pool) and torch.equal(ch, want_hw_pool)


def test_updates_in_place_are_seen_by_autograd():
    """A cache that autograd has kept cannot be stepped unnoticed, and one that asks for a gradient is refused."""
    x, z, U, cache, sw = make(2, 1, 64, 7, 4, torch.bfloat16)
    w = torch.randn(2, 8, 4, device="cuda").bfloat16()
    steps = (lambda c: lowrank_dynamic_convolution_step(x, z, U[0], c, sw[0]), lambda c: headwise_dynamic_convolution_step(x, w, c))
    for step in steps:
        c, p = cache.clone(), torch.ones((), device="cuda", dtype=torch.bfloat16, requires_grad=True)
        kept = (c * p).sum()
        step(c)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            kept.backward()
        with pytest.raises(RuntimeError, match="no gradient"):
            step(cache.clone().requires_grad_())
        with torch.no_grad():
            step(cache.clone().requires_grad_())
        with torch.inference_mode():
            inside = cache.clone()
            step(inside)
        step(inside)  # (inference tensors have no counter, and may be stepped anywhere)
