"""GPU: the vocabulary loss and its gradients against the definition in 64 bits.

Tolerances (relative 2-norm):
  loss : fp32 from fp32 logits whose terms are exact products; a logit's sum of D <= 512
         terms is off by at most 512 * 2^-24 of their absolute sum, which the tests keep
         below 16: 16 * 512 * 2^-24 = 4.9e-4 absolute at the worst, 1e-5 relative in the
         loss's own size at the usual square root of it;
  bf16 gradients: the logits' gradient rounded once and the result once, each by less than
         2^-9 of the values in the root mean square: 2 * 2^-9;
  fp32 gradients: sums of up to 512 terms at 2^-24, and exp() of logits off by the same
         relative amount: 1024 * 2^-24.
"""
from __future__ import annotations

import math

import pytest
import torch

from dynamic_conv1d_b200 import _lib
from dynamic_conv1d_b200 import check_device, linear_cross_entropy

pytestmark = pytest.mark.gpu

GRAD = {torch.bfloat16: 2.0**-8, torch.float32: 1024 * 2.0**-24}
LOSS = 1e-5
BOTH = [torch.bfloat16, torch.float32]
IGNORE = -100


def rel(a, b):
    a, b = a.detach().double(), b.detach().double()
    n, d = torch.linalg.vector_norm(b), torch.linalg.vector_norm(a - b)
    return (d / n if n > 0 else d).item()


def make(N, D, V, dtype, seed=0, scale=1.5, ignored=0.2):
    g = torch.Generator(device="cuda").manual_seed(seed)
    h = torch.randn(N, D, device="cuda", generator=g).to(dtype)
    w = (torch.randn(V, D, device="cuda", generator=g) * scale * D**-0.5).to(dtype)
    t = torch.randint(0, V, (N,), device="cuda", generator=g)
    drop = torch.rand(N, device="cuda", generator=g) < ignored
    if N:
        drop[0] = False
    return h, w, torch.where(drop, torch.full_like(t, IGNORE), t)


def definition(h, w, t, up, reduction):
    """(loss, dhidden, dweight) in 64 bits for upstream gradient `up`."""
    h, w = h.double(), w.double()
    keep = t != IGNORE
    l = h @ w.T
    lse = torch.logsumexp(l, 1)
    rows = torch.where(keep, lse - l.gather(1, t.clamp(min=0)[:, None])[:, 0], 0.0)
    n = keep.sum()
    loss = {"none": rows, "sum": rows.sum(), "mean": rows.sum() / n}[reduction]
    f = (up.double() if reduction != "mean" else up.double() / n).expand(len(t)) * keep
    d = torch.exp(l - lse[:, None])
    d.scatter_add_(1, t.clamp(min=0)[:, None], -torch.ones_like(d[:, :1]))
    d *= f[:, None]
    return loss, d @ w, d.T @ h


def check(h, w, t, reduction="mean", up=None, loss_tol=LOSS):
    if up is None:
        up = torch.tensor(1.0, device="cuda")
    own = [x.detach().requires_grad_() for x in (h, w)]
    loss = linear_cross_entropy(*own, t, reduction=reduction)
    loss.backward(up)
    check_device(loss)
    rl, rh, rw = definition(h, w, t, up, reduction)
    assert loss.dtype == torch.float32 and loss.shape == rl.shape
    got = (rel(loss, rl), rel(own[0].grad, rh), rel(own[1].grad, rw))
    assert got[0] <= loss_tol and got[1] <= GRAD[h.dtype] and got[2] <= GRAD[h.dtype], got
    return loss.detach(), own[0].grad, own[1].grad


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("N,D,V", [(1, 8, 2), (1, 64, 1), (3, 16, 7), (5, 13, 30), (64, 64, 64), (65, 64, 65), (127, 72, 300), (128, 128, 256),
                                   (129, 136, 257), (200, 256, 1000), (257, 512, 511), (300, 33, 513), (2, 512, 5000), (1000, 8, 300)])
def test_sizes(dtype, N, D, V):
    check(*make(N, D, V, dtype, seed=N + V))


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
def test_reductions(dtype, reduction):
    h, w, t = make(150, 64, 500, dtype)
    up = torch.randn(150, device="cuda") if reduction == "none" else torch.tensor(0.37, device="cuda")
    check(h, w, t, reduction, up)


@pytest.mark.parametrize("dtype", BOTH)
def test_shapes_and_expanded_upstream(dtype):
    h, w, t = make(60, 64, 200, dtype)
    h3, t3 = h.view(4, 15, 64).requires_grad_(), t.view(4, 15)
    rows = linear_cross_entropy(h3, w, t3, reduction="none")
    assert rows.shape == (4, 15)
    rows.sum().backward()  # an expanded scalar as upstream gradient
    _, rh, _ = definition(h, w, t, torch.tensor(1.0, device="cuda"), "sum")
    assert rel(h3.grad.view(60, 64), rh) <= GRAD[dtype]


@pytest.mark.parametrize("dtype", BOTH)
def test_several_pieces(dtype):
    """More rows and words than one piece of the vocabulary holds."""
    N, V = (33000, 9001) if dtype == torch.bfloat16 else (17000, 9001)
    check(*make(N, 16, V, dtype))


@pytest.mark.parametrize("dtype", BOTH)
def test_more_rows_than_one_launch(dtype):
    """The forward takes 32768 rows at a time."""
    h, w, t = make(40001, 16, 200, dtype)
    rows = linear_cross_entropy(h, w, t, reduction="none")
    want, _, _ = definition(h, w, t, torch.ones(40001, device="cuda"), "none")
    assert rel(rows, want) <= LOSS
    check(h, w, t)


def test_long_inner_dimensions():
    """Few tiles, long sums: the inner dimension is spread over several CTAs."""
    check(*make(20, 128, 30000, torch.bfloat16))
    check(*make(20, 64, 9000, torch.float32))
    check(*make(6000, 64, 100, torch.bfloat16))


def test_unaligned_tensors():
    """Views that begin off 16 bytes: read through aligned copies."""
    N, D, V = 200, 64, 500
    h, w, t = make(N, D, V, torch.bfloat16)
    shift = lambda x: torch.cat([x.new_zeros(1), x.flatten()])[1:].view(x.shape)  # noqa: E731
    check(shift(h), shift(w), t)


def test_channels_beyond_one_chain():
    """More than 2048 products in a logit: summed in parts (bf16)."""
    for D in (2056, 4096, 5000):
        check(*make(130, D, 300, torch.bfloat16), loss_tol=2 * LOSS)


@pytest.mark.parametrize("dtype", BOTH)
def test_gradient_of_one_side(dtype):
    h, w, t = make(100, 64, 300, dtype)
    _, rh, rw = check(h, w, t)
    a = h.detach().requires_grad_()
    linear_cross_entropy(a, w, t).backward()
    assert torch.equal(a.grad, rh)
    b = w.detach().requires_grad_()
    linear_cross_entropy(h, b, t).backward()
    assert torch.equal(b.grad, rw)


@pytest.mark.parametrize("dtype", BOTH)
def test_all_rows_ignored(dtype):
    h, w, t = make(70, 64, 100, dtype)
    t = torch.full_like(t, IGNORE)
    for reduction, want in (("mean", float("nan")), ("sum", 0.0)):
        own = [x.detach().requires_grad_() for x in (h, w)]
        loss = linear_cross_entropy(*own, t, reduction=reduction)
        loss.backward()
        assert (loss.isnan() if want != want else loss == want).item()
        assert own[0].grad.count_nonzero() == 0 and own[1].grad.count_nonzero() == 0
    assert linear_cross_entropy(h, w, t, reduction="none").count_nonzero() == 0


@pytest.mark.parametrize("dtype", BOTH)
def test_target_outside_the_vocabulary(dtype):
    h, w, t = make(70, 64, 100, dtype, ignored=0.0)
    t[3], t[4] = 100, -1
    rows = linear_cross_entropy(h, w, t, reduction="none")
    assert rows[3].isnan() and rows[4].isnan() and rows.isnan().sum() == 2
    own = [x.detach().requires_grad_() for x in (h, w)]
    linear_cross_entropy(*own, t).backward()
    assert own[0].grad[3].count_nonzero() == 0 and own[0].grad.isfinite().all() and own[1].grad.isfinite().all()
    # another index to ignore: -1 is then an ignored row, -100 is outside
    t2 = t.clone()
    t2[3] = 5
    assert linear_cross_entropy(h, w, t2, ignore_index=-1).isfinite()


@pytest.mark.parametrize("dtype", BOTH)
def test_large_logits(dtype):
    """Logits of several hundred: nothing overflows, and a row dominated by one word is exact
    there.  The loss is then a difference of logits of about 400 computed with 2^-24 * 64 each."""
    h, w, t = make(90, 64, 400, dtype, scale=100.0)
    own = [x.detach().requires_grad_() for x in (h, w)]
    loss = linear_cross_entropy(*own, t)
    loss.backward()
    rl, rh, rw = definition(h, w, t, torch.tensor(1.0, device="cuda"), "mean")
    assert rel(loss, rl) <= 1e-4
    # exp() of logits off by 400 * 64 * 2^-24 = 1.5e-3
    tol = GRAD[dtype] + 1.5e-3
    assert rel(own[0].grad, rh) <= tol and rel(own[1].grad, rw) <= tol


def test_infinite_and_nan_rows():
    h, w, t = make(80, 64, 300, torch.bfloat16, ignored=0.0)
    h = h.clone()
    h[7, 3] = float("nan")
    rows = linear_cross_entropy(h, w, t, reduction="none")
    assert rows[7].isnan() and rows.isnan().sum() == 1


def test_gradient_against_differences():
    """Central difference in fp32 along a direction: step 1e-2, error of the third order
    (1e-4 of the derivative's size, measured on the definition in 64 bits) plus the fp32
    loss's own rounding 1e-6 / 1e-2."""
    h, w, t = make(40, 32, 60, torch.float32)
    for i in range(2):
        x = [h, w]
        a = x[i].detach().requires_grad_()
        x[i] = a
        linear_cross_entropy(x[0], x[1], t).backward()
        e = torch.randn(a.shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2))
        e /= torch.linalg.vector_norm(e)
        with torch.no_grad():
            f = lambda s: linear_cross_entropy(*[y + s * e if j == i else y for j, y in enumerate((h, w))], t).double()  # noqa: E731
            dif = (f(1e-2) - f(-1e-2)) / 2e-2
        ana = (a.grad.double() * e.double()).sum()
        assert abs(dif - ana) <= 1e-4 * torch.linalg.vector_norm(a.grad) + 1e-4


def test_empty_batch():
    h, w, t = make(0, 64, 100, torch.bfloat16)
    w.requires_grad_()
    loss = linear_cross_entropy(h, w, t, reduction="sum")
    loss.backward()
    assert loss == 0 and w.grad.count_nonzero() == 0
    assert linear_cross_entropy(h, w, t).isnan()
    assert linear_cross_entropy(h, w, t, reduction="none").shape == (0,)


def test_weight_of_another_type():
    h, w, t = make(50, 64, 100, torch.bfloat16)
    w32 = w.float().requires_grad_()
    linear_cross_entropy(h, w32, t).backward()
    _, _, rw = definition(h, w, t, torch.tensor(1.0, device="cuda"), "mean")
    assert w32.grad.dtype == torch.float32 and rel(w32.grad, rw) <= GRAD[torch.bfloat16]


def test_same_bits_again_and_other_stream():
    h, w, t = make(300, 128, 3000, torch.bfloat16)
    one = check(h, w, t)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        own = [x.detach().requires_grad_() for x in (h, w)]
        loss = linear_cross_entropy(*own, t)
        loss.backward()
    torch.cuda.current_stream().wait_stream(st)
    for a, b in zip(one, (loss.detach(), own[0].grad, own[1].grad)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("N,D,V", [(300, 256, 600), (130, 320, 700), (700, 1000, 900), (1021, 256, 4999), (40, 2048, 300), (2000, 129, 257)])
def test_fp32_keeps_its_digits(N, D, V):
    """fp32 tensors are multiplied as three bf16 parts: 24 digits, of whose products those below
    2^-23 are left out (2^-22 of a sum, for three of them), in tensor-core sums of 256 that lose
    at most 2^-30 each time (2^-22), added up in fp32 (2^-24 for each 256).  Logits of up to 8 are
    then off by 8 * 2^-21 = 2^-18 and exp() by that factor; the gradients' own sums add 2^-21
    each: below 2^-17, where two parts, or bf16, would not come."""
    h, w, t = make(N, D, V, torch.float32, seed=D)
    own = [x.detach().requires_grad_() for x in (h, w)]
    loss = linear_cross_entropy(*own, t)
    loss.backward()
    check_device(loss)
    rl, rh, rw = definition(h, w, t, torch.tensor(1.0, device="cuda"), "mean")
    got = (rel(loss, rl), rel(own[0].grad, rh), rel(own[1].grad, rw))
    assert max(got) <= 2.0**-17, got


@pytest.mark.parametrize("N,D,V", [(1021, 257, 4999), (130, 2051, 300), (17000, 12, 9001), (40, 30, 30000), (1, 1, 1)])
def test_bf16_widths_off_16_bytes(N, D, V):
    """Rows that are no multiple of 16 bytes are copied with padding."""
    check(*make(N, D, V, torch.bfloat16, seed=D))


def test_fp32_unaligned_and_odd_widths():
    """The parts are copies of their own: any base and any width, the same result."""
    shift = lambda x: torch.cat([x.new_zeros(1), x.flatten()])[1:].view(x.shape)  # noqa: E731
    for D in (64, 66, 67):
        h, w, t = make(200, D, 500, torch.float32)
        for a, b in zip(check(h, w, t), check(shift(h), shift(w), t)):
            assert torch.equal(a, b)


def test_fp32_vocabulary_larger_than_its_parts_at_once():
    """512 MB of parts hold 10752 words of 8192 channels."""
    check(*make(40, 8192, 11000, torch.float32), loss_tol=2 * LOSS)


def test_fp32_extremes():
    """Numbers that would round to infinity in bf16 stay finite; NaN and infinite rows are NaN, and
    ignored ones count for nothing in the loss."""
    h, w, t = make(80, 64, 300, torch.float32, ignored=0.0)
    h, w = h.clone(), w.clone()
    h[:, 5] = 1e-30
    w[:, 5] = 0.0
    w[7, 5] = torch.finfo(torch.float32).max  # a logit of 3.4e8 in every row
    rows = linear_cross_entropy(h, w, torch.full_like(t, 8), reduction="none")
    want, _, _ = definition(h, w, torch.full_like(t, 8), torch.ones(80, device="cuda"), "none")
    assert rel(rows, want) <= LOSS
    w[7, 5] = 0.0
    h[3, 3], h[4, 3], h[5, 3] = float("nan"), float("inf"), float("-inf")
    rows = linear_cross_entropy(h, w, t, reduction="none")
    assert rows[3:6].isnan().all() and rows.isnan().sum() == 3
    t[3:6] = IGNORE
    assert linear_cross_entropy(h, w, t).isfinite()


def test_fp32_same_bits_again():
    h, w, t = make(300, 136, 3000, torch.float32)
    for a, b in zip(check(h, w, t), check(h, w, t)):
        assert torch.equal(a, b)


def test_refusals():
    h, w, t = make(10, 64, 50, torch.bfloat16)
    good = dict(hidden=h, weight=w, target=t)
    for bad in (dict(hidden=h.cpu()), dict(hidden=h.half(), weight=w.half()), dict(hidden=h[:, ::2]), dict(weight=w[:, :32]), dict(weight=w.T),
                dict(target=t[:5]), dict(target=t.int()), dict(target=t.cpu()), dict(reduction="max")):
        with pytest.raises((AssertionError, TypeError, RuntimeError)):
            linear_cross_entropy(**(good | bad))


def test_no_second_derivative():
    """The gradients are no functions of the inputs to autograd: differentiating them is an error, not a
    constant."""
    h, w, t = make(20, 64, 50, torch.float32)
    h.requires_grad_()
    loss = linear_cross_entropy(h, w, t)
    (g,) = torch.autograd.grad(loss, h, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiated again"):
        (h.sum() + g.square().sum()).backward()
    (g1,) = torch.autograd.grad(linear_cross_entropy(h, w, t), h)
    assert torch.equal(g, g1)


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("D", [64, 65, 512])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_rows_that_count_for_nothing_may_hold_anything(dtype, bad, D, reduction):
    """Hidden states of ignored rows, and of rows whose target is no word, reach neither gradient."""
    h, w, t = make(300, D, 700, dtype)
    ignored = (t == IGNORE).nonzero()[:, 0]
    up = torch.randn(300, device="cuda") if reduction == "none" else torch.tensor(1.0, device="cuda")

    def grads(h, t, need_h=True):
        own = [h.detach().requires_grad_(need_h), w.detach().requires_grad_()]
        loss = linear_cross_entropy(*own, t, reduction=reduction)
        loss.backward(up)
        check_device(loss)
        return loss.detach(), own[0].grad, own[1].grad

    hb = h.clone()
    hb[ignored] = bad
    want, got = grads(h, t), grads(hb, t)
    for a, b in zip(want, got):
        assert b.isfinite().all() and torch.equal(a, b)
    assert got[1][ignored].count_nonzero() == 0
    assert torch.equal(grads(hb, t, False)[2], want[2])
    t = t.clone()
    t[ignored[::2]] = 700  # no word either: the loss says so, the gradients leave it out
    _, _, rw = grads(h, t)
    _, gh, gw = grads(hb, t)
    assert gh.isfinite().all() and torch.equal(gw, rw)


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("D", [64, 65, 2056])
@pytest.mark.parametrize("first,count", [(0, 1), (0, 16), (0, 32), (0, 128), (128, 128), (256, 256), (300, 1), (320, 80), (0, 400)])
def test_words_that_are_nan(dtype, D, first, count):
    """One NaN among a row's logits makes its loss NaN, whichever words have it."""
    h, w, t = make(150, D, 400, dtype, ignored=0.0)
    w = w.clone()
    w[first:first + count] = float("nan")
    t = torch.where((t >= first) & (t < first + count), torch.full_like(t, 200 if first != 128 else 50), t)
    assert linear_cross_entropy(h, w, t, reduction="none").isnan().all()
    assert linear_cross_entropy(h, w, t).isnan()


@pytest.mark.parametrize("D", [8, 9, 2056])
@pytest.mark.parametrize("first,count", [(0, 1), (0, 32), (0, 128), (256, 256), (320, 80)])
def test_words_that_are_excluded(D, first, count):
    """Logits of minus infinity take their words out of the sum; a row with nothing else, or with plus
    infinity, has no loss."""
    h, w, t = make(150, D, 400, torch.bfloat16, ignored=0.0)
    h[:, 0], w = 1.0, w.clone()
    w[first:first + count, 0] = -float("inf")
    t = torch.where((t >= first) & (t < first + count), torch.full_like(t, 200), t)
    keep = [v for v in range(400) if not first <= v < first + count]
    own = [x.detach().requires_grad_() for x in (h, w)]
    rows = linear_cross_entropy(*own, t, reduction="none")
    l = h.double() @ w[keep].double().T
    lt = (h.double() * w[t].double()).sum(1)
    assert rel(rows, torch.logsumexp(l, 1) - lt) <= 2 * LOSS
    w[0, 0] = float("inf")
    assert linear_cross_entropy(h, w, t, reduction="none").isnan().all()
    w[:, 0] = -float("inf")
    assert linear_cross_entropy(h, w, t, reduction="none").isnan().all()


def dominated(c, D, V, dtype):
    """Rows whose target's logit is c + r_t, all others being r_v in [-3, 3]: exact in every product and sum
    (c and r are multiples of 1/32, below 128).  Returns (hidden, weight, target, loss in 64 bits)."""
    N = len(c)
    g = torch.Generator(device="cuda").manual_seed(N)
    r = (torch.randn(V, device="cuda", generator=g).clamp(-3, 3) * 32).round() / 32
    t = torch.randperm(V, device="cuda", generator=g)[:N]
    h, w = torch.zeros(N, D, device="cuda"), torch.zeros(V, D, device="cuda")
    i = torch.arange(N, device="cuda")
    h[i, i], w[t, i] = torch.tensor(c, device="cuda"), 1.0
    h[:, N], w[:, N] = 1.0, r
    l = h.double() @ w.double().T
    d = l - l.gather(1, t[:, None])
    d[i, t] = -math.inf
    return h.to(dtype), w.to(dtype), t, torch.log1p(d.exp().sum(1))


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("D", [16, 17])
@pytest.mark.parametrize("V", [500, 50000])
@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
def test_rows_dominated_by_their_target(dtype, D, V, reduction):
    """A confident row's loss and gradient keep their digits, row by row: they are what the other words
    add, not a difference of two large numbers.

    Each other word's exponent, below 128, is rounded to 2^-18 (2^-18.5 of the word's share) and its
    factor log2(e) is off by 2^-26 (2^-20), exp() by 2^-22, and up to 100 sums by 2^-24 each (2^-17.3): 1e-5
    together.  In fp32 the gradient's products add 2^-20; in bf16 it is rounded twice (2^-8 each)."""
    c = [0.0, 4.0, 10.0, 14.0, 18.0, 22.0, 25.0, 32.0, 60.0]
    h, w, t, want = dominated(c, D, V, dtype)
    own = [x.requires_grad_() for x in (h, w)]
    loss = linear_cross_entropy(*own, t, reduction=reduction)
    up = torch.linspace(1, 2, len(c), device="cuda") if reduction == "none" else torch.tensor(1.0, device="cuda")
    loss.backward(up)
    check_device(loss)
    ref = {"none": want, "sum": want.sum(), "mean": want.mean()}[reduction]
    assert ((loss.detach().double() - ref).abs() <= 1e-5 * ref).all()
    # channel n is in row n's target alone: its gradients are the target's own
    n = torch.arange(len(c), device="cuda")
    dl = torch.expm1(-want) * (up.double() if reduction == "none" else 1.0 / (len(c) if reduction == "mean" else 1))
    tol = 1.1e-5 if dtype == torch.float32 else 2.0**-7
    dh = own[0].grad[n, n].double()
    assert ((dh - dl).abs() <= tol * dl.abs()).all(), (dh / dl - 1)
    dw, to = own[1].grad[t, n].double(), dl * torch.tensor(c, device="cuda")
    assert ((dw - to).abs() <= tol * to.abs()).all(), (dw / to - 1)


@pytest.mark.parametrize("dtype", BOTH)
def test_equal_logits(dtype):
    """Many words share the maximum: log(V), and a gradient of 1/V (2^-22: log1p of an exact sum)."""
    for V in (1, 2, 31, 128, 129, 5000):
        h, w = torch.ones(3, 16, device="cuda", dtype=dtype), torch.full((V, 16), 0.5, device="cuda", dtype=dtype)
        rows = linear_cross_entropy(h, w, torch.tensor([0, V // 2, V - 1], device="cuda"), reduction="none")
        assert ((rows.double() - math.log(V)).abs() <= 2.0**-22 * math.log(V)).all()


@pytest.mark.parametrize("dtype", BOTH)
def test_callers_that_keep_lse_alone(dtype):
    """The library without DYNCONV_LOSS_KEEP_ROWS: lse has N numbers and none is written behind them; the
    same loss, and gradients that differ by lse's rounding only."""
    N, D, V = 130, 64, 300
    h, w, t = make(N, D, V, dtype)
    rl, rh, rw = check(h, w, t)
    lib, code = _lib.load(), _lib.dtype_code(dtype)
    stats, lse, loss = torch.empty(2, device="cuda"), torch.full((N + 8,), 7.0, device="cuda"), torch.empty((), device="cuda")
    dh, dw, up = torch.empty_like(h), torch.empty_like(w), torch.ones((), device="cuda")
    n = max(lib.dynconv_vocab_loss_fwd_workspace_bytes(N, D, V, code), lib.dynconv_vocab_loss_bwd_workspace_bytes(N, D, V, code, 1, 1))
    ws = torch.empty(n, device="cuda", dtype=torch.uint8)
    tail = (ws.data_ptr(), n, N, D, V, IGNORE, 2, code, _lib.raw_stream(h))
    _lib.check(lib.dynconv_vocab_loss_fwd(*(x.data_ptr() for x in (h, w, t, loss, lse, stats)), *tail))
    _lib.check(lib.dynconv_vocab_loss_bwd(*(x.data_ptr() for x in (h, w, t, lse, stats, up, dh, dw)), *tail))
    check_device(h)
    assert torch.equal(loss, rl) and (lse[N:] == 7.0).all()
    assert rel(lse[:N], torch.logsumexp(h.double() @ w.double().T, 1)) <= LOSS
    assert rel(dh, rh) <= GRAD[dtype] and rel(dw, rw) <= GRAD[dtype]


def long_rows(D, signed):
    """Rows whose targets have logits of 5 to 40, among 300 words of about one (all h positive: and among the
    other rows' targets)."""
    N, V = 12, 300
    g = torch.Generator(device="cuda").manual_seed(D)
    h = torch.rand(N, D, device="cuda", generator=g).add_(0.5)
    if signed:
        h = torch.where(torch.rand(N, D, device="cuda", generator=g) < 0.5, -h, h)
    h = h.bfloat16()
    w = (torch.randn(V, D, device="cuda", generator=g) * D**-0.5).bfloat16()
    t = torch.randperm(V, device="cuda", generator=g)[:N]
    size = torch.tensor([5.0, 10.0, 20.0, 40.0], device="cuda").repeat(3)
    w[t] = (h.float() * (size / h.float().square().sum(1))[:, None]).bfloat16()
    return h, w, t, size


@pytest.mark.parametrize("signed", [False, True])
@pytest.mark.parametrize("D", [2056, 4096, 5000])
def test_rows_of_long_sums(D, signed):
    """Loss and gradient row by row where a logit has more than 2048 products (bf16).

    A logit of 40 is a sum whose products the tensor core truncates, by 2^-30 of the sum for each of
    2048: 8e-5, and so is every word's share.  dl is rounded by 2^-8 of each entry, the result by 2^-8."""
    h, w, t, _ = long_rows(D, signed)
    l = h.double() @ w.double().T
    i = torch.arange(len(t), device="cuda")
    share = (l - l.gather(1, t[:, None])).exp()
    share[i, t] = 0.0
    want = torch.log1p(share.sum(1))
    dl = share * torch.exp(-want)[:, None]
    dl[i, t] = torch.expm1(-want)
    own = h.requires_grad_()
    rows = linear_cross_entropy(own, w, t, reduction="none")
    rows.sum().backward()
    assert ((rows.detach().double() - want).abs() <= 2e-4 * want).all(), rows.detach().double() / want - 1
    ref = dl @ w.double()
    size = lambda x: torch.linalg.vector_norm(x.double(), dim=1)  # noqa: E731
    err, terms = size(own.grad.double() - ref), dl.abs() @ size(w)
    assert (err <= (2.0**-8 + 2e-4) * terms + 2.0**-8 * size(ref)).all(), err / terms


@pytest.mark.parametrize("D", [64, 2048, 2056, 4096, 8192])
def test_forward_and_backward_add_up_alike(D):
    """A gradient without the rows' losses is a difference of the backward's logit and the forward's sums:
    the logits are the same bits in both, so what is left at the target of a row that it has to itself is
    the rounding of lse, twice (2^-24 of it each), of the exponent and of exp(): less than 4 * 2^-24 of lse."""
    h, w, t, size = long_rows(D, True)
    w = w * 0.01
    w[t] *= 100
    N, V = len(t), w.shape[0]
    lib = _lib.load()
    stats, lse, loss = torch.empty(2, device="cuda"), torch.empty(N, device="cuda"), torch.empty((), device="cuda")
    dh, up = torch.empty_like(h), torch.ones((), device="cuda")
    n = max(lib.dynconv_vocab_loss_fwd_workspace_bytes(N, D, V, 0), lib.dynconv_vocab_loss_bwd_workspace_bytes(N, D, V, 0, 1, 0))
    ws = torch.empty(n, device="cuda", dtype=torch.uint8)
    tail = (ws.data_ptr(), n, N, D, V, IGNORE, 1, 0, _lib.raw_stream(h))
    _lib.check(lib.dynconv_vocab_loss_fwd(*(x.data_ptr() for x in (h, w, t, loss, lse, stats)), *tail))
    _lib.check(lib.dynconv_vocab_loss_bwd(*(x.data_ptr() for x in (h, w, t, lse, stats, up, dh)), None, *tail))
    check_device(h)
    # the largest logits: the other words have exp(-40) of the row, below fp32's rounding of the rest
    big = size == 40
    along = (dh.double() * w[t].double()).sum(1) / w[t].double().square().sum(1)  # dl at the target
    assert (along[big].abs() <= 4 * 2.0**-24 * 40).all(), along


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("D", [64, 65])
def test_hidden_gradient_alone_with_ignored_rows_of_anything(dtype, D):
    h, w, t = make(300, D, 700, dtype)
    hb = torch.where((t == IGNORE)[:, None], torch.full_like(h, float("nan")), h)
    want, got = (torch.autograd.grad(linear_cross_entropy(x.requires_grad_(), w, t), x)[0] for x in (h, hb))
    assert torch.equal(got, want) and got[t == IGNORE].count_nonzero() == 0
