"""CPU: the entry points of the operators around the convolutions reject bad arguments before
touching the GPU, size their workspaces, and their Python forms refuse what they cannot do."""
from __future__ import annotations

import copy

import pytest
import torch

import dynamic_conv1d_b200 as dc
from dynamic_conv1d_b200 import _lib

SHAPE, ALIGN, UNSUPPORTED, WORKSPACE, ARGUMENT = 1, 2, 3, 6, 7


def test_step_validation():
    lib = _lib.load()

    def lr(slots=None, slot_bytes=0, B=1, n=1, D=64, R=7, W=4, G=1, dtype=0):
        return lib.dynconv_lr_step(None, None, None, None, None, None, slots, slot_bytes, B, n, D, R, W, G, dtype, 0, None)

    assert lr() == ARGUMENT
    assert lr(B=0) == 0
    assert lr(W=9) == UNSUPPORTED and lr(R=65) == UNSUPPORTED and lr(dtype=5) == UNSUPPORTED
    assert lr(B=2, n=1) == SHAPE and lr(D=0) == SHAPE and lr(G=17) == SHAPE and lr(B=1 << 17, n=1 << 17) == SHAPE
    assert lr(slots=16, slot_bytes=2) == ARGUMENT
    hw = lambda **k: lib.dynconv_hw_step(None, None, None, None, None, None, 0, k.get("B", 1), 1, 64, k.get("H", 4), 4, 0, 0, None)  # noqa: E731
    assert hw() == ARGUMENT and hw(H=5) == SHAPE and hw(B=0) == 0


def test_attention_validation():
    lib = _lib.load()

    def fwd(B=1, T=4, H=2, dk=64, dv=64, dtype=0):
        return lib.dynconv_la_fwd(*([None] * 8), None, 0, B, T, H, dk, dv, 1.0, dtype, None)

    assert fwd() == ARGUMENT
    assert fwd(dk=257) == UNSUPPORTED and fwd(dv=0) == UNSUPPORTED and fwd(dtype=9) == UNSUPPORTED
    assert fwd(H=0) == SHAPE and fwd(B=1 << 16) == SHAPE and fwd(T=-1) == SHAPE and fwd(T=1 << 31) == SHAPE
    assert fwd(T=0) == 0 and fwd(B=0) == 0
    assert lib.dynconv_la_bwd(*([None] * 12), None, 0, 1, 4, 2, 64, 64, 1.0, 0, None) == ARGUMENT
    assert lib.dynconv_la_step(*([None] * 7), 0, None, 1, 1, 2, 64, 64, 1.0, 0, None) == ARGUMENT
    # short inputs with many heads need no segment states; a long one with a few heads does
    assert lib.dynconv_la_workspace_bytes(8, 100, 64, 64, 64, 0, 0) == 0
    assert lib.dynconv_la_workspace_bytes(1, 1 << 16, 4, 128, 128, 0, 0) >= 4 * 128 * 128 * 4


def test_loss_validation():
    lib = _lib.load()

    def fwd(N=4, D=64, V=100, reduction=2, dtype=0, stats=None):
        return lib.dynconv_vocab_loss_fwd(None, None, None, None, None, stats, None, 0, N, D, V, -100, reduction, dtype, None)

    assert fwd() == ARGUMENT
    assert fwd(D=0) == SHAPE and fwd(V=0) == SHAPE and fwd(N=-1) == SHAPE and fwd(V=1 << 23) == SHAPE
    assert fwd(reduction=3) == ARGUMENT and fwd(dtype=4) == UNSUPPORTED
    bwd = lambda dh=None, dw=None: lib.dynconv_vocab_loss_bwd(*([None] * 6), dh, dw, None, 0, 4, 64, 100, -100, 2, 0, None)  # noqa: E731
    assert bwd() == 0  # nothing wanted
    assert bwd(dh=256) == ARGUMENT
    # a piece of the vocabulary, not the logits: 131072 words x 65536 rows in bf16 would be 16 GiB
    n = lib.dynconv_vocab_loss_bwd_workspace_bytes(65536, 1024, 131072, 0, 0, 1)
    assert 0 < n <= (1 << 30)
    assert lib.dynconv_vocab_loss_bwd_workspace_bytes(0, 64, 100, 0, 1, 1) == 0


def test_loss_workspace_of_fp32_parts():
    lib = _lib.load()
    N, D, V = 4096, 2048, 131072
    parts = 6 * N * D + (512 << 20)  # of hidden, and of as many words as 512 MB hold
    n = lib.dynconv_vocab_loss_fwd_workspace_bytes(N, D, V, 1)
    assert parts - (8 << 20) < n <= parts + 8 * N * (V // 64 + 2) + (1 << 20)
    n = lib.dynconv_vocab_loss_bwd_workspace_bytes(N, D, V, 1, 1, 1)
    assert 0 < n < 6 * N * D + (2 << 30)
    # a vocabulary too wide for 1024 words of it in 512 MB still has a workspace
    assert lib.dynconv_vocab_loss_fwd_workspace_bytes(1, 1 << 20, 5000, 1) >= 6 * 1024 << 20
    # bf16 rows of whole 16 bytes are read in place, others are copied
    assert lib.dynconv_vocab_loss_fwd_workspace_bytes(N, 2048, 1000, 0) < 2 << 20
    assert lib.dynconv_vocab_loss_fwd_workspace_bytes(N, 2049, 1000, 0) >= 2 * 2056 * (N + 1000)
    # an unaligned workspace, or an unaligned tensor that is used in place, is refused before any launch
    for k in (0, 1):
        args = [256, 256, 256, 256, 256, 256, 256, 1 << 30, 4, 64, 100, -100, 2]
        args[k] = 264
        assert lib.dynconv_vocab_loss_fwd(*args, 0, None) == ALIGN
    for k in (0, 1, 6, 7):
        args = [256, 256, 256, 256, 256, 256, 256, 256, 256, 1 << 30, 4, 64, 100, -100, 2]
        args[k] = 264
        assert lib.dynconv_vocab_loss_bwd(*args, 0, None) == ALIGN
    args = [256, 256, 256, 256, 256, 256, 264, 1 << 30, 4, 64, 100, -100, 2]
    assert lib.dynconv_vocab_loss_fwd(*args, 1, None) == ALIGN
    args = [256, 256, 256, 256, 256, 256, 256, 256, 264, 1 << 30, 4, 64, 100, -100, 2]
    assert lib.dynconv_vocab_loss_bwd(*args, 1, None) == ALIGN


def test_python_refuses_cpu_tensors():
    x, z, U, c = torch.zeros(1, 8), torch.zeros(1, 3), torch.zeros(3, 16), torch.zeros(1, 1, 8)
    with pytest.raises(AssertionError):
        dc.lowrank_dynamic_convolution_step(x, z, U, c)
    with pytest.raises(AssertionError):
        dc.headwise_dynamic_convolution_step(x, torch.zeros(1, 8, 2), c)
    q = torch.zeros(1, 2, 1, 8)
    with pytest.raises(AssertionError):
        dc.decay_linear_attention(q, q, q, torch.zeros(1))
    with pytest.raises(AssertionError):
        dc.decay_linear_attention_step(q[:, 0], q[:, 0], q[:, 0], torch.zeros(1, 1, 8, 8), torch.zeros(1))
    with pytest.raises(AssertionError):
        dc.linear_cross_entropy(torch.zeros(2, 8), torch.zeros(5, 8), torch.zeros(2, dtype=torch.int64))


@pytest.mark.parametrize("T,W", [(0, 4), (1, 4), (2, 4), (3, 4), (10, 4), (5, 1)])
def test_convolution_cache(T, W):
    x = torch.randn(2, T, 6)
    c = dc.convolution_cache(x, W)
    padded = torch.cat([torch.zeros(2, W - 1, 6), x], 1)
    assert torch.equal(c, padded[:, T:T + W - 1])
    assert c.data_ptr() != x.data_ptr()


def test_layer_arguments():
    with pytest.raises(ValueError):
        dc.ConvolvedLinearAttention(64, 5)
    with pytest.raises(ValueError):
        dc.ConvolvedLinearAttention(64, 4, R=14)
    m = dc.ConvolvedLinearAttention(64, 4).to(torch.bfloat16)
    assert m.log_decay.dtype == torch.float32 and (m.log_decay < 0).all()


def test_gradients_that_cannot_be_differentiated():
    """The mark on a backward whose kernels autograd does not see: ordinary gradients as they are, an error
    for a second derivative whether or not the upstream gradient asks for one."""

    class Cube(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, unused):
            ctx.save_for_backward(x)
            return x**3

        @staticmethod
        @_lib.differentiable_once
        def backward(ctx, d):
            return 3 * ctx.saved_tensors[0]**2 * d, None

    x = torch.tensor([1.0, 2.0], requires_grad=True)
    y = Cube.apply(x, None)
    y.sum().backward(retain_graph=True)
    assert x.grad.tolist() == [3.0, 12.0] and not x.grad.requires_grad
    for loss in (y.sum(), y.square().sum()):
        (g,) = torch.autograd.grad(loss, x, create_graph=True)
        with pytest.raises(RuntimeError, match="differentiated again"):
            (x.sum() + g.sum()).backward()
    (g,) = torch.autograd.grad(Cube.apply(2 * x, None).sum(), x, create_graph=True)  # (through an operator of torch's)
    assert g.tolist() == [24.0, 96.0]
    with pytest.raises(RuntimeError, match="differentiated again"):
        g.sum().backward()


def test_layer_decays_wherever_they_are_first_used():
    """The decays of a layer are the same constants whichever context asks first: an evaluation under
    inference mode before training, or a layer that was built without storage."""
    want = dc.ConvolvedLinearAttention(64, 4).log_decay
    exact = torch.log1p(-torch.exp2(-torch.linspace(5, 12, 4, dtype=torch.float64)))
    assert torch.equal(want, exact.float())
    m = dc.ConvolvedLinearAttention(64, 4)
    m.to("meta")
    with torch.inference_mode():
        assert m.log_decay.device.type == "meta" and not m.log_decay.is_inference()
    p = torch.ones(4, device="meta", requires_grad=True)
    (p * m.log_decay).sum().backward()  # (an inference tensor cannot be kept for this)
    with torch.device("meta"):
        m = dc.ConvolvedLinearAttention(64, 4)
    assert m.log_decay.device.type == "meta"
    m.to_empty(device="cpu")
    assert torch.equal(m.log_decay, want)
    with torch.inference_mode():
        m = dc.ConvolvedLinearAttention(64, 4)
    assert torch.equal(m.log_decay, want) and not m.log_decay.is_inference()
    m = copy.deepcopy(dc.ConvolvedLinearAttention(64, 4).to("meta"))
    assert m.log_decay.device.type == "meta" and m.to_empty(device="cpu").log_decay.equal(want)
