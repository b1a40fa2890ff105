"""CPU: the entry points of the gated delta rule and of the norms reject bad arguments before touching the GPU,
and size what they keep and work in."""
from __future__ import annotations

import pytest
import torch

import dynamic_conv1d_b200 as dc
from dynamic_conv1d_b200 import _lib
from dynamic_conv1d_b200.norm import _pair, _rows

SHAPE, ALIGN, UNSUPPORTED, WORKSPACE, ARGUMENT = 1, 2, 3, 6, 7


def test_rule_validation():
    lib = _lib.load()

    def fwd(B=1, T=4, H=2, dk=64, dv=64, dtype=0):
        return lib.dynconv_delta_fwd(*([None] * 9), 0, None, None, 0, B, T, H, dk, dv, 1.0, dtype, None)

    def bwd(B=1, T=4, H=2, dk=64, dv=64, dtype=0):
        return lib.dynconv_delta_bwd(*([None] * 5), 0, *([None] * 10), 0, B, T, H, dk, dv, 1.0, dtype, None)

    def step(B=1, n=1, H=2, dk=64, dv=64, dtype=0, slots=None, slot_bytes=0):
        return lib.dynconv_delta_step(*([None] * 7), slots, slot_bytes, None, B, n, H, dk, dv, 1.0, dtype, None)

    for call in (fwd, bwd, step):
        assert call() == ARGUMENT
        assert call(dk=129) == UNSUPPORTED and call(dk=0) == UNSUPPORTED and call(dv=257) == UNSUPPORTED and call(dtype=9) == UNSUPPORTED
        assert call(H=0) == SHAPE and call(B=1 << 16) == SHAPE and call(B=-1) == SHAPE and call(H=1 << 40) == SHAPE
        assert call(B=0) == 0
    assert fwd(T=-1) == SHAPE and bwd(T=1 << 31) == SHAPE and fwd(T=0) == 0 and bwd(T=0) == 0
    assert step(B=2, n=1) == SHAPE and step(n=-1) == SHAPE and step(slots=16, slot_bytes=2) == ARGUMENT


def test_rule_workspaces_and_alignment():
    """Addresses that are never used: the call is refused before a launch."""
    lib = _lib.load()
    assert lib.dynconv_delta_workspace_bytes(1, 0, 2, 64, 64, 0, 0) == 0 and lib.dynconv_delta_kept_bytes(1, 4, 2, 200, 64, 0) == 0
    # one state of 64 x 64 and 64 tokens' r in two parts for each of two heads' two chunks
    assert lib.dynconv_delta_kept_bytes(1, 100, 2, 64, 64, 0) == 2 * 2 * (64 * 64 * 2 + 2 * 64 * 64 * 2)
    assert lib.dynconv_delta_workspace_bytes(1, 100, 2, 64, 64, 0, 1) > lib.dynconv_delta_workspace_bytes(1, 100, 2, 64, 64, 0, 0)
    # widths that are read through copies need room for them
    assert lib.dynconv_delta_workspace_bytes(1, 100, 2, 63, 64, 0, 0) > lib.dynconv_delta_workspace_bytes(1, 100, 2, 64, 64, 0, 0)
    import ctypes

    B, T, H, d = 1, 4, 2, 64
    dense = lambda n: [T * H * n, H * n, n]  # noqa: E731
    need = lib.dynconv_delta_workspace_bytes(B, T, H, d, d, 0, 0)

    def fwd(q=1 << 20, strides=None, ws=1 << 20, n=need, kept=None, kept_bytes=0):
        s = (ctypes.c_int64 * 18)(*(strides or dense(d)), *dense(d), *dense(d), *dense(1), *dense(1), *dense(d))
        return lib.dynconv_delta_fwd(q, *([1 << 20] * 4), None, 1 << 20, None, kept, kept_bytes, s, ws, n, B, T, H, d, d, 1.0, 0, None)

    assert fwd(ws=None) == WORKSPACE and fwd(n=need - 1) == WORKSPACE and fwd(kept=1 << 20, kept_bytes=10) == WORKSPACE
    assert fwd(ws=(1 << 20) + 8) == ALIGN and fwd(q=(1 << 20) + 2) == ALIGN
    assert fwd(strides=[T * H * d, H * d + 1, d]) == ALIGN and fwd(strides=[T * H * d, H * d, 0]) == ALIGN


def test_norm_validation():
    lib = _lib.load()
    g = lambda N=1, G=1, D=64, dtype=0: lib.dynconv_gated_norm_fwd(*([None] * 5), N, G, D, 1e-6, 1.0, dtype, None)  # noqa: E731
    r = lambda N=1, D=64, dtype=0: lib.dynconv_residual_norm_fwd(*([None] * 4), 1.0, None, None, N, D, 1e-6, dtype, None)  # noqa: E731
    for call in (g, r):
        assert call() == ARGUMENT and call(N=0) == 0 and call(N=-1) == SHAPE and call(D=0) == SHAPE
        assert call(D=16385) == UNSUPPORTED and call(dtype=3) == UNSUPPORTED
    assert g(N=1 << 40, G=1 << 30) == SHAPE
    assert lib.dynconv_gated_norm_bwd(*([None] * 9), 0, 1, 1, 64, 1e-6, 1.0, 0, None) == ARGUMENT
    assert lib.dynconv_residual_norm_bwd(*([None] * 4), 1.0, *([None] * 7), 0, 1, 64, 1e-6, 0, None) == ARGUMENT
    assert lib.dynconv_norm_workspace_bytes(0) == 0 and lib.dynconv_norm_workspace_bytes(16385) == 0
    assert lib.dynconv_norm_workspace_bytes(64) % 256 == 0


def test_rows_fold():
    """Leading dimensions fold into two where their strides allow it; the rows' addresses stay the same."""
    t = torch.arange(3 * 20 * 384.0).view(3, 20, 384)
    for x in (t, t[..., 128:256].unflatten(-1, (2, 64)), t[..., ::2], t[:, :1], t[1], t[0, 0], t.transpose(0, 1), t[:, ::2, :64],
              t[..., :256].unflatten(-1, (4, 64)).transpose(1, 2), t[:0]):
        y, n, g, outer, inner = _rows(x)
        assert n * g * x.shape[-1] == x.numel()
        flat = torch.as_strided(y, (n, g, x.shape[-1]), (outer, inner, 1), y.storage_offset())
        assert torch.equal(flat.reshape(x.shape), x)
    x, z = t[..., 128:256].unflatten(-1, (2, 64)), torch.randn(3, 20, 2, 64)
    for a, b in ((x, z), (z, x), (x, z.transpose(0, 1).contiguous().transpose(0, 1)), (x, x)):
        p, q, n, g, s = _pair(a, b)
        for y, src, o, i in ((p, a, s[0], s[1]), (q, b, s[2], s[3])):
            assert torch.equal(torch.as_strided(y, (n, g, 64), (o, i, 1), y.storage_offset()).reshape(a.shape), src)


def test_python_refuses_cpu_tensors():
    t = torch.zeros(1, 4, 2, 8)
    with pytest.raises(AssertionError):
        dc.gated_delta_rule(t, t, t, t[..., 0], t[..., 0])
    with pytest.raises(AssertionError):
        dc.gated_delta_rule_step(t[0], t[0], t[0], torch.zeros(4, 2, 8, 8), t[0, ..., 0], t[0, ..., 0])
    with pytest.raises(AssertionError):
        dc.gated_rms_norm(t)
    with pytest.raises(AssertionError):
        dc.residual_rms_norm(t, t, t[0, 0, 0])


def test_layer_arguments():
    with pytest.raises(ValueError):
        dc.ConvolvedGatedDelta(100, 3)
    with pytest.raises(ValueError):
        dc.ConvolvedGatedDelta(256, 1)
    with pytest.raises(ValueError):
        dc.ConvolvedGatedDelta(64, 2, R=16)
    m = dc.ConvolvedGatedDelta(64, 2)
    # the steps that the bias stands for lie between 0.001 and 0.1
    steps = torch.nn.functional.softplus(m.dt_bias)
    assert ((steps > 9e-4) & (steps < 0.11)).all()
    assert dc.ResidualRMSNorm(8).scale is None and dc.ResidualRMSNorm(8, layer_scale=0.5).scale.shape == (8,)


def test_step_sizes():
    """A step's sequences and heads are bounded each by itself: their product is no dimension of its grid."""
    lib = _lib.load()
    step = lambda B, H: lib.dynconv_delta_step(*([None] * 7), None, 0, None, B, B, H, 64, 64, 1.0, 0, None)  # noqa: E731
    assert step(2048, 33) == ARGUMENT and step(65535, 65535) == ARGUMENT  # (past the sizes: no tensors)
    assert step(65536, 1) == SHAPE and step(1, 65536) == SHAPE and step(1, 0) == SHAPE and step(-1, 2) == SHAPE


def test_sizes_whose_product_overflows():
    lib = _lib.load()
    for B, H in ((1 << 62, 4), (1 << 48, 1 << 16), (1 << 61, 8)):
        assert lib.dynconv_delta_fwd(*([None] * 9), 0, None, None, 0, B, 1, H, 64, 64, 1.0, 0, None) == SHAPE
        assert lib.dynconv_delta_kept_bytes(B, 1, H, 64, 64, 0) == 0


def test_float32_weights_flag():
    """Beside either type; what is no type stays none with it."""
    lib = _lib.load()
    for dtype, want in ((256, ARGUMENT), (257, ARGUMENT), (258, UNSUPPORTED), (512, UNSUPPORTED), (-256, UNSUPPORTED), (-1, UNSUPPORTED)):
        assert lib.dynconv_gated_norm_fwd(*([None] * 5), 1, 1, 64, 1e-6, 1.0, dtype, None) == want
        assert lib.dynconv_gated_norm_bwd(*([None] * 9), 0, 1, 1, 64, 1e-6, 1.0, dtype, None) == want
        assert lib.dynconv_residual_norm_fwd(*([None] * 4), 1.0, None, None, 1, 64, 1e-6, dtype, None) == want
        assert lib.dynconv_residual_norm_bwd(*([None] * 4), 1.0, *([None] * 7), 0, 1, 64, 1e-6, dtype, None) == want


def test_float32_gates_flag():
    lib = _lib.load()
    for dtype, want in ((256, ARGUMENT), (257, ARGUMENT), (258, UNSUPPORTED), (512, UNSUPPORTED), (-256, UNSUPPORTED)):
        assert lib.dynconv_delta_fwd(*([None] * 9), 0, None, None, 0, 1, 4, 2, 64, 64, 1.0, dtype, None) == want
        assert lib.dynconv_delta_bwd(*([None] * 5), 0, *([None] * 10), 0, 1, 4, 2, 64, 64, 1.0, dtype, None) == want
        assert lib.dynconv_delta_step(*([None] * 7), None, 0, None, 1, 1, 2, 64, 64, 1.0, dtype, None) == want
    # what the rule keeps and works in does not depend on the gates' type
    for dtype in (0, 1):
        assert lib.dynconv_delta_kept_bytes(1, 100, 2, 64, 64, dtype + 256) == lib.dynconv_delta_kept_bytes(1, 100, 2, 64, 64, dtype) > 0
        for back in (0, 1):
            assert lib.dynconv_delta_workspace_bytes(1, 100, 2, 64, 64, dtype + 256, back) == lib.dynconv_delta_workspace_bytes(1, 100, 2, 64, 64, dtype, back)
