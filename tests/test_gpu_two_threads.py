"""GPU: calls of one kernel in different launch shapes from two host threads at once, each on a stream of its own.
Both threads have to get what each gets alone.

The library's own calls are recorded once and then repeated back to back, since a whole Python call spends too little
of its time inside the library for two of them to meet there.  Each side is recorded on its own stream and nothing
is allocated afterwards, so the memory that its calls name stays theirs."""
from __future__ import annotations

import threading

import pytest
import torch

from dynamic_conv1d_b200 import _lib, check_device, decay_linear_attention, gated_delta_rule, lowrank_dynamic_convolution

pytestmark = pytest.mark.gpu


def rnd(*shape, seed, dtype=torch.float32):
    return torch.randn(*shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)).to(dtype)


def rule(B, H, seed, dtype):
    """Few heads: a team of warps to a CTA; many: four, with other stages."""
    T, d = 64, 128
    q, k = (torch.nn.functional.normalize(rnd(B, T, H, d, seed=seed + i), dim=-1).to(dtype) for i in range(2))
    g, beta = -rnd(B, T, H, seed=seed + 3, dtype=dtype).abs(), rnd(B, T, H, seed=seed + 4, dtype=dtype).sigmoid()
    return gated_delta_rule, [q, k, rnd(B, T, H, d, seed=seed + 2, dtype=dtype), g, beta]


def attention(d, seed):
    """Widths on the CUDA cores, whose shared memory goes by them."""
    decay = torch.full((3,), -0.1, device="cuda")
    return lambda *x: decay_linear_attention(*x, decay), [rnd(2, 40, 3, d, seed=seed + i) for i in range(3)]


def convolution(R, seed):
    return lowrank_dynamic_convolution, [rnd(2, 60, 64, seed=seed), rnd(2, 60, R, seed=seed + 1), rnd(R, 8 * 64, seed=seed + 2)]


PAIRS = {
    "rule_bf16": lambda: (rule(1, 1, 0, torch.bfloat16), rule(4, 16, 10, torch.bfloat16)),
    "rule_f32": lambda: (rule(1, 1, 0, torch.float32), rule(4, 16, 10, torch.float32)),
    "attention_f32": lambda: (attention(100, 0), attention(250, 10)),
    "convolution_f32": lambda: (convolution(32, 0), convolution(64, 10)),
}


class Recorder:
    """The library, keeping every launching call that is made through it."""

    def __init__(self, lib):
        self.lib, self.calls = lib, []

    def __getattr__(self, name):
        fn = getattr(self.lib, name)
        if name.endswith("_bytes") or name in ("dynconv_last_error", "dynconv_status_string"):
            return fn

        def call(*args):
            self.calls.append((name, fn, args))
            return fn(*args)

        return call


@pytest.mark.parametrize("name", PAIRS)
def test_two_threads(name, monkeypatch):
    lib = _lib.load()
    kept, recorded = [], []
    for f, args in PAIRS[name]():
        leaves = [t.requires_grad_() for t in args]
        up = torch.ones_like(f(*leaves))
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        recorder = Recorder(lib)
        monkeypatch.setattr(_lib, "load", lambda r=recorder: r)
        with torch.cuda.stream(stream):
            y = f(*leaves)
            results = [y.detach(), *torch.autograd.grad(y, leaves, up)]
        stream.synchronize()
        want = [t.clone() for t in results]  # (not on that stream, whose freed workspaces are written again)
        monkeypatch.setattr(_lib, "load", lambda: lib)
        assert len(recorder.calls) >= 2  # (forward and backward)
        recorded.append(recorder.calls)
        kept.append((leaves, up, y, results, want, stream))
    start, failed = threading.Barrier(2), []

    def run(i):
        torch.cuda.set_device(0)
        start.wait()
        for _ in range(2000):
            for what, fn, args in recorded[i]:
                status = fn(*args)
                if status:
                    failed.append((i, what, status, lib.dynconv_last_error()))
                    return

    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not failed, failed
    for _, _, _, results, want, _ in kept:
        assert all(torch.equal(a, b) for a, b in zip(results, want))
    check_device(kept[0][1])
