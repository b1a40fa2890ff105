"""CPU: which calls the operators hand to autograd although no input asks for a gradient."""
from __future__ import annotations

import torch
from torch.autograd import forward_ad

from dynamic_conv1d_b200 import _lib


def test_watched():
    seen = []

    def f(x):
        seen.append(_lib.watched())
        return 2 * x

    x = torch.ones(3)
    f(x)
    with torch.no_grad():
        f(x)
    with torch.inference_mode():
        f(x)
    assert seen == [False] * 3
    with forward_ad.dual_level():
        f(x)
        with torch.no_grad():
            f(x)
    torch.func.jvp(f, (x,), (x,))
    torch.jit.trace(f, (x,), check_trace=False)
    assert seen[3:] == [True] * 4
    f(x)
    assert not seen[-1]
