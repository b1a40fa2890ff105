"""GPU: the gated delta rule and the norms at sizes and layouts where other tests say little."""
from __future__ import annotations

import pytest
import torch

from dynamic_conv1d_b200 import check_device, gated_delta_rule_step
from test_gpu_gated_delta import BF16, F32, F32_TOL, STEP, check, inputs, recurrence, rel

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_step_of_more_heads_than_a_grid_dimension(dtype):
    """2048 sequences of 33 heads: 67584 states."""
    ts, S0, _, _ = inputs(2048, 1, 33, 8, 12, dtype, seed=1)
    ts, S = [t[:, 0] for t in ts], S0.clone()
    o = gated_delta_rule_step(*ts[:3], S, *ts[3:])
    ro, rS = recurrence(*(t[:, None].double() for t in ts), S0.double(), 8**-0.5)
    check_device(o)
    assert rel(o, ro[:, 0]) <= (2 * STEP if dtype == BF16 else F32_TOL) and rel(S, rS) <= F32_TOL


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("dk,dv", [(64, 16), (128, 16), (128, 32), (64, 48)])
def test_few_columns_of_many_chains(dtype, dk, dv):
    """Fewer slices of 16 columns than the teams that so many chains would have."""
    check(*inputs(4, 130, 50, dk, dv, dtype, seed=dv), states=dv != 32)
