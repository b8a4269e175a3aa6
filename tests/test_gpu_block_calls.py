"""Calls of the block's operators that their documentation allows and the formulas' cases
do not make, against the formulas in 64 bits.  Bounds as in ``test_gpu_block``."""

import pytest
import torch

from multics_amd import kernels
from tests.gpu_util import need_gpu, say
from tests.test_gpu_block import BF16, FP16, _linear_case

pytestmark = pytest.mark.gpu


# ---- values that are not numbers --------------------------------------------------------

@pytest.mark.parametrize("t,N", [(BF16, 264), (FP16, 264), (BF16, 77)])
@pytest.mark.parametrize("act", ["gelu_tanh", "gelu", "silu"])
def test_gradient_of_a_nan_before_the_activation(act, t, N):
    """It reaches the gradients of its row and its channel, and no others."""
    need_gpu()
    M, K = 150, 64
    x, w, b, _, gate, dy = _linear_case(M, K, N, act, 3, False, t)
    z = (x.float() @ w.float().t() + b.float()).to(t)
    say("a NaN before the activation", act, t, N)
    clean = kernels.linear_act_backward(dy, x, w, preact=z, activation=act, gate=gate)
    z[70, 5] = float("nan")
    got = kernels.linear_act_backward(dy, x, w, preact=z, activation=act, gate=gate)
    rows = torch.arange(M, device="cuda") != 70
    cols = torch.arange(N, device="cuda") != 5
    assert torch.isnan(got["x"][70]).all() and torch.equal(got["x"][rows], clean["x"][rows])
    assert torch.isnan(got["weight"][5]).all() and torch.equal(got["weight"][cols], clean["weight"][cols])
    assert torch.isnan(got["bias"][5]) and torch.equal(got["bias"][cols], clean["bias"][cols])
    assert torch.isnan(got["gate"][1, 5])                    # (50 rows a gate)
    got["gate"][1, 5] = clean["gate"][1, 5]
    assert torch.equal(got["gate"], clean["gate"])
