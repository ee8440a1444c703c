"""The training and serving operators on the GPU: traced calls, modules around them, and the ends of the types'
ranges, against plain forms in 64 bits (operator_refs.py)."""

import math

import pytest
import torch

import operator_refs as ref
from test_gpu_operators import DTYPES, IDS, ffn_inputs, loss_inputs, no_device_errors, rnd  # noqa: F401

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------------------
# modules
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("fused", [True, False])
@pytest.mark.parametrize("name", ["w_gate", "w_up", "w_down"])
def test_mlp_with_an_adapter_in_inference(name, fused):
    """The projections that inference reads as weights (fused, or stacked into one) run as modules where they
    are more than that."""
    from mamba3_b200 import SwiGLU

    class Doubled(torch.nn.Linear):
        def forward(self, x):
            return 2 * super().forward(x)

    torch.manual_seed(0)
    mlp = SwiGLU(64, 128, fused=fused).cuda().bfloat16()
    old = getattr(mlp, name)
    new = Doubled(old.in_features, old.out_features, bias=False).cuda().bfloat16()
    new.load_state_dict(old.state_dict())
    setattr(mlp, name, new)
    x = rnd(5, 64, seed=1, dtype=torch.bfloat16)
    with torch.no_grad():
        y = mlp(x)
        g, u = mlp.w_gate(x).double(), mlp.w_up(x).double()
        a, w = g * torch.sigmoid(g) * u, mlp.w_down.weight.double() * (2.0 if name == "w_down" else 1.0)
        want = a @ w.t()
    # at most three roundings of the activation (silu, the product; fp32 sums) and two of the result
    ref.check(y, (want, 3 * 2.0 ** -8 * (a.abs() @ w.abs().t()) + 2 * 2.0 ** -8 * want.abs()), name)
