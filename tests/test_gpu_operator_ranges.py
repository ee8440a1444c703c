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


# ---------------------------------------------------------------------------
# traced calls
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("rows", [6, 40])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("grad", [True, False])
def test_loss_under_compile(rows, reduction, grad):
    from mamba3_b200 import linear_cross_entropy

    torch._dynamo.reset()
    h, w, t = loss_inputs(rows, 64, 333, torch.bfloat16, 0.2)
    leaves = [h.requires_grad_(grad), w.requires_grad_(grad)]
    call = lambda a, b: linear_cross_entropy(a, b, t, reduction=reduction)  # noqa: E731
    eager, got = call(*leaves), torch.compile(call, backend="aot_eager", fullgraph=True)(*leaves)
    assert torch.equal(got, eager)
    if grad:
        dl = rnd(rows, seed=9) if reduction == "none" else torch.tensor(0.5, device="cuda")
        for a, b in zip(torch.autograd.grad(got, leaves, dl), torch.autograd.grad(eager, leaves, dl)):
            assert torch.equal(a, b)


@pytest.mark.parametrize("rows", [6, 40])
@pytest.mark.parametrize("grad", [True, False])
def test_ffn_under_compile(rows, grad):
    torch._dynamo.reset()
    t = ffn_inputs(rows, 64, 72, torch.bfloat16, True, True)
    leaves = {k: v.requires_grad_(grad) for k, v in t.items()}
    from test_gpu_operators import ffn_call

    eager, got = ffn_call(leaves), torch.compile(ffn_call, backend="aot_eager", fullgraph=True)(leaves)
    assert torch.equal(got, eager)
    if grad:
        dout = rnd(rows, 64, seed=9, dtype=torch.bfloat16)
        vs = list(leaves.values())
        for a, b in zip(torch.autograd.grad(got, vs, dout), torch.autograd.grad(eager, vs, dout)):
            assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("rows", [6, 40])
def test_custom_ops_as_torch_checks_them(rows, dtype):
    """Schema, fake and traced forms of the four ops, with and without what the backward passes read."""
    ops, check = torch.ops.mamba3_b200, torch.library.opcheck
    t = ffn_inputs(rows, 40, 56, dtype, True, True)
    ins = [t[k] for k in ("x", "w_gate", "w_up", "w_down", "b_gate", "b_up", "b_down")]
    utils = ("test_schema", "test_faketensor")
    for save in (True, False):
        check(ops.gated_ffn_fwd.default, (*ins, t["residual"], 0.5, save), test_utils=utils)
    _, act, gu = ops.gated_ffn_fwd(*ins, t["residual"], 0.5, True)
    for want in ([True] * 7, [False, True] * 3 + [False]):
        check(ops.gated_ffn_bwd.default, (*ins, 0.5, act, gu, t["x"], want), test_utils=utils)
    h, w, tg = loss_inputs(rows, 40, 333, dtype)
    for reduction in ("mean", "sum", "none"):
        check(ops.linear_xent_fwd.default, (h, w, tg, -100, reduction), test_utils=utils)
        loss, saved = ops.linear_xent_fwd(h, w, tg, -100, reduction)
        for a, b in ((True, True), (True, False), (False, True)):
            check(ops.linear_xent_bwd.default, (rows, w, saved, torch.ones_like(loss), -100, reduction, a, b),
                  test_utils=utils)
