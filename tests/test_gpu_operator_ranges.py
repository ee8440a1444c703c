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


# ---------------------------------------------------------------------------
# fp16's range
# ---------------------------------------------------------------------------
def scaled(want, by, dtype):
    """(value, bound) of a result that is linear in a factor `by` (a power of two): the bound's own least step
    is one of the unscaled result, so the result's is added."""
    return want[0] * by, want[1] * by + ref.least(dtype)


@pytest.mark.parametrize("scale,size", [(2.0 ** -10, 1.0), (2.0 ** -18, 256.0), (2.0 ** 16, 2.0 ** -5), (1.0, 1.0)])
def test_fp16_loss_per_token_keeps_small_weights(scale, size):
    """The caller's mean over 1000 tokens (weights near 1e-3, or smaller) and a loss scaler's 65536: softmax times
    weight is 5e-8 and less, or its one-hot part past 65504, and the gradients are within fp16 all the same."""
    from mamba3_b200 import linear_cross_entropy

    n, d, v = 1000, 64, 20000
    h = ((rnd(n, d, seed=1) * 0.5 + 1.0) * size).half().requires_grad_(True)
    w = (rnd(v, d, seed=2) * 0.02 / max(size, 1.0) + 0.01).half().requires_grad_(True)
    t = torch.randint(0, v, (n,), device="cuda", generator=torch.Generator(device="cuda").manual_seed(3))
    t[::7] = -100
    dl = (1.0 + 0.5 * rnd(n, seed=4).tanh()) * scale
    dl[::14] = 2.0 ** 40 * scale  # of ignored tokens: no part in the range
    dl[3] = -dl[3]
    dh, dw = torch.autograd.grad(linear_cross_entropy(h, w, t, reduction="none"), (h, w), dl)
    want = ref.loss(h, w, t, reduction="none", dloss=dl / scale)
    ref.check(dh, scaled(want["hidden"], scale, torch.float16), "dhidden")
    ref.check(dw, scaled(want["weight"], scale, torch.float16), "dweight")


def test_fp16_loss_per_token_with_weights_that_are_no_numbers():
    """Zero weights alone; an infinite or NaN weight stays in its own token's row of the hidden gradient."""
    from mamba3_b200 import linear_cross_entropy

    h, w, t = loss_inputs(40, 64, 300, torch.float16)
    h.requires_grad_(True)
    y = linear_cross_entropy(h, w, t, reduction="none")
    dl = torch.zeros(40, device="cuda")
    dh, = torch.autograd.grad(y, h, dl, retain_graph=True)
    assert not dh.any()
    dl = rnd(40, seed=5) * 2.0 ** -12
    want = ref.loss(h, w, t, reduction="none", dloss=dl * 2.0 ** 12)
    want = scaled(want["hidden"], 2.0 ** -12, torch.float16)
    for bad in (math.inf, math.nan):
        dl[7] = bad
        dh, = torch.autograd.grad(y, h, dl, retain_graph=True)
        assert not torch.isfinite(dh[7]).any()
        keep = torch.arange(40, device="cuda") != 7
        ref.check(dh[keep], (want[0][keep], want[1][keep]), "the others")


@pytest.mark.parametrize("n,d,f", [(100, 64, 72), (300, 128, 264), (20, 40, 24)])
@pytest.mark.parametrize("scale", [1.0, 2.0 ** -5])
def test_fp16_ffn_keeps_small_output_gradients(n, d, f, scale):
    """Output gradients of a few of fp16's smallest steps (an unscaled mean loss): dg and du keep their 11 bits.  They
    are brought up until the largest output gradient, 4 steps here, is 2^-8: half a smallest step there, 2^-25,
    is 2^-15 of the steps that the plain form below counts in, in each of dg and du."""
    from test_gpu_operators import ffn_call, ffn_want

    t = ffn_inputs(n, d, f, torch.float16, True, False)
    t["x"] = t["x"].abs()
    for v in t.values():
        v.requires_grad_(True)
    steps = torch.randint(-4, 5, (n, d), device="cuda", generator=torch.Generator(device="cuda").manual_seed(8))
    dout = (steps.double() * 2.0 ** -24).half()
    grads = torch.autograd.grad(ffn_call(t, scale), list(t.values()), dout)
    want = ffn_want(t, scale, (steps.double() / scale).half())  # the largest near 1 after the factor
    x, wg, wu = (t[k].detach().double().abs() for k in ("x", "w_gate", "w_up"))
    least = {"x": (wg.sum(0) + wu.sum(0)).expand(n, d), "w_gate": x.sum(0).expand(f, d), "w_up": x.sum(0).expand(f, d),
             "b_gate": torch.full((f,), float(n), device="cuda"), "b_up": torch.full((f,), float(n), device="cuda")}
    for k, g in zip(t, grads):
        value, bound = want[k]
        ref.check(g, scaled((value, bound + 2.0 ** -15 * least.get(k, 0)), 2.0 ** -24 * scale, torch.float16), f"d{k}")


def test_fp16_ffn_output_gradients_at_their_ends():
    """All zero, and one that is not finite: its row's gradients alone (and the sums over rows) are no numbers."""
    from test_gpu_operators import ffn_call, ffn_want

    t = ffn_inputs(30, 64, 72, torch.float16, False, False)
    x = t["x"].requires_grad_(True)
    y = ffn_call(t)
    g, = torch.autograd.grad(y, x, torch.zeros_like(y), retain_graph=True)
    assert not g.any()
    steps = torch.randint(-4, 5, (30, 64), device="cuda", generator=torch.Generator(device="cuda").manual_seed(8))
    value, bound = ffn_want(t, 1.0, steps.half())["x"]
    both = (t["w_gate"].double().abs() + t["w_up"].double().abs()).sum(0)  # 2^-15 of dg and du, as above
    want = scaled((value, bound + 2.0 ** -15 * both), 2.0 ** -24, torch.float16)
    for bad in (math.inf, math.nan):
        dout = (steps.double() * 2.0 ** -24).half()
        dout[11, 5] = bad
        g, = torch.autograd.grad(y, x, dout, retain_graph=True)
        keep = torch.arange(30, device="cuda") != 11
        assert not torch.isfinite(g[11]).any()
        ref.check(g[keep], (want[0][keep], want[1][keep]), "the others")


@pytest.mark.parametrize("d,width", [(13, 13), (13, 16), (24, 24), (21, 40), (5, 8), (264, 264)])
def test_fp16_ffn_finds_the_largest_output_gradient(d, width):
    """Small output gradients but for one of 100 in the last column of a row: a factor for the small ones alone would
    make its row infinite."""
    from test_gpu_operators import ffn_call, ffn_want

    n, f = 70, 40
    t = ffn_inputs(n, d, f, torch.float16, False, False)
    for v in t.values():
        v.requires_grad_(True)
    buf = torch.full((n, width), 7.0, device="cuda", dtype=torch.float16)  # what lies between the rows has no part
    buf[:, :d] = rnd(n, d, seed=3) * 2.0 ** -18
    buf[n - 1, d - 1] = 100.0
    dout = buf[:, :d]
    grads = torch.autograd.grad(ffn_call(t), list(t.values()), dout)
    want = ffn_want(t, 1.0, dout)
    for k, g in zip(t, grads):
        ref.check(g, want[k], f"d{k}")


# ---------------------------------------------------------------------------
# large logits
# ---------------------------------------------------------------------------
def ladder(n, v, d, top, gap, dtype):
    """Hidden states and weights whose logits are exact: `top` at column i % v of row i, top - gap elsewhere
    (products of powers of two in two columns)."""
    h, w = torch.zeros(n, d, device="cuda"), torch.zeros(v, d, device="cuda")
    i = torch.arange(n, device="cuda") % v
    w[:, 0] = 1.0
    h[:, 0] = top - gap
    at = 1 + i % (d - 1)
    h[torch.arange(n, device="cuda"), at] = gap
    w[torch.arange(1, d, device="cuda") - 1, torch.arange(1, d, device="cuda")] = 1.0
    return h.to(dtype), w.to(dtype), at - 1


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("n", [4, 40, 300])
@pytest.mark.parametrize("top,gap", [(128.0, 16.0), (4096.0, 16.0), (16384.0, 128.0), (-4096.0, 32.0)])
def test_sure_tokens_with_large_logits(n, top, gap, dtype):
    """One logit `gap` above 399 equal ones: loss log(1 + 399 e^-gap) for it and gap more for another, whatever the
    logits' size; never below zero.  Each term that is added to the 1 of the largest is rounded to 2^-24 of it: at
    most 48 of them (128 columns a thread, a quarter of them one after the other, and the joins), its logarithm and
    the loss to half a step each; the exponentials' 2 steps and the exponent's rounding (2^-24 of up to 185) weigh
    e^-gap."""
    from mamba3_b200 import linear_cross_entropy

    v, d = 400, 64
    h, w, best = ladder(n, v, d, top, gap, dtype)
    z = h.double() @ w.double().t()
    assert bool((z.amax(1) == top).all()) and bool((z.sort(1)[0][:, -2] == top - gap).all())
    rest = 399 * math.exp(-gap)
    want = math.log1p(rest)
    err = 48 * 2.0 ** -24 + (3 * 2.0 ** -23 + 185 * 2.0 ** -24) * rest
    y = linear_cross_entropy(h, w, best, reduction="none")
    assert bool((y >= 0).all()) and bool(((y.double() - want).abs() <= err + 2.0 ** -23 * want).all())
    y = linear_cross_entropy(h, w, best + 100, reduction="none")
    assert bool(((y.double() - want - gap).abs() <= err + 2.0 ** -23 * (want + gap)).all())


@pytest.mark.parametrize("n", [4, 40, 300])
def test_probabilities_of_large_logits_sum_to_one(n):
    """fp32, logits of 4096 and more and 399 others up to 2 below: the sum over the vocabulary of softmax - onehot, read off a
    weight column of ones, is 0.  Each probability is off by its exponent's roundings (2^-24 of up to 3, and of the
    sum's logarithm, up to 9 in powers of two), the hardware exponential (2^-22) and what its sum had (16 steps);
    the product's sum adds sum_error: 64 steps of 2^-23 of the 2 that all magnitudes sum to."""
    from mamba3_b200 import linear_cross_entropy

    v, d = 400, 16
    h, w = torch.zeros(n, d, device="cuda"), torch.zeros(v, d, device="cuda")
    h[:, 0], h[:, 1] = 4096.0 + torch.arange(n, device="cuda"), 1.0
    w[:, 0], w[:, 1] = 1.0, -torch.arange(v, device="cuda") / 256.0
    w[:, 2] = 1.0  # times 0 in the logits
    h.requires_grad_(True)
    t = torch.full((n,), 399, device="cuda")
    dh, = torch.autograd.grad(linear_cross_entropy(h, w, t, reduction="sum"), h)
    assert bool((dh[:, 2].abs() <= 64 * 2.0 ** -23 * 2).all()), float(dh[:, 2].abs().max())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("n", [4, 40, 300])
def test_loss_of_very_negative_logits(n, dtype):
    """Rows whose logits all lie near -1e35: differences of 1e32 and more, so the loss is that to the best one."""
    from mamba3_b200 import linear_cross_entropy

    v, d = 300, 64
    h, w = torch.zeros(n, d, device="cuda", dtype=dtype), torch.zeros(v, d, device="cuda", dtype=dtype)
    h[:, 0] = 2.0 ** 60
    w[:, 0] = -(2.0 ** 56) * (1 + (torch.arange(v, device="cuda") % 100 + 1) / 128.0)
    w[7, 0] = -(2.0 ** 56)
    z = h.double() @ w.double().t()
    for t in (torch.full((n,), 7, device="cuda"), torch.arange(n, device="cuda") % v):
        want = z.amax(1) - z[torch.arange(n, device="cuda"), t]
        a = h.clone().requires_grad_(True)
        y = linear_cross_entropy(a, w, t, reduction="none")
        assert bool(((y.double() - want).abs() <= 2.0 ** -23 * z.abs().amax(1) * (want > 0)).all())
        g, = torch.autograd.grad(y.sum(), a)
        assert bool(torch.isfinite(g).all())


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("n", [6, 40, 300])
def test_loss_of_infinite_logits(n, dtype):
    """Vocabulary rows of -infinity leave the others as they are; a token all of whose logits are, or one of
    +infinity, has no loss."""
    from mamba3_b200 import linear_cross_entropy

    h, w, t = loss_inputs(n, 64, 300, dtype)
    a, b = h.abs() + 0.5, w.clone()
    b[7], b[150] = float("-inf"), float("-inf")
    t[(t == 7) | (t == 150)] = 8
    keep = torch.ones(300, dtype=torch.bool, device="cuda")
    keep[7] = keep[150] = False
    want = ref.loss(a, b[keep], t - (t > 7).long() - (t > 150).long(), reduction="sum", dloss=1.0)
    b.requires_grad_(True)
    y = linear_cross_entropy(a, b, t, reduction="sum")
    ref.check(y, want["loss"], "loss")
    dw, = torch.autograd.grad(y, b)
    assert not dw[~keep].any()
    ref.check(dw[keep], want["weight"], "dweight")
    t[0] = 7
    assert linear_cross_entropy(a, b, t, reduction="none")[0].item() == math.inf
    for x in (math.inf, -math.inf):
        assert torch.isnan(linear_cross_entropy(a, torch.full_like(w, x), t, reduction="none")).all()
        c = w.clone()
        c[9] = x
        y = linear_cross_entropy(a, c, t, reduction="none")
        assert bool(torch.isnan(y).all() if x > 0 else torch.isfinite(y[t != 9]).all())


# ---------------------------------------------------------------------------
# fp32 operands
# ---------------------------------------------------------------------------
def test_fp32_products_of_one_sign():
    """Sums of sixteen equal products of values with all 24 bits set, in every remainder's sign: no error averages
    out.  Two steps for the last sum of sixteen products (in two halves; the passes before it are 2^-8 of it and less),
    half a step for the loss's own rounding, and 2^-24 for the plane pairs that are left out.  The loss of two logits z > 16 and 0 is z for the second
    to within e^-16."""
    from mamba3_b200 import linear_cross_entropy

    n = 600
    v = 1.0 + torch.rand(n, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)) * 0.99
    v[:6] = torch.tensor([1 + 2.0 ** -7 - 2.0 ** -23, 1 + 2.0 ** -7 - 2.0 ** -15 - 2.0 ** -23, 2 - 2.0 ** -23,
                          1 + 2.0 ** -8, 1 + 2.0 ** -8 - 2.0 ** -23, 1.0], device="cuda")
    h = v[:, None].expand(n, 16).contiguous()
    t = torch.ones(n, dtype=torch.long, device="cuda")
    for c in (1 + 2.0 ** -7 - 2.0 ** -23, 2 - 2.0 ** -23, 1 + 2.0 ** -8 - 2.0 ** -16 + 2.0 ** -23, 1.0):
        w = torch.zeros(2, 16, device="cuda")
        w[0] = c
        y = linear_cross_entropy(h, w, t, reduction="none").double()
        z = 16 * v.double() * float(w[0, 0])
        want = z + torch.log1p(torch.exp(-z))
        bound = 3 * 2.0 ** -23 * want
        off = (y - want).abs()
        assert bool((off <= bound).all()), (c, float((off / want).max()))


@pytest.mark.parametrize("n", [6, 40, 300])
def test_fp32_infinities_are_those_of_the_sums(n):
    """Infinite inputs of the fp32 feed-forward: as in plain fp32 arithmetic, infinite where one sign meets
    finite values that are not zero, and nothing else touched."""
    from mamba3_b200 import gated_ffn

    d, f = 64, 72
    x, w = rnd(n, d, seed=1).abs() + 0.5, rnd(f, d, seed=2).abs() * d ** -0.5 + 0.01
    wd = rnd(d, f, seed=3).abs() * f ** -0.5 + 0.01
    wd[5] = -wd[5]
    x[2, 3] = math.inf
    y = gated_ffn(x, w, w, wd)
    rows = torch.arange(n, device="cuda") != 2
    assert torch.isfinite(y[rows]).all()
    assert bool((y[2][torch.arange(d, device="cuda") != 5] == math.inf).all()) and y[2, 5].item() == -math.inf
    x[2, 3] = math.nan
    y = gated_ffn(x, w, w, wd)
    assert torch.isfinite(y[rows]).all() and torch.isnan(y[2]).all()


# ---------------------------------------------------------------------------
# long sums of 16-bit operands
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DTYPES[:2], ids=IDS[:2])
@pytest.mark.parametrize("n", [40, 300])
@pytest.mark.parametrize("k", [1024, 4096, 8192, 8200])
def test_loss_of_long_sums_of_one_sign(k, n, dtype):
    """The tensor core cuts off each sum of sixteen products (perhaps in two halves), always downwards where all are
    positive: at most two steps of 2^-23 of the sum so far, half of the whole on average over the 64 of a group
    of 1024: 65 steps.  The groups' sums and the loss's own rounding, five.  The loss of two logits z and 0 is z for the
    second."""
    from mamba3_b200 import linear_cross_entropy

    h = 1.0 + torch.rand(n, k, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    w = torch.zeros(2, k, device="cuda")
    w[0] = (1.0 + torch.rand(k, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2))) / 16
    h, w = h.to(dtype), w.to(dtype)
    t = torch.ones(n, dtype=torch.long, device="cuda")
    z = h.double() @ w[0].double()
    y = linear_cross_entropy(h, w, t, reduction="none").double()
    assert bool(((y - z).abs() <= 70 * 2.0 ** -23 * z).all()), float(((y - z).abs() / z).max())


@pytest.mark.parametrize("dtype", DTYPES[:2], ids=IDS[:2])
@pytest.mark.parametrize("n", [40, 300])
def test_gradient_of_sure_tokens_uses_the_loss_s_logits(n, dtype):
    """d_model 4096: exp(loss) is 1 / p of the target, and the gradient along a weight column of ones that no logit
    reads is 0: the backward pass makes the same logits as the forward pass, or the probabilities' sum would be off by
    the cut-off sums' bias.  399 other logits about 8 below: dz is rounded to 16 bits (2^-8, 2^-11 of each), the sums
    to 2^-18 of all magnitudes; the gradient of the target's own column is p - 1 within the same."""
    from mamba3_b200 import linear_cross_entropy

    v, d = 400, 4096
    g = torch.Generator(device="cuda").manual_seed(3)
    h = (1.0 + torch.rand(n, d, device="cuda", generator=g)) / 32
    w = (torch.rand(v, d, device="cuda", generator=g) * 0.5 + 0.5) * 0.1
    w[5] = w[5] + 0.04
    h[:, 0] = 0.0
    w[:, 0] = 1.0
    h, w = h.to(dtype).requires_grad_(True), w.to(dtype)
    t = torch.full((n,), 5, device="cuda")
    y = linear_cross_entropy(h, w, t, reduction="none")
    p = torch.softmax(h.detach().double() @ w.double().t(), 1)
    rest = 1.0 - p[:, 5]
    dh, = torch.autograd.grad(y.sum(), h)
    assert bool((rest < 0.5).all()) and bool((rest > 1e-6).all())
    bound = 2 * rest * (2 * ref.half_step(dtype) + 2.0 ** -18) + 2 * 2.0 ** -22 + ref.least(dtype)
    assert bool((dh[:, 0].double().abs() <= bound).all()), float((dh[:, 0].double().abs() / bound).max())


# ---------------------------------------------------------------------------
# sums over the rows
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("n", [1, 20, 33, 300])
@pytest.mark.parametrize("frozen", [(), ("b_gate",), ("b_up",), ("b_down",)])
def test_bias_gradients_are_sums_of_what_is_not_rounded(n, frozen, dtype):
    """Inputs whose products are exact in any type (steps of 2^-5, sums of 16): the bias gradients are then off by their
    one rounding and 2^-18 of the summands' magnitudes (the hardware's exponential and reciprocal, a few steps of
    2^-22 each, and the fp32 sums)."""
    from mamba3_b200 import gated_ffn

    d, f = 16, 200
    g = torch.Generator(device="cuda").manual_seed(n)
    ints = lambda *s, top: torch.randint(-top, top + 1, s, device="cuda", generator=g).to(dtype)  # noqa: E731
    t = {"x": ints(n, d, top=1), "w_gate": ints(f, d, top=7) / 32, "w_up": ints(f, d, top=7) / 32,
         "w_down": ints(d, f, top=7) / 32, "b_gate": ints(f, top=7) / 32, "b_up": ints(f, top=7) / 32,
         "b_down": ints(d, top=7) / 32}
    for k, v in t.items():
        v.requires_grad_(k not in frozen)
    y = gated_ffn(t["x"], t["w_gate"], t["w_up"], t["w_down"], b_gate=t["b_gate"], b_up=t["b_up"], b_down=t["b_down"])
    dout = ints(n, d, top=3) / 4
    names = [k for k in ("b_gate", "b_up", "b_down") if k not in frozen]
    grads = torch.autograd.grad(y, [t[k] for k in names], dout)
    q = {k: v.detach().double() for k, v in t.items()}
    a, b, da = q["x"] @ q["w_gate"].t() + q["b_gate"], q["x"] @ q["w_up"].t() + q["b_up"], dout.double() @ q["w_down"]
    s = torch.sigmoid(a)
    terms = {"b_gate": da * b * s * (1 + a * (1 - s)), "b_up": da * a * s, "b_down": dout.double()}
    for k, got in zip(names, grads):
        want = terms[k].sum(0)
        ref.check(got, (want, ref.rounded(want, 2.0 ** -18 * terms[k].abs().sum(0), dtype)), k)


# ---------------------------------------------------------------------------
# captured, and from several threads
# ---------------------------------------------------------------------------
def captured(step):
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    return graph, out


@pytest.mark.parametrize("d", [64, 2000])
def test_fp16_steps_captured_follow_their_gradients_range(d):
    """The factors of the fp16 backward passes are made on the device: a replay with output gradients and weights of
    another size gives the eager call's values."""
    from mamba3_b200 import gated_ffn, linear_cross_entropy

    n, f, v = 70, 72, 500
    t = ffn_inputs(n, d, f, torch.float16, True, False)
    h, w, tg = loss_inputs(n, d, v, torch.float16, 0.2)
    leaves = [q.requires_grad_(True) for q in (*t.values(), h, w)]
    dout, dl = torch.zeros(n, d, device="cuda", dtype=torch.float16), torch.zeros(n, device="cuda")

    def step():
        y = gated_ffn(*leaves[:4], b_gate=leaves[4], b_up=leaves[5], b_down=leaves[6])
        loss = linear_cross_entropy(leaves[7], leaves[8], tg, reduction="none")
        return (y.detach(), loss.detach(), *torch.autograd.grad((y, loss), leaves, (dout, dl)))

    graph, got = captured(step)
    for seed, scale in ((1, 1.0), (2, 2.0 ** -18), (3, 0.0), (4, 2.0 ** 6)):
        dout.copy_(rnd(n, d, seed=seed) * scale)
        dl.copy_(rnd(n, seed=seed + 9) * scale)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, step()):
            assert torch.equal(a, b) and bool(torch.isfinite(a).all())


def test_calls_from_several_threads_on_one_stream():
    """Each thread's workspaces are its own until its kernels are launched: all get the values of a call alone."""
    import threading

    from mamba3_b200 import clip_grads, gated_ffn, linear_cross_entropy

    jobs = []
    for i, (n, d, f, v, dtype) in enumerate([(40, 130, 72, 333, torch.float32), (300, 65, 130, 777, torch.bfloat16),
                                             (9, 33, 40, 1000, torch.float16), (5, 64, 72, 2000, torch.bfloat16)]):
        t = ffn_inputs(n, d, f, dtype, True, True, seed=10 * i)
        h, w, tg = loss_inputs(n, d, v, dtype, 0.1, seed=10 * i)
        tg[0] = 1
        jobs.append(([q.requires_grad_(True) for q in (*t.values(), h, w)], tg))

    def step(leaves, tg):
        y = gated_ffn(*leaves[:4], b_gate=leaves[4], b_up=leaves[5], b_down=leaves[6], residual=leaves[7])
        loss = linear_cross_entropy(leaves[8], leaves[9], tg)
        grads = torch.autograd.grad(y.float().square().sum() + loss, leaves)
        outs = [torch.empty_like(g) for g in grads]
        return [y.detach(), loss.detach(), *grads, clip_grads(grads, 0.1, out=outs), *outs]

    want = [step(*j) for j in jobs]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        try:
            for _ in range(30):
                got = step(*jobs[i])
                wrong.extend((i, k) for k, (a, b) in enumerate(zip(got, want[i])) if not torch.equal(a, b))
        except Exception as e:  # noqa: BLE001 - reported by the test
            wrong.append((i, e))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(jobs))]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not wrong, wrong[:5]


@pytest.mark.parametrize("ckpt", [False, True])
@pytest.mark.parametrize("cast", [None, torch.bfloat16, torch.float16])
def test_lm_without_logits_under_autocast_and_checkpointing(cast, ckpt):
    from mamba3_b200 import KulaMambaLM

    torch.manual_seed(0)
    lm = KulaMambaLM(vocab_size=203, d_model=64, n_layers=2, d_state=16, headdim=16, fused_mlp=True,
                     gradient_checkpointing=ckpt).cuda().train()
    ids = torch.randint(0, 203, (2, 40), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    losses, grads = [], []
    for logits in (True, False):
        lm.zero_grad()
        with torch.autocast("cuda", cast or torch.bfloat16, enabled=cast is not None):
            loss = lm(ids, ids, return_logits=logits)["loss"]
        loss.backward()
        losses.append(loss.detach())
        grads.append([p.grad.clone() for p in lm.parameters()])
    torch.testing.assert_close(losses[1].float(), losses[0].float(), rtol=2e-3, atol=0)
    for a, b in zip(*grads):
        assert b.dtype == torch.float32 and (a - b).norm() <= 3e-2 * a.norm()


def test_loss_of_small_integer_targets_and_expanded_weights():
    """int8 and uint8 targets, an expanded incoming gradient, one row of hidden states for every token."""
    from mamba3_b200 import linear_cross_entropy

    h, w, t = loss_inputs(60, 64, 100, torch.bfloat16)
    want = ref.loss(h, w, t, reduction="none", dloss=torch.full((60,), 0.5, device="cuda"))
    for dt in (torch.int8, torch.uint8):
        a = h.clone().requires_grad_(True)
        y = linear_cross_entropy(a, w, t.to(dt), reduction="none")
        ref.check(y, want["loss"], str(dt))
        g, = torch.autograd.grad(y, a, torch.tensor(0.5, device="cuda").expand(60))
        ref.check(g, want["hidden"], str(dt))
    row = h[:1].clone().requires_grad_(True)
    g, = torch.autograd.grad(linear_cross_entropy(row.expand(60, 64), w, t, reduction="sum"), row)
    same = ref.loss(h[:1].expand(60, 64), w, t, reduction="sum", dloss=1.0)["hidden"]
    ref.check(g, (same[0].sum(0, keepdim=True), same[1].sum(0, keepdim=True) * 2 + 60 * 2.0 ** -8 * same[0].abs().sum(0, keepdim=True)), "one row")
