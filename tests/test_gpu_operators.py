"""The training and serving operators on the GPU: gated feed-forward, the head's cross entropy and gradient
clipping, against plain forms in 64 bits with derived bounds (operator_refs.py)."""

import math

import pytest
import torch

import operator_refs as ref

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]
IDS = ["bf16", "fp16", "fp32"]


def rnd(*shape, seed, std=1.0, dtype=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, device="cuda", generator=g) * std).to(dtype)


@pytest.fixture(autouse=True)
def no_device_errors():
    from mamba3_b200 import check_device_errors

    yield
    torch.cuda.synchronize()
    check_device_errors()


# ---------------------------------------------------------------------------
# gated feed-forward
# ---------------------------------------------------------------------------
def ffn_inputs(n, d, f, dtype, bias, residual, seed=0):
    t = {"x": rnd(n, d, seed=seed + 1, dtype=dtype), "w_gate": rnd(f, d, seed=seed + 2, std=d ** -0.5, dtype=dtype),
         "w_up": rnd(f, d, seed=seed + 3, std=d ** -0.5, dtype=dtype),
         "w_down": rnd(d, f, seed=seed + 4, std=f ** -0.5, dtype=dtype)}
    if bias:
        t.update(b_gate=rnd(f, seed=seed + 5, std=0.3, dtype=dtype), b_up=rnd(f, seed=seed + 6, std=0.3, dtype=dtype),
                 b_down=rnd(d, seed=seed + 7, std=0.3, dtype=dtype))
    if residual:
        t["residual"] = rnd(n, d, seed=seed + 8, dtype=dtype)
    return t


def ffn_call(t, scale=1.0):
    from mamba3_b200 import gated_ffn

    kw = {k: v for k, v in t.items() if k not in ("x", "w_gate", "w_up", "w_down")}
    return gated_ffn(t["x"], t["w_gate"], t["w_up"], t["w_down"], residual_scale=scale, **kw)


def ffn_want(t, scale=1.0, dout=None):
    return ref.ffn(t["x"], t["w_gate"], t["w_up"], t["w_down"], t.get("b_gate"), t.get("b_up"), t.get("b_down"),
                   t.get("residual"), scale, dout)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("n,d,f", [(1, 64, 64), (1, 768, 2112), (2, 40, 24), (5, 320, 896), (8, 256, 512),
                                   (9, 128, 136), (17, 768, 2112), (31, 33, 65), (64, 200, 328), (100, 96, 100),
                                   (128, 128, 128), (129, 72, 40), (256, 768, 2112), (257, 130, 258), (300, 1, 1),
                                   (513, 264, 520), (1025, 512, 1032)])
def test_ffn_forward(n, d, f, dtype):
    t = ffn_inputs(n, d, f, dtype, bias=(n + d) % 2 == 0, residual=n % 3 != 0)
    ref.check(ffn_call(t, 0.3), ffn_want(t, 0.3)["out"], "out")


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("n,d,f,bias,residual", [(1, 64, 64, True, True), (2, 48, 40, False, False),
                                                 (7, 323, 97, True, True), (64, 128, 256, False, True),
                                                 (129, 72, 40, True, False), (256, 264, 136, True, True),
                                                 (300, 768, 2112, False, True), (777, 65, 130, True, True),
                                                 (2050, 128, 320, True, True)])
def test_ffn_gradients(n, d, f, bias, residual, dtype):
    t = ffn_inputs(n, d, f, dtype, bias, residual)
    leaves = {k: v.requires_grad_(True) for k, v in t.items()}
    y = ffn_call(t, 0.7)
    dout = rnd(n, d, seed=77, dtype=dtype)
    grads = torch.autograd.grad(y, list(leaves.values()), dout)
    want = ffn_want(t, 0.7, dout)
    ref.check(y, want["out"], "out")
    for k, g in zip(leaves, grads):
        ref.check(g, want[k], f"d{k}")


def test_ffn_gradients_against_differences():
    """Directional derivatives in fp32 from the operator's own outputs: (L(p + h v) - L(p - h v)) / 2h.
    With values of order 1, h = 2^-6 leaves a truncation error of order h^2 = 2.4e-4 of the derivative's scale
    and a rounding error of order 2^-20 / h; 1 % of |v| |dL/dp| / sqrt(numel) stays well above both."""
    t = ffn_inputs(40, 48, 56, torch.float32, True, True)
    for v in t.values():
        v.requires_grad_(True)
    w = rnd(40, 48, seed=5)
    grads = torch.autograd.grad((ffn_call(t, 0.5) * w).sum(), list(t.values()))
    for i, (k, p) in enumerate(t.items()):
        v = rnd(*p.shape, seed=100 + i, std=p.numel() ** -0.5)
        h = 2.0 ** -6
        with torch.no_grad():
            up = (ffn_call({**t, k: p + h * v}, 0.5).double() * w).sum()
            dn = (ffn_call({**t, k: p - h * v}, 0.5).double() * w).sum()
        slope, want = float((up - dn) / (2 * h)), float((grads[i].double() * v).sum())
        assert abs(slope - want) < 0.01 * float(grads[i].double().norm()), (k, slope, want)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_ffn_strides_and_shapes(dtype):
    """Rows inside a wider buffer (aligned and not), a transposed input and weights, 3-d inputs, an
    expanded incoming gradient."""
    from mamba3_b200 import gated_ffn

    d, f, n = 64, 72, 50
    t = ffn_inputs(n, d, f, dtype, False, True)
    want = ffn_want(t)["out"]
    for off, width in ((0, 96), (8, 100), (3, 101)):
        buf = torch.zeros(n, width, device="cuda", dtype=dtype)
        buf[:, off:off + d] = t["x"]
        res = torch.zeros(n, width, device="cuda", dtype=dtype)
        res[:, off:off + d] = t["residual"]
        s = dict(t, x=buf[:, off:off + d], residual=res[:, off:off + d])
        ref.check(ffn_call(s), want, f"rows at {off} of {width}")
    s = dict(t, x=t["x"].t().contiguous().t(), w_gate=t["w_gate"].t().contiguous().t(),
             w_down=t["w_down"].t().contiguous().t())
    ref.check(ffn_call(s), want, "transposed")
    y = gated_ffn(t["x"].view(5, 10, d), t["w_gate"], t["w_up"], t["w_down"], residual=t["residual"].view(5, 10, d))
    assert y.shape == (5, 10, d)
    ref.check(y.view(n, d), want, "3-d")
    x = t["x"].clone().requires_grad_(True)
    y = gated_ffn(x, t["w_gate"], t["w_up"], t["w_down"])
    y.sum().backward()  # the incoming gradient has stride 0
    ref.check(x.grad, ffn_want({k: v for k, v in t.items() if k != "residual"},
                               dout=torch.ones(n, d, device="cuda", dtype=dtype))["x"], "expanded gradient")
    x1 = gated_ffn(t["x"][7], t["w_gate"], t["w_up"], t["w_down"])
    assert x1.shape == (d,)


def test_ffn_empty_and_partial_gradients():
    from mamba3_b200 import gated_ffn

    t = ffn_inputs(6, 32, 48, torch.bfloat16, False, False)
    e = gated_ffn(t["x"][:0], t["w_gate"], t["w_up"], t["w_down"])
    assert e.shape == (0, 32)
    w = t["w_up"].clone().requires_grad_(True)
    g, = torch.autograd.grad(gated_ffn(t["x"][:0], t["w_gate"], w, t["w_down"]).sum(), w)
    assert g.shape == w.shape and not g.any()
    want = ffn_want(t, dout=torch.ones(6, 32, device="cuda", dtype=torch.bfloat16))
    for k in t:
        s = {j: v.clone().requires_grad_(j == k) for j, v in t.items()}
        ffn_call(s).sum().backward()
        ref.check(s[k].grad, want[k], k)
        assert all(s[j].grad is None for j in t if j != k)


def test_ffn_values_at_the_ends():
    """Large gates of both signs (the exponential over- and underflows) and values that are not finite."""
    from mamba3_b200 import gated_ffn

    d = f = 64
    x = torch.zeros(5, d, device="cuda", dtype=torch.bfloat16)
    x[0, 0], x[1, 0], x[2, 0], x[3, 0], x[4, 0] = 300.0, -300.0, float("nan"), float("inf"), 0.0
    eye = torch.eye(f, d, device="cuda", dtype=torch.bfloat16)
    y = gated_ffn(x, eye, eye, eye)
    assert y[0, 0].item() == 90112.0  # 300^2 in bf16
    assert y[1, 0].item() == 0.0 and y[4, 0].item() == 0.0
    assert torch.isnan(y[2]).any() and not torch.isfinite(y[3]).all()
    assert torch.isfinite(y[[0, 1, 4]]).all()  # rows do not mix


def test_ffn_autocast_and_masters():
    from mamba3_b200 import gated_ffn

    t = ffn_inputs(20, 64, 72, torch.float32, False, True)
    for v in t.values():
        v.requires_grad_(True)
    with torch.autocast("cuda", torch.bfloat16):
        y = ffn_call(t)
    assert y.dtype == torch.bfloat16
    y.float().sum().backward()
    assert all(v.grad.dtype == torch.float32 for v in t.values())
    low = {k: v.detach().bfloat16() for k, v in t.items()}
    assert torch.equal(y, gated_ffn(low["x"], low["w_gate"], low["w_up"], low["w_down"], residual=low["residual"]))


# ---------------------------------------------------------------------------
# cross entropy of the head
# ---------------------------------------------------------------------------
def loss_inputs(n, d, v, dtype, masked=0.0, seed=0, ignore=-100):
    h, w = rnd(n, d, seed=seed + 1, dtype=dtype), rnd(v, d, seed=seed + 2, std=2.0 * d ** -0.5, dtype=dtype)
    g = torch.Generator(device="cuda").manual_seed(seed + 3)
    t = torch.randint(0, v, (n,), device="cuda", generator=g)
    if masked:
        t[torch.rand(n, device="cuda", generator=g) < masked] = ignore
    return h, w, t


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("n,d,v,masked", [(1, 64, 1, 0), (1, 64, 1000, 0), (2, 8, 3, 0), (7, 250, 503, 0.3),
                                          (64, 128, 255, 0), (100, 768, 257, 0.5), (128, 64, 640, 0.1),
                                          (129, 72, 1025, 0), (255, 33, 129, 0.9), (256, 256, 4000, 0),
                                          (511, 136, 997, 0.4), (1030, 96, 513, 0.2)])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_loss_and_gradients(n, d, v, masked, reduction, dtype):
    from mamba3_b200 import linear_cross_entropy

    h, w, t = loss_inputs(n, d, v, dtype, masked)
    if masked:
        t[n // 2] = v - 1
    h.requires_grad_(True), w.requires_grad_(True)
    y = linear_cross_entropy(h, w, t, reduction=reduction)
    assert y.dtype == torch.float32
    dl = rnd(n, seed=9) if reduction == "none" else torch.tensor(0.75, device="cuda")
    dh, dw = torch.autograd.grad(y, (h, w), dl)
    want = ref.loss(h, w, t, reduction=reduction, dloss=dl)
    ref.check(y, want["loss"], "loss")
    ref.check(dh, want["hidden"], "dhidden")
    ref.check(dw, want["weight"], "dweight")
    with torch.no_grad():
        assert torch.equal(linear_cross_entropy(h, w, t, reduction=reduction), y)


def test_loss_in_pieces_of_the_vocabulary():
    """Enough tokens that softmax - onehot is formed in two pieces of the vocabulary (the second ragged)."""
    from mamba3_b200 import linear_cross_entropy

    h, w, t = loss_inputs(33000, 64, 4100, torch.bfloat16, 0.0)
    t[5] = -100
    t[6] = 4099
    h.requires_grad_(True), w.requires_grad_(True)
    y = linear_cross_entropy(h, w, t, reduction="sum")
    dh, dw = torch.autograd.grad(y, (h, w))
    want = ref.loss(h, w, t, reduction="sum", dloss=1.0)
    ref.check(y, want["loss"], "loss")
    ref.check(dh, want["hidden"], "dhidden")
    ref.check(dw, want["weight"], "dweight")


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_loss_ignored_tokens(dtype):
    """All tokens ignored, another ignore_index (a valid id), NaN and infinity in ignored rows."""
    from mamba3_b200 import linear_cross_entropy

    h, w, t = loss_inputs(70, 64, 300, dtype)
    none = torch.full_like(t, -100)
    for reduction, want in (("mean", math.nan), ("sum", 0.0)):
        a, b = h.clone().requires_grad_(True), w.clone().requires_grad_(True)
        y = linear_cross_entropy(a, b, none, reduction=reduction)
        assert y.item() == want or (math.isnan(want) and math.isnan(y.item()))
        y.backward()
        assert not a.grad.any() and not b.grad.any()
    t = t % 5
    a, b = h.clone(), w.clone().requires_grad_(True)
    a[t == 3] = float("nan")
    a[(t == 3).nonzero()[0]] = float("inf")
    a.requires_grad_(True)
    y = linear_cross_entropy(a, b, t, ignore_index=3)
    dh, dw = torch.autograd.grad(y, (a, b))
    want = ref.loss(h, w, t, ignore=3, dloss=1.0)
    ref.check(y, want["loss"], "loss")
    ref.check(dh, want["hidden"], "dhidden")
    ref.check(dw, want["weight"], "dweight")


def test_loss_large_logits():
    """Logits of several thousands: the running maximum keeps the sums finite; a sure token has loss 0."""
    from mamba3_b200 import linear_cross_entropy

    h, w, t = loss_inputs(50, 64, 400, torch.bfloat16)
    h = h * 512
    want = ref.loss(h, w, t, reduction="none")
    y = linear_cross_entropy(h, w, t, reduction="none")
    ref.check(y, want["loss"], "loss")
    sure = (h.double() @ w.double().t()).argmax(1)
    y = linear_cross_entropy(h, w, sure, reduction="none")
    ref.check(y, ref.loss(h, w, sure, reduction="none")["loss"], "sure")
    bad = h.clone()
    bad[3, 5] = float("nan")
    y = linear_cross_entropy(bad, w, t, reduction="none")
    assert torch.isnan(y).nonzero().flatten().tolist() == [3]


def test_loss_target_out_of_range():
    from mamba3_b200 import M3bError, check_device_errors, linear_cross_entropy

    h, w, t = loss_inputs(20, 64, 100, torch.bfloat16)
    for bad in (100, -1, 2 ** 40):
        s = t.clone()
        s[4] = bad
        a = h.clone().requires_grad_(True)
        y = linear_cross_entropy(a, w, s, reduction="none")
        assert torch.isnan(y).nonzero().flatten().tolist() == [4]
        g, = torch.autograd.grad(y.sum(), a)
        assert torch.isnan(g).any(1).nonzero().flatten().tolist() == [4]
        with pytest.raises(M3bError, match="invalid argument"):
            check_device_errors()


def test_loss_shapes_strides_and_integer_types():
    from mamba3_b200 import linear_cross_entropy

    h, w, t = loss_inputs(60, 64, 200, torch.bfloat16)
    want = ref.loss(h, w, t, reduction="none")["loss"]
    for dt in (torch.int32, torch.int64, torch.int16):
        ref.check(linear_cross_entropy(h, w, t.to(dt), reduction="none"), want, str(dt))
    y = linear_cross_entropy(h.view(3, 20, 64), w, t.view(3, 20), reduction="none")
    assert y.shape == (3, 20)
    for off, width in ((8, 80), (3, 71)):
        buf = torch.zeros(60, width, device="cuda", dtype=torch.bfloat16)
        buf[:, off:off + 64] = h
        ref.check(linear_cross_entropy(buf[:, off:off + 64], w, t, reduction="none"), want, f"rows at {off}")
    ref.check(linear_cross_entropy(h, w.t().contiguous().t(), t, reduction="none"), want, "transposed weight")
    shift = linear_cross_entropy(h.view(3, 20, 64)[:, :-1], w, t.view(3, 20)[:, 1:], reduction="sum")
    full = t.view(3, 20).roll(-1, 1).clone()
    full[:, -1] = -100
    assert torch.equal(shift, linear_cross_entropy(h.view(3, 20, 64), w, full, reduction="sum"))
    e = linear_cross_entropy(h[:0], w, t[:0])
    assert math.isnan(e.item())
    assert linear_cross_entropy(h[:0], w, t[:0], reduction="sum").item() == 0.0
    assert linear_cross_entropy(h[:0], w, t[:0], reduction="none").shape == (0,)
    a, b = h[:0].clone().requires_grad_(True), w.clone().requires_grad_(True)
    linear_cross_entropy(a, b, t[:0], reduction="sum").backward()
    assert a.grad.shape == (0, 64) and not b.grad.any()


def test_loss_gradient_against_differences():
    """As for the feed-forward: central differences along a random direction, fp32."""
    from mamba3_b200 import linear_cross_entropy

    h, w, t = loss_inputs(40, 48, 90, torch.float32, 0.2)
    h.requires_grad_(True), w.requires_grad_(True)
    grads = torch.autograd.grad(linear_cross_entropy(h, w, t, reduction="sum"), (h, w))
    for i, p in enumerate((h, w)):
        v, s = rnd(*p.shape, seed=50 + i, std=p.numel() ** -0.5), 2.0 ** -6
        with torch.no_grad():
            f = lambda q: linear_cross_entropy(q if i == 0 else h, q if i else w, t, reduction="none").double().sum()  # noqa: E731
            slope = float((f(p + s * v) - f(p - s * v)) / (2 * s))
        want = float((grads[i].double() * v).sum())
        assert abs(slope - want) < 0.01 * float(grads[i].double().norm()), (i, slope, want)


# ---------------------------------------------------------------------------
# gradient clipping
# ---------------------------------------------------------------------------
SIZES = [1, 2, 7, 8, 255, 256, 1000, 8191, 8192, 8193, 100_001]


def grad_list(sizes, dtype, seed=0, std=0.01, pad=0):
    """Tensors at every alignment `pad` gives: views into one buffer, pad values apart."""
    buf = rnd(sum(sizes) + pad * len(sizes) + 16, seed=seed, std=std, dtype=dtype)
    got, at = [], 0
    for n in sizes:
        got.append(buf[at:at + n])
        at += n + pad
    return got


def clip_want(gs, max_norm, inf=False):
    v = [g.double() for g in gs]
    norm = max(float(x.abs().max()) for x in v if x.numel()) if inf else math.sqrt(sum(float((x * x).sum()) for x in v))
    return norm, [x * min(1.0, max_norm / (norm + 1e-6)) for x in v]


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("pad", [0, 1, 8])
@pytest.mark.parametrize("inf", [False, True])
def test_clip_in_place(dtype, pad, inf):
    from mamba3_b200 import clip_grads

    gs = grad_list(SIZES, dtype, pad=pad)
    for max_norm in (0.5, 1e-3, 1e6):
        want_norm, want = clip_want(gs, max_norm, inf)
        before = [g.clone() for g in gs]
        norm = clip_grads(gs, max_norm, math.inf if inf else 2.0)
        # fp32 sums of 32 squares, then fp64: 34 half steps of 2^-24, halved by the root, and its own rounding
        assert abs(norm.item() - want_norm) <= 20 * 2.0 ** -24 * want_norm
        for g, w, b in zip(gs, want, before):
            if max_norm == 1e6:
                assert torch.equal(g, b)
                continue
            # the factor (the norm's error and one rounding), the product's rounding, the result's
            err = w.abs() * (22 * 2.0 ** -24 + ref.half_step(dtype)) + ref.least(dtype)
            assert bool(((g.double() - w).abs() <= err).all())


@pytest.mark.parametrize("src,dst", [(torch.bfloat16, torch.float32), (torch.float16, torch.float16),
                                     (torch.float32, torch.bfloat16), (torch.float32, torch.float32)])
def test_clip_into_other_tensors(src, dst):
    from mamba3_b200 import clip_grads

    gs = grad_list(SIZES + [0], src, pad=3)
    outs = [torch.full(g.shape, 7.0, device="cuda", dtype=dst) for g in gs]
    for max_norm in (0.25, 1e6, math.inf):
        norm, want = clip_want(gs, max_norm)
        before = [g.clone() for g in gs]
        clip_grads(gs, max_norm, out=outs)
        for g, b, o, w in zip(gs, before, outs, want):
            assert torch.equal(g, b)
            err = w.abs() * (22 * 2.0 ** -24 + ref.half_step(dst)) + ref.least(dst)
            assert bool(((o.double() - w).abs() <= err).all())


def test_clip_many_tensors_mixed_types_and_orders():
    from mamba3_b200 import clip_grads

    gs = []
    for i in range(300):
        gs.append(rnd(1 + 37 * i % 501, seed=i, dtype=DTYPES[i % 3]))
    gs.append(rnd(40, 60, seed=400).t())  # dense in another order
    gs.append(rnd(3, 8, 5, seed=401, dtype=torch.bfloat16).permute(2, 0, 1))
    norm, want = clip_want(gs, 3.0)
    got = clip_grads(gs, 3.0)
    assert abs(got.item() - norm) <= 20 * 2.0 ** -24 * norm
    for g, w in zip(gs, want):
        # the factor 3 / 270 brings fp16 values below 0.0055 under its smallest normal, 2^-14: half a subnormal more
        err = w.abs() * (22 * 2.0 ** -24 + ref.half_step(g.dtype)) + ref.least(g.dtype)
        assert bool(((g.double() - w).abs() <= err).all())


def test_clip_special_values():
    from mamba3_b200 import clip_grads

    z = [torch.zeros(1000, device="cuda") for _ in range(3)]
    assert clip_grads(z, 1.0).item() == 0.0 and not any(t.any() for t in z)
    for scale in (1e-25, 1e25):  # squares past fp32's range at both ends
        g = [rnd(9000, seed=3) * scale, rnd(10, seed=4) * scale]
        norm, _ = clip_want(g, 1.0)
        assert abs(clip_grads([t.clone() for t in g], math.inf).item() - norm) <= 20 * 2.0 ** -24 * norm
    for bad in (math.nan, math.inf):
        for inf in (False, True):
            g = [rnd(5000, seed=5), rnd(100, seed=6)]
            g[1][3] = bad
            norm = clip_grads(g, 1.0, math.inf if inf else 2.0)
            assert math.isnan(norm.item()) if math.isnan(bad) else math.isinf(norm.item())
            if math.isnan(bad):
                assert all(torch.isnan(t).all() for t in g)
            else:
                assert not g[0].any() and torch.isnan(g[1][3]) and int(torch.isnan(g[1]).sum()) == 1


def test_clip_grad_norm_matches_torch():
    from mamba3_b200 import clip_grad_norm_

    def model(seed):
        torch.manual_seed(seed)
        m = torch.nn.Sequential(torch.nn.Linear(65, 33), torch.nn.LayerNorm(33), torch.nn.Linear(33, 7)).cuda()
        m(rnd(20, 65, seed=2)).square().sum().backward()
        return m

    a, b = model(1), model(1)
    na = clip_grad_norm_(a.parameters(), 0.7)
    nb = torch.nn.utils.clip_grad_norm_(b.parameters(), 0.7)
    torch.testing.assert_close(na, nb, rtol=1e-6, atol=0)
    for p, q in zip(a.parameters(), b.parameters()):
        torch.testing.assert_close(p.grad, q.grad, rtol=2e-6, atol=0)
    a[0].weight.grad[0, 0] = math.nan
    with pytest.raises(RuntimeError, match="not finite"):
        clip_grad_norm_(a.parameters(), 0.7, error_if_nonfinite=True)


# ---------------------------------------------------------------------------
# streams, graphs, the three together
# ---------------------------------------------------------------------------
def test_operators_on_another_stream_and_twice_at_once():
    from mamba3_b200 import gated_ffn, linear_cross_entropy

    t = ffn_inputs(300, 128, 136, torch.bfloat16, False, False)
    h, w, tg = loss_inputs(300, 128, 1000, torch.bfloat16, 0.2)
    y0, l0 = gated_ffn(t["x"], t["w_gate"], t["w_up"], t["w_down"]), linear_cross_entropy(h, w, tg)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            got.append((gated_ffn(t["x"], t["w_gate"], t["w_up"], t["w_down"]), linear_cross_entropy(h, w, tg)))
    torch.cuda.synchronize()
    for y, l in got:
        assert torch.equal(y, y0) and torch.equal(l, l0)


def test_training_step_captured_and_replayed():
    """Loss through the feed-forward, its gradients and their clipping in one CUDA graph, replayed on new
    inputs: the same values as the eager calls, bit for bit."""
    from mamba3_b200 import clip_grads, gated_ffn, linear_cross_entropy

    t = ffn_inputs(200, 64, 136, torch.bfloat16, False, True)
    _, w, tg = loss_inputs(200, 64, 500, torch.bfloat16, 0.3)
    leaves = [v.requires_grad_(True) for v in (t["x"], t["w_gate"], t["w_up"], t["w_down"], w)]

    def step():
        y = gated_ffn(*leaves[:4], residual=leaves[0], residual_scale=0.5)
        loss = linear_cross_entropy(y, leaves[4], tg)
        grads = torch.autograd.grad(loss, leaves)
        norm = clip_grads(grads, 0.05)
        return (loss.detach(), norm, *grads)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    for seed in (1, 2):
        with torch.no_grad():
            leaves[0].copy_(rnd(200, 64, seed=seed, dtype=torch.bfloat16))
            tg.copy_(torch.randint(0, 500, (200,), device="cuda"))
            if seed == 2:
                tg[:150] = -100
        g.replay()
        got = [o.clone() for o in out]
        torch.cuda.synchronize()
        for a, b in zip(got, step()):
            assert torch.equal(a, b)


def test_lm_training_step_uses_the_operators():
    """KulaMambaLM with fused_mlp and return_logits=False: the plain model's loss and gradients within the
    model's bf16 rounding, then clipping by the global norm."""
    from mamba3_b200 import KulaMambaLM, clip_grad_norm_

    cfg = dict(vocab_size=203, d_model=64, n_layers=2, d_state=16, headdim=16)
    torch.manual_seed(0)
    a = KulaMambaLM(**cfg).cuda().train()
    torch.manual_seed(0)
    b = KulaMambaLM(**cfg, fused_mlp=True).cuda().train()
    ids = torch.randint(0, 203, (2, 40), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    labels = ids.clone()
    labels[0, :10] = -100
    ra, rb = a(ids, labels), b(ids, labels, return_logits=False)
    assert set(rb) == {"loss"}
    torch.testing.assert_close(rb["loss"], ra["loss"], rtol=2e-3, atol=0)
    ra["loss"].backward()
    rb["loss"].backward()
    for (n, p), q in zip(a.named_parameters(), b.parameters()):
        err = (p.grad - q.grad).norm() / p.grad.norm()
        assert err < 3e-2, (n, float(err))
    norm = clip_grad_norm_(b.parameters(), 0.1)
    total = torch.sqrt(sum(p.grad.double().square().sum() for p in b.parameters()))
    assert norm.item() > 0.1 and abs(total.item() - 0.1) < 1e-5
    rc = b(ids, labels)  # with logits too: the plain loss
    torch.testing.assert_close(rc["loss"], rb["loss"], rtol=1e-4, atol=0)
    assert rc["logits"].shape == (2, 40, 203)


def test_lm_decode_with_the_fused_mlp():
    """Greedy decoding through GraphDecoder and generate: the operator in the decode step, the same tokens from
    both."""
    from mamba3_b200 import GraphDecoder, KulaMambaLM

    torch.manual_seed(0)
    lm = KulaMambaLM(vocab_size=97, d_model=64, n_layers=2, d_state=16, headdim=16, fused_mlp=True)
    lm = lm.cuda().bfloat16().eval()
    ids = torch.randint(0, 97, (3, 9), device="cuda", generator=torch.Generator(device="cuda").manual_seed(4))
    out = lm.generate(ids, max_new_tokens=12, temperature=0.0)
    dec = GraphDecoder(lm, 3, 12, compact=False)
    assert torch.equal(dec.generate(ids), out)


# ---------------------------------------------------------------------------
# calls at the edges of what the documentation allows
# ---------------------------------------------------------------------------
def test_loss_frozen_weight_or_hidden():
    from mamba3_b200 import linear_cross_entropy

    h, w, t = loss_inputs(90, 64, 300, torch.bfloat16, 0.2)
    want = ref.loss(h, w, t, dloss=1.0)
    a = h.clone().requires_grad_(True)
    linear_cross_entropy(a, w, t).backward()
    ref.check(a.grad, want["hidden"], "hidden alone")
    b = w.clone().requires_grad_(True)
    linear_cross_entropy(h, b, t).backward()
    ref.check(b.grad, want["weight"], "weight alone")


def test_loss_small_probabilities_in_fp16():
    """A sure prediction over a large vocabulary: the other 19,999 probabilities are near 2e-9, which fp16 alone
    would drop, but together they are the whole gradient along what the others share."""
    from mamba3_b200 import linear_cross_entropy

    n, d, v = 64, 64, 20000
    h, w, t = loss_inputs(n, d, v, torch.float16)
    w = (w * 0.02).contiguous()
    h[:, 0], h[:, 1] = 10.0, 0.0
    w[:, 0], w[:, 1] = 0.0, 1.0
    w[7] = 0.0
    w[7, 0] = 2.0  # the target's logit 20 above the rest: 4e-5 of the mass on all others
    t.fill_(7)
    h.requires_grad_(True)
    (linear_cross_entropy(h, w, t) * 1024.0).backward()
    p = torch.softmax(h.detach().double() @ w.double().t(), 1)
    p[:, 7] = 0.0
    want = 1024.0 * p.sum(1) / n
    # two roundings to fp16 (the scaled probability, the result) and fp32 logits of 20 and their log-sum
    err = (2 * 2.0 ** -11 + 8 * 2.0 ** -20) * want
    assert bool(((h.grad[:, 1].double() - want).abs() <= err).all())


def test_ffn_offsets_past_32_bits():
    """act, g and u, dg and du of more than 2^31 values: the last rows against the plain form, and the weight
    gradient's sum over all rows through a product with few live rows."""
    from mamba3_b200 import gated_ffn

    n, d, f = 400_200, 32, 5504
    x = torch.zeros(n, d, device="cuda", dtype=torch.bfloat16)
    live = torch.tensor([0, 1, 255, 256, 390_167, 390_168, n - 2, n - 1], device="cuda")  # 2^31 / 5504 = 390,167
    x[live] = rnd(len(live), d, seed=1, dtype=torch.bfloat16)
    t = ffn_inputs(1, d, f, torch.bfloat16, False, False)
    leaves = [v.requires_grad_(True) for v in (x, t["w_gate"], t["w_up"], t["w_down"])]
    y = gated_ffn(*leaves)
    dout = torch.zeros_like(y)
    dout[live] = rnd(len(live), d, seed=2, dtype=torch.bfloat16)
    grads = torch.autograd.grad(y, leaves, dout)
    small = dict(t, x=x.detach()[live])
    want = ffn_want(small, dout=dout[live])
    ref.check(y[live], want["out"], "out")
    ref.check(grads[0][live], want["x"], "dx")
    for g, k in zip(grads[1:], ("w_gate", "w_up", "w_down")):
        value, bound = want[k]
        ref.check(g, (value, bound * 2), k)  # the other rows add zeros, in more steps than the bound counts
    dead = torch.ones(n, dtype=torch.bool, device="cuda")
    dead[live] = False
    assert not y[dead].any() and not grads[0][dead].any()


def test_loss_offsets_past_32_bits():
    """softmax - onehot of more than 2^31 values in one piece: the last tokens' gradients."""
    from mamba3_b200 import linear_cross_entropy

    n, d, v = 1_060_000, 16, 2050
    h, w, _ = loss_inputs(300, d, v, torch.bfloat16)
    t = torch.randint(0, v, (n,), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    big = h.repeat(n // 300 + 1, 1)[:n].contiguous().requires_grad_(True)
    y = linear_cross_entropy(big, w, t, reduction="sum")
    dh, = torch.autograd.grad(y, big)
    for s in (slice(0, 300), slice(n - 300, n)):
        want = ref.loss(big[s], w, t[s], reduction="sum", dloss=1.0)
        ref.check(dh[s], want["hidden"], f"rows {s}")


def test_clip_offsets_past_32_bits():
    from mamba3_b200 import clip_grads

    n = (1 << 31) + 8200
    g = torch.zeros(n, device="cuda", dtype=torch.bfloat16)
    at = torch.tensor([0, 5, (1 << 31) - 1, 1 << 31, n - 1], device="cuda")
    g[at] = 2.0
    norm = clip_grads([g], 1.0)
    assert abs(norm.item() - math.sqrt(20.0)) < 1e-5
    want = torch.tensor(2.0 / (math.sqrt(20.0) + 1e-6)).bfloat16().item()
    assert g[at].tolist() == [want] * 5 and int((g != 0).sum()) == 5


def test_operators_under_compile():
    """As opaque nodes of a traced graph, forward and backward: the eager values."""
    from mamba3_b200 import gated_ffn, linear_cross_entropy

    t = ffn_inputs(40, 64, 72, torch.bfloat16, False, True)
    _, w, tg = loss_inputs(40, 64, 200, torch.bfloat16, 0.2)

    def step(x, wg, wu, wd, w):
        y = gated_ffn(x, wg, wu, wd, residual=x, residual_scale=0.5)
        return linear_cross_entropy(y, w, tg)

    leaves = [v.clone().requires_grad_(True) for v in (t["x"], t["w_gate"], t["w_up"], t["w_down"], w)]
    eager = step(*leaves)
    want = torch.autograd.grad(eager, leaves)
    got = torch.compile(step, backend="aot_eager")(*leaves)
    assert torch.equal(got, eager)
    for a, b in zip(torch.autograd.grad(got, leaves), want):
        assert torch.equal(a, b)


def test_gradients_are_the_same_every_time():
    """Jobs are drawn in an order that changes from run to run; the sums are not."""
    from mamba3_b200 import gated_ffn, linear_cross_entropy

    t = ffn_inputs(1000, 256, 520, torch.bfloat16, False, False)
    h, w, tg = loss_inputs(1000, 256, 5000, torch.bfloat16, 0.3)
    leaves = [v.requires_grad_(True) for v in t.values()] + [h.requires_grad_(True), w.requires_grad_(True)]
    first = None
    for _ in range(5):
        g = torch.autograd.grad(gated_ffn(*leaves[:4]).float().square().sum() + linear_cross_entropy(*leaves[4:], tg),
                                leaves)
        if first is None:
            first = g
        assert all(torch.equal(a, b) for a, b in zip(g, first))


# ---------------------------------------------------------------------------
# cross entropy of a few rows
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("n,d,v,ignored", [(1, 8, 5, ()), (1, 513, 2000, ()), (2, 1100, 33, (1,)), (3, 1, 1000, ()),
                                           (4, 512, 19000, (0,)), (5, 2052, 700, (2, 3)), (6, 130, 40003, ()),
                                           (8, 768, 4097, ()), (8, 67, 515, (0, 1, 2, 4, 5, 6, 7)), (9, 512, 515, (8,))])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_loss_of_few_rows(n, d, v, ignored, reduction, dtype):
    from mamba3_b200 import linear_cross_entropy

    h, w, t = loss_inputs(n, d, v, dtype)
    clean = h.clone()
    for r in ignored:
        t[r] = -100
        h[r] = float("nan")
    kept = [r for r in range(n) if r not in ignored]
    t[kept[0]], t[kept[-1]] = 0, v - 1
    h.requires_grad_(True), w.requires_grad_(True)
    y = linear_cross_entropy(h, w, t, reduction=reduction)
    dl = rnd(n, seed=9) if reduction == "none" else torch.tensor(-1.5, device="cuda")
    dh, dw = torch.autograd.grad(y, (h, w), dl, retain_graph=True)
    want = ref.loss(clean, w, t, reduction=reduction, dloss=dl)
    ref.check(y, want["loss"], "loss")
    ref.check(dh, want["hidden"], "dhidden")
    ref.check(dw, want["weight"], "dweight")
    again = torch.autograd.grad(linear_cross_entropy(h, w, t, reduction=reduction), (h, w), dl)
    assert torch.equal(again[0], dh) and torch.equal(again[1], dw)
    # one gradient alone.  (Nine rows take the general form, which may split a product's sum in other places
    # when it runs alone: other orders of the same terms, each within the bound of every order.)
    only_h, = torch.autograd.grad(linear_cross_entropy(h, w.detach(), t, reduction=reduction), h, dl)
    only_w, = torch.autograd.grad(linear_cross_entropy(h.detach(), w, t, reduction=reduction), w, dl)
    ref.check(only_h, want["hidden"], "dhidden alone")
    ref.check(only_w, want["weight"], "dweight alone")
    if n <= 8:
        assert torch.equal(only_h, dh) and torch.equal(only_w, dw)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_loss_of_few_rows_at_its_edges(dtype):
    """No kept row, targets out of range, infinite and large logits, rows and weights that start anywhere."""
    from mamba3_b200 import M3bError, check_device_errors, linear_cross_entropy

    h, w, t = loss_inputs(6, 64, 300, dtype)
    none = torch.full_like(t, -100)
    for reduction, want in (("mean", math.nan), ("sum", 0.0)):
        a, b = h.clone().requires_grad_(True), w.clone().requires_grad_(True)
        y = linear_cross_entropy(a, b, none, reduction=reduction)
        assert y.item() == want or (math.isnan(want) and math.isnan(y.item()))
        y.backward()
        assert not a.grad.any() and not b.grad.any()
    assert not linear_cross_entropy(h, w, none, reduction="none").any()
    for bad in (300, -1, 2 ** 40):
        s = t.clone()
        s[4] = bad
        a = h.clone().requires_grad_(True)
        y = linear_cross_entropy(a, w, s, reduction="none")
        assert torch.isnan(y).nonzero().flatten().tolist() == [4]
        g, = torch.autograd.grad(y.sum(), a)
        assert torch.isnan(g).any(1).nonzero().flatten().tolist() == [4]
        with pytest.raises(M3bError, match="invalid argument"):
            check_device_errors()
    # columns of -infinity leave the others as they are; a row of them, or one of +infinity, has no loss
    a, b = h.abs(), w.clone()
    b[7] = float("-inf")
    s = t.clone()
    s[s == 7] = 8
    keep = torch.arange(300, device="cuda") != 7
    want = ref.loss(a, b[keep], s - (s > 7).long(), reduction="none")["loss"]
    ref.check(linear_cross_entropy(a, b, s, reduction="none"), want, "a column of -infinity")
    for x in (float("inf"), float("-inf")):
        assert torch.isnan(linear_cross_entropy(a, torch.full_like(b, x), s, reduction="none")).all()
    ref.check(linear_cross_entropy(h * 512, w, t, reduction="none"), ref.loss(h * 512, w, t, reduction="none")["loss"], "large")
    want = ref.loss(h, w, t, dloss=1.0)
    for off, width in ((8, 80), (3, 71)):
        buf = torch.full((6, width), float("nan"), device="cuda", dtype=dtype)
        buf[:, off:off + 64] = h
        flat = torch.empty(300 * 64 + 8, device="cuda", dtype=dtype)
        moved = flat[off:off + 300 * 64].view(300, 64) if off == 3 else w.clone()
        moved.copy_(w)
        a, b = buf[:, off:off + 64].detach().requires_grad_(True), moved.detach().requires_grad_(True)
        y = linear_cross_entropy(a, b, t)
        ref.check(y, want["loss"], f"rows at {off}")
        dh, dw = torch.autograd.grad(y, (a, b))
        ref.check(dh, want["hidden"], "dhidden")
        ref.check(dw, want["weight"], "dweight")


def test_loss_of_few_rows_captured():
    from mamba3_b200 import linear_cross_entropy

    h, w, t = loss_inputs(5, 200, 3001, torch.bfloat16)
    h.requires_grad_(True), w.requires_grad_(True)

    def step():
        y = linear_cross_entropy(h, w, t)
        return (y,) + torch.autograd.grad(y, (h, w))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for seed in (1, 2):
        g = torch.Generator(device="cuda").manual_seed(seed)
        with torch.no_grad():
            h.copy_(torch.randn(5, 200, device="cuda", generator=g))
            t.copy_(torch.randint(0, 3001, (5,), device="cuda", generator=g))
            t[seed] = -100
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, step()):
            assert torch.equal(a, b)


def test_loss_of_few_rows_offsets_past_32_bits():
    """A weight of more than 2^31 values, zero but for a few rows: the sums have closed forms."""
    from mamba3_b200 import linear_cross_entropy

    d, v = 2048, (1 << 20) + 77
    w = torch.zeros(v, d, device="cuda", dtype=torch.bfloat16)
    at = torch.tensor([0, 5, 1 << 20, v - 1], device="cuda")
    w[at] = rnd(4, d, seed=2, std=2.0 * d ** -0.5, dtype=torch.bfloat16)
    h = rnd(3, d, seed=1, dtype=torch.bfloat16).requires_grad_(True)
    t = torch.tensor([v - 1, 1 << 20, 9], device="cuda")
    y = linear_cross_entropy(h, w.requires_grad_(True), t, reduction="sum")
    dh, dw = torch.autograd.grad(y, (h, w))
    H, W = h.detach().double(), w.detach()[at].double()
    z = H @ W.t()
    lse = (z.exp().sum(1) + (v - 4)).log()
    loss = lse.sum() - z[0, 3] - z[1, 2]
    # 600 steps of 2^-23 for the statistics (as in the plain form), 2^-14 with the logits' sums
    assert abs(y.item() - loss.item()) <= 2.0 ** -14 * 3 + 2.0 ** -23 * abs(loss.item())
    p = (z - lse[:, None]).exp()
    rest = (-lse).exp()  # of every zero row
    dz = p.clone()
    dz[0, 3] -= 1.0
    dz[1, 2] -= 1.0
    want, by = dz @ W, dz.abs() @ W.abs()
    assert bool(((dh.double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -13 * by + 2.0 ** -60).all())
    for row, c in ((0, dz[:, 0]), (5, dz[:, 1]), (1 << 20, dz[:, 2]), (v - 1, dz[:, 3]), (9, rest - torch.tensor(
            [0.0, 0.0, 1.0], device="cuda", dtype=torch.float64)), (v - 2, rest)):
        want, by = c @ H, c.abs() @ H.abs()
        assert bool(((dw[row].double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -13 * by).all()), row


def test_loss_of_few_rows_under_compile():
    from mamba3_b200 import linear_cross_entropy

    h, w, t = loss_inputs(6, 64, 333, torch.bfloat16)
    leaves = [h.requires_grad_(True), w.requires_grad_(True)]
    eager = linear_cross_entropy(*leaves, t)
    want = torch.autograd.grad(eager, leaves)
    got = torch.compile(lambda a, b: linear_cross_entropy(a, b, t), backend="aot_eager")(*leaves)
    assert torch.equal(got, eager)
    for a, b in zip(torch.autograd.grad(got, leaves), want):
        assert torch.equal(a, b)


def test_block_with_another_module_as_its_mlp():
    from mamba3_b200 import KulaMambaBlock

    blk = KulaMambaBlock(64, d_state=16, headdim=16).cuda().bfloat16()
    blk.mlp = torch.nn.Linear(64, 64).cuda().bfloat16()
    x = rnd(2, 64, 64, seed=1, dtype=torch.bfloat16)
    assert blk(x).shape == x.shape
    blk.train()
    blk(x.requires_grad_(True)).float().sum().backward()
    assert blk.mlp.weight.grad.any()
