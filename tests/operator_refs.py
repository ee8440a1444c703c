"""Plain 64-bit forms of the training and serving operators, with the error their kernels may make.

Every function returns values and, beside each, a bound on the kernel's error derived from the roundings
it makes: the tensor cores add 16 products at a time into fp32, so a sum of K products is off by at most
(K / 16 + 8) steps of 2^-23 of the sum of their magnitudes (six times as many steps for fp32 operands,
which travel as three bf16 planes); operands of a following product and results are rounded once to their
dtype (half a step: 2^-8 for bf16, 2^-11 for fp16, 2^-24 for fp32, or half the smallest subnormal).
"""

import torch

F64 = torch.float64


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def least(dtype):
    """Half the smallest subnormal: what rounding may take from a value near zero."""
    f = torch.finfo(dtype)
    return f.tiny * f.eps / 2


def sum_error(k, dtype):
    """Relative to the sum of magnitudes of k products."""
    return (k / 16 * (6 if dtype == torch.float32 else 1) + 8) * 2.0 ** -23


def rounded(v, err, dtype):
    return err + half_step(dtype) * (v.abs() + err) + least(dtype)


def operand_step(dtype):
    """Rounding of a value that a following product reads: fp32 keeps its 24 bits in three planes."""
    return 2.0 ** -23 if dtype == torch.float32 else half_step(dtype)


def ffn(x, wg, wu, wd, bg=None, bu=None, bd=None, residual=None, scale=1.0, dout=None):
    """{name: (value, bound)} of the gated feed-forward and, with dout, its gradients."""
    dt = x.dtype
    d, f = x.shape[1], wg.shape[0]
    n = x.shape[0]
    X, G, U, D = (t.detach().to(F64) for t in (x, wg, wu, wd))
    g, u = X @ G.t(), X @ U.t()
    eg, eu = sum_error(d, dt) * (X.abs() @ G.abs().t()), sum_error(d, dt) * (X.abs() @ U.abs().t())
    if bg is not None:
        g, u = g + bg.detach().to(F64), u + bu.detach().to(F64)
        eg, eu = eg + 2.0 ** -23 * g.abs(), eu + 2.0 ** -23 * u.abs()
    sig = torch.sigmoid(g)
    # the hardware exponential (2 + 1.2 |g| steps) and divide (2), and the products: |g| < 40 keeps this above them
    es = 2.0 ** -23 * (8 + 2 * g.abs().clamp(max=40))
    act = g * sig
    a = act * u
    ea = 1.1 * eg * u.abs() + act.abs() * eu + eg * eu * 1.1 + es * a.abs() + 2.0 ** -126
    ea = ea + operand_step(dt) * (a.abs() + ea) + (least(dt) if dt != torch.float32 else 0)
    y = a @ D.t()
    ey = sum_error(f, dt) * (a.abs() @ D.abs().t()) + ea @ D.abs().t()
    if bd is not None:
        y = y + bd.detach().to(F64)
    y, ey = y * scale, (ey + 2.0 ** -22 * y.abs()) * abs(scale)
    if residual is not None:
        r = residual.detach().to(F64)
        y, ey = y + r, ey + 2.0 ** -23 * (y.abs() + r.abs())
    out = {"out": (y, rounded(y, ey, dt))}
    if dout is None:
        return out
    dy = dout.detach().to(F64)
    da = scale * (dy @ D)
    eda = abs(scale) * (sum_error(d, dt) + 2.0 ** -22) * (dy.abs() @ D.abs())
    pg, pu = u * sig * (1 + g * (1 - sig)), act
    if dt != torch.float32:  # the forward keeps the upper 24 bits of g and u, 16 of them significant: off by less than one step, 2^-15 of 1..2
        eg, eu = eg + 2.0 ** -15 * g.abs(), eu + 2.0 ** -15 * u.abs()
    # d/dg of u sig (1 + g (1 - sig)) is at most u / 2 in magnitude; 1 - sig and the sum are within 3 steps
    epg = 0.5 * u.abs() * eg + 1.1 * eu + 4 * es * u.abs() * sig * (1 + g.abs())
    epu = 1.1 * eg + es * act.abs()
    res = {}
    for name, p, ep in (("g", pg, epg), ("u", pu, epu)):
        v = da * p
        e = eda * (p.abs() + ep) + da.abs() * ep + 2.0 ** -22 * v.abs()
        e = e + operand_step(dt) * (v.abs() + e) + (least(dt) if dt != torch.float32 else 0)
        res[name] = (v, e)
    (dg, edg), (du, edu) = res["g"], res["u"]
    c = sum_error(2 * f, dt)
    dx = dg @ G + du @ U
    out["x"] = (dx, rounded(dx, c * (dg.abs() @ G.abs() + du.abs() @ U.abs()) + edg @ G.abs() + edu @ U.abs(), dt))
    c = sum_error(n, dt)
    for name, v, e, o in (("w_gate", dg, edg, X), ("w_up", du, edu, X)):
        w = v.t() @ o
        out[name] = (w, rounded(w, c * (v.abs().t() @ o.abs()) + e.t() @ o.abs(), dt))
    w = scale * (dy.t() @ a)
    out["w_down"] = (w, rounded(w, abs(scale) * (c * (dy.abs().t() @ a.abs()) + dy.abs().t() @ ea) + 2.0 ** -22 * w.abs(),
                                dt))
    plain = n * 2.0 ** -24 + 2.0 ** -22  # a plain fp32 sum over the rows
    for name, v, e in (("b_gate", dg, edg), ("b_up", du, edu), ("b_down", scale * dy, 0 * dy)):
        s = v.sum(0)
        out[name] = (s, rounded(s, plain * v.abs().sum(0) + e.sum(0), dt))
    out["residual"] = (dy, torch.zeros_like(dy))
    return out


def loss(h, w, t, ignore=-100, reduction="mean", dloss=None):
    """{name: (value, bound)}: the loss and, with dloss (a number, or one per token for "none"), gradients."""
    dt = h.dtype
    n, d = h.shape
    v = w.shape[0]
    keep = t != ignore
    k = int(keep.sum())
    H, W = h.detach()[keep].to(F64), w.detach().to(F64)
    tk = t[keep].long()
    rows = torch.arange(k, device=h.device)
    z = H @ W.t()
    ez = (sum_error(d, dt) * (H.abs() @ W.abs().t())) if k else z
    top = ez.amax(1) if k else z.sum(1)
    lse = torch.logsumexp(z, 1)
    # statistics: powers of two of scaled logits (a step each of the largest logit), sums of v terms in
    # up to 512 parts, and the join
    big = z.abs().amax(1) if k else lse
    el = top + 2.0 ** -22 * (big + lse.abs()) + 600 * 2.0 ** -23
    li = lse - z[rows, tk]
    eli = el + top + 2.0 ** -22 * (lse.abs() + big)
    if reduction == "none":
        full = torch.zeros(n, dtype=F64, device=h.device)
        ef = torch.zeros_like(full)
        full[keep], ef[keep] = li, rounded(li, eli, torch.float32)
        out = {"loss": (full, ef)}
    else:
        c = 1.0 / k if reduction == "mean" and k else float("nan") if reduction == "mean" else 1.0
        s = li.sum() * c
        out = {"loss": (s, rounded(s, (eli.sum() + 2.0 ** -24 * li.abs().sum()) * c, torch.float32))}
    if dloss is None:
        return out
    if reduction == "none":
        roww, alpha = dloss.detach().to(F64)[keep], 1.0
    else:
        roww = torch.ones(k, dtype=F64, device=h.device)
        alpha = float(dloss) * ((1.0 / k if k else 0.0) if reduction == "mean" else 1.0)
    p = torch.exp(z - lse[:, None])
    ep = p * (ez + el[:, None] + 2.0 ** -22 * (2 + big[:, None] + lse.abs()[:, None]))
    p[rows, tk] -= 1.0
    dz = p * roww[:, None]
    e = (ep + 2.0 ** -22 * p.abs()) * roww.abs()[:, None]
    e = e + operand_step(dt) * (dz.abs() + e) + (least(dt) if dt != torch.float32 else 0)
    dh = torch.zeros(n, d, dtype=F64, device=h.device)
    eh = torch.zeros_like(dh)
    g = alpha * (dz @ W)
    eg = abs(alpha) * ((sum_error(v, dt) + 2.0 ** -20) * (dz.abs() @ W.abs()) + e @ W.abs())
    dh[keep], eh[keep] = g, rounded(g, eg, dt)
    dw = alpha * (dz.t() @ H)
    ew = abs(alpha) * ((sum_error(k, dt) + 2.0 ** -22) * (dz.abs().t() @ H.abs()) + e.t() @ H.abs())
    out["hidden"] = (dh, eh)
    out["weight"] = (dw, rounded(dw, ew, dt))
    return out


def check(got, want, what=""):
    """Every element of got within its bound of want = (value, bound); both NaN where either is."""
    value, bound = want
    assert got.shape == value.shape, (what, got.shape, value.shape)
    g = got.detach().to(F64)
    nan = torch.isnan(value)
    assert torch.equal(torch.isnan(g), nan), f"{what}: NaN in other places"
    off = (g - value).abs()
    bad = (off > bound) & ~nan
    if bool(bad.any()):
        ratio = (off / bound.clamp(min=1e-300))[bad].max()
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} elements past their bound, by up to "
                             f"{float(ratio):.2f} times (largest error {float(off[bad].max()):.3g})")
