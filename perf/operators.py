"""Workloads of the training and serving operators around the Mamba-3 layers.

Three operators that a KulaMambaLM step needs beside the SSM layer, each in its plain form (elementary torch
operations in 32 bits, rounded once at the end) and, with ``own`` true, as calls of the package:

* ``linear_cross_entropy(hidden, weight, targets)``: the language-model loss straight from the final hidden states and
  the lm_head weight.  logits = hidden weight^T, loss = mean over the kept tokens of logsumexp(logits) - logits[target];
  gradients for hidden and weight.
* ``gated_ffn(x, w_gate, w_up, w_down, ...)``: the blocks' gated feed-forward, silu(x Wg^T + bg) * (x Wu^T + bu) through
  Wd^T (+ bd), with the block's scaled residual; gradients for every input.
* ``clip_grads(grads, max_norm, out=...)``: the global 2-norm over many gradients and the clipped gradients, here
  written to the optimizer's main gradients.
"""

import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}
IGNORE = -100

# The work of the largest listed case of each operator; a drawn case costs no more.
CE_MOST = 16384 * 2048 * 50257
FFN_MOST = 16384 * 2048 * 5504
CLIP_MOST = 600_000_000


def listed():
    return [
        # The loss of a fine-tuning step of the 768-wide LM (vocabulary 32,000): two packed rows of 2048 tokens, of
        # which the prompts' tokens (four in ten) carry no loss.
        {"name": "loss_finetune_bf16", "op": "loss", "dtype": "bf16", "tokens": 4096, "d": 768, "vocab": 32000,
         "masked": 0.4, "train": True},
        # The loss of a pretraining micro-batch of a 2048-wide LM with a byte-pair vocabulary of odd size.
        {"name": "loss_pretrain_bf16", "op": "loss", "dtype": "bf16", "tokens": 16384, "d": 2048, "vocab": 50257,
         "masked": 0.0, "train": True},
        # Validation loss on one document of odd length, fp16, no gradients.
        {"name": "loss_eval_fp16", "op": "loss", "dtype": "fp16", "tokens": 1021, "d": 1024, "vocab": 32000,
         "masked": 0.0, "train": False},
        # A small model trained in full precision, ragged everywhere.
        {"name": "loss_small_fp32", "op": "loss", "dtype": "fp32", "tokens": 500, "d": 250, "vocab": 5003,
         "masked": 0.1, "train": True},
        # One sequence decoding: a single token through a block's MLP (d_model 768, the block's own d_ff 2112) with the
        # block's residual; latency.
        {"name": "ffn_decode_one_bf16", "op": "ffn", "dtype": "bf16", "tokens": 1, "d": 768, "ff": 2112, "bias": False,
         "residual": True, "train": False},
        # The batch-256 decode step of the same model.
        {"name": "ffn_decode_256_bf16", "op": "ffn", "dtype": "bf16", "tokens": 256, "d": 768, "ff": 2112,
         "bias": False, "residual": True, "train": False},
        # A training step's MLP of the same model: eight rows of 2048 tokens, forward and backward.
        {"name": "ffn_train_bf16", "op": "ffn", "dtype": "bf16", "tokens": 16384, "d": 768, "ff": 2112, "bias": False,
         "residual": True, "train": True},
        # The MLP of the 2048-wide model (d_ff 5504), a large training micro-batch in fp16.
        {"name": "ffn_wide_train_fp16", "op": "ffn", "dtype": "fp16", "tokens": 16384, "d": 2048, "ff": 5504,
         "bias": False, "residual": False, "train": True},
        # Full precision, biases, sizes that are no multiple of anything.
        {"name": "ffn_odd_train_fp32", "op": "ffn", "dtype": "fp32", "tokens": 777, "d": 323, "ff": 897, "bias": True,
         "residual": True, "train": True},
        # A small model's gradients: a few short tensors; latency.
        {"name": "clip_small_fp32", "op": "clip", "dtype": "fp32", "out": "fp32", "tensors": 18, "numel": 250_007,
         "clips": True},
        # The 24-layer LM's bf16 gradients (about 240 M values in 400 tensors) into fp32 main gradients.
        {"name": "clip_lm_bf16", "op": "clip", "dtype": "bf16", "out": "fp32", "tensors": 400, "numel": 238_000_000,
         "clips": True},
        # A larger model's fp32 gradients whose norm is below the limit: they pass through as they are.
        {"name": "clip_large_fp32", "op": "clip", "dtype": "fp32", "out": "fp32", "tensors": 290, "numel": 600_000_000,
         "clips": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """A feature width: mostly a multiple of 64, some of 8, some of nothing."""
    w, kind = _log(rng, lo, hi), rng.random()
    return max(lo, w // 64 * 64) if kind < 0.6 else max(lo, w // 8 * 8) if kind < 0.85 else w


def draw(rng):
    op = rng.choice(["loss", "ffn", "clip"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op == "loss":
        d, vocab = _width(rng, 128, 2048), _log(rng, 1000, 50257)
        # full precision models here are small
        most = CE_MOST // 16 if dtype == "fp32" else CE_MOST
        tokens = min(_log(rng, 1, 16384), max(1, most // (d * vocab)))
        return {"op": "loss", "dtype": dtype, "tokens": tokens, "d": d, "vocab": vocab,
                "masked": round(rng.choice([0.0, rng.uniform(0.0, 0.9)]), 3), "train": rng.random() < 0.7}
    if op == "ffn":
        d = _width(rng, 64, 2048)
        ff = max(16, min(5504, int(d * rng.uniform(1.5, 4.0)) // rng.choice([64, 64, 8, 1])
                         * rng.choice([64, 64, 8, 1])))
        most = FFN_MOST // 16 if dtype == "fp32" else FFN_MOST
        tokens = min(_log(rng, 1, 16384), max(1, most // (d * ff)))
        return {"op": "ffn", "dtype": dtype, "tokens": tokens, "d": d, "ff": ff, "bias": rng.random() < 0.3,
                "residual": rng.random() < 0.6, "train": rng.random() < 0.6}
    tensors = _log(rng, 1, 500)
    return {"op": "clip", "dtype": dtype, "out": "fp32" if rng.random() < 0.6 else dtype, "tensors": tensors,
            "numel": max(tensors, _log(rng, 1000, CLIP_MOST // 2)), "clips": rng.random() < 0.7}


def _sizes(case):
    """The tensors' lengths of a clip case: a few large ones (projections, the embedding), many short ones (norm
    weights, biases), together case["numel"] or a little less."""
    n, total = case["tensors"], case["numel"]
    share = [1.0 if i % 4 == 0 else 0.4 if i % 4 == 1 else 0.0005 for i in range(n)]
    whole = sum(share)
    return [max(1, int(total * s / whole)) for s in share]


def _views(flat, sizes):
    """Views of one buffer, each starting on a multiple of 128 values, as a bucketed gradient buffer lays them out."""
    at, got = 0, []
    for n in sizes:
        got.append(flat[at:at + n])
        at += -(-n // 128) * 128
    return got


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape, std=1.0):
        return torch.randn(*shape, device="cuda", generator=g).mul_(std).to(dt)

    if case["op"] == "loss":
        n, d, v = case["tokens"], case["d"], case["vocab"]
        targets = torch.randint(0, v, (n,), device="cuda", generator=g)
        if case["masked"]:
            targets[torch.rand(n, device="cuda", generator=g) < case["masked"]] = IGNORE
            targets[n // 2] = 7  # one token at least carries a loss
        s = {"hidden": normal(n, d), "weight": normal(v, d, std=2.5 / math.sqrt(d)), "targets": targets}
        leaves = ("hidden", "weight")
    elif case["op"] == "ffn":
        n, d, f = case["tokens"], case["d"], case["ff"]
        s = {"x": normal(n, d), "w_gate": normal(f, d, std=1.0 / math.sqrt(d)),
             "w_up": normal(f, d, std=1.0 / math.sqrt(d)), "w_down": normal(d, f, std=1.0 / math.sqrt(f))}
        if case["bias"]:
            s.update(b_gate=normal(f, std=0.2), b_up=normal(f, std=0.2), b_down=normal(d, std=0.2))
        if case["residual"]:
            s["residual"] = normal(n, d)
        leaves = tuple(s)
        s["scale"] = 1.0 / math.sqrt(2 * 24) if case["residual"] else 1.0  # the depth scaling of 24 layers
        if case["train"]:
            s["grad"] = normal(n, d)
    else:
        sizes = _sizes(case)
        length = sum(-(-n // 128) * 128 for n in sizes)
        flat = torch.zeros(length, device="cuda", dtype=dt)
        flat.normal_(0.0, 1e-3, generator=g)
        pad = torch.ones(length, device="cuda", dtype=torch.bool)
        for t in _views(pad, sizes):
            t.zero_()
        flat.masked_fill_(pad, 0.0)
        out = torch.zeros(length, device="cuda", dtype=DTYPES[case["out"]])
        norm = 1e-3 * math.sqrt(sum(sizes))
        return {"op": "clip", "flat": flat, "grads": _views(flat, sizes), "flat_out": out, "outs": _views(out, sizes),
                "max_norm": norm * (0.31 if case["clips"] else 3.0)}
    s["op"], s["train"], s["leaves"] = case["op"], case["train"], leaves
    if case["train"]:
        for k in leaves:
            s[k].requires_grad_(True)
    return s


def _loss_plain(hidden, weight, targets):
    logits = hidden.float() @ weight.float().t()
    top = logits.detach().amax(dim=1, keepdim=True)
    lse = (logits - top).exp().sum(dim=1).log() + top.squeeze(1)
    keep = targets != IGNORE
    picked = logits.gather(1, targets.clamp(min=0).unsqueeze(1)).squeeze(1)
    return (lse - picked).masked_fill(~keep, 0.0).sum() / keep.sum()


def _ffn_plain(s):
    x = s["x"].float()
    gate, up = x @ s["w_gate"].float().t(), x @ s["w_up"].float().t()
    if "b_gate" in s:
        gate, up = gate + s["b_gate"].float(), up + s["b_up"].float()
    y = (gate / (1.0 + (-gate).exp()) * up) @ s["w_down"].float().t()
    if "b_down" in s:
        y = y + s["b_down"].float()
    y = y * s["scale"]
    if "residual" in s:
        y = y + s["residual"].float()
    return y.to(s["x"].dtype)


def run(s):
    if own:
        import mamba3_b200 as m

    if s["op"] == "clip":
        if own:
            norm = m.clip_grads(s["grads"], s["max_norm"], out=s["outs"])
        else:
            norm = s["flat"].double().square().sum().sqrt()
            scale = (s["max_norm"] / (norm + 1e-6)).clamp(max=1.0)
            s["flat_out"].copy_(s["flat"].float() * scale.float())
            norm = norm.float()
        return norm, s["flat_out"]
    if s["op"] == "loss":
        with torch.set_grad_enabled(s["train"]):
            if own:
                y = m.linear_cross_entropy(s["hidden"], s["weight"], s["targets"], ignore_index=IGNORE)
            else:
                y = _loss_plain(s["hidden"], s["weight"], s["targets"])
    else:
        with torch.set_grad_enabled(s["train"]):
            if own:
                y = m.gated_ffn(s["x"], s["w_gate"], s["w_up"], s["w_down"], b_gate=s.get("b_gate"),
                                b_up=s.get("b_up"), b_down=s.get("b_down"), residual=s.get("residual"),
                                residual_scale=s["scale"])
            else:
                y = _ffn_plain(s)
    if not s["train"]:
        return y
    grads = torch.autograd.grad(y, [s[k] for k in s["leaves"]], s.get("grad"))
    return (y.detach(), *grads)


def work(case):
    b = SIZE[case["dtype"]]
    if case["op"] == "loss":
        # the kept tokens' logits, and their products with the weight and the hidden states in the backward pass
        n, d, v = case["tokens"], case["d"], case["vocab"]
        kept = max(1, round(n * (1 - case["masked"])))
        moved = (kept * d + v * d) * b + n * 8
        return {"bytes": moved + ((n * d + v * d) * b if case["train"] else 0),
                "flops": (6 if case["train"] else 2) * kept * d * v}
    if case["op"] == "ffn":
        n, d, f = case["tokens"], case["d"], case["ff"]
        rows = 2 + (1 if case["residual"] else 0)
        moved = (rows * n * d + 3 * d * f + (2 * f + d if case["bias"] else 0)) * b
        if case["train"]:  # the incoming gradient, and the gradients of the input and the weights
            moved += (2 * n * d + 3 * d * f + (2 * f + d if case["bias"] else 0)) * b
        return {"bytes": moved, "flops": (18 if case["train"] else 6) * n * d * f}
    n = sum(_sizes(case))
    return {"bytes": n * (b + SIZE[case["out"]]), "flops": 3 * n}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "clip":
        total, parts = 0.0, s["flat"].split(1 << 26)
        for p in parts:
            total += float(torch.dot(p.double(), p.double()))
        norm = math.sqrt(total)
        c = min(1.0, s["max_norm"] / (norm + 1e-6))
        return torch.tensor(norm, dtype=torch.float64), torch.cat([p.double() * c for p in parts])
    with torch.no_grad():
        if case["op"] == "loss":
            return _loss_exact(s)
        return _ffn_exact(s)


def _loss_exact(s):
    """loss = 1/n sum_i (lse_i - z_i[t_i]); dL/dz_i = (softmax(z_i) - e_{t_i}) / n, over pieces of the kept tokens."""
    keep = torch.nonzero(s["targets"] != IGNORE).squeeze(1)
    w, n = s["weight"].double(), keep.numel()
    loss = torch.zeros((), dtype=torch.float64, device="cuda")
    dh = torch.zeros(s["hidden"].shape, dtype=torch.float64, device="cuda")
    dw = torch.zeros_like(w)
    for at in keep.split(2048):
        h, t = s["hidden"][at].double(), s["targets"][at]
        z = torch.mm(h, w.t())
        rows = torch.arange(at.numel(), device="cuda")
        lse = torch.logsumexp(z, 1)
        loss += (lse - z[rows, t]).sum()
        if s["train"]:
            z = torch.exp(z - lse[:, None])
            z[rows, t] -= 1.0
            z /= n
            dh[at] = torch.mm(z, w)
            dw.addmm_(z.t(), h)
    return (loss / n, dh, dw) if s["train"] else loss / n


def _ffn_exact(s):
    x, wg, wu, wd = (s[k].double() for k in ("x", "w_gate", "w_up", "w_down"))
    zero = torch.zeros((), dtype=torch.float64, device="cuda")
    bg, bu, bd = (s[k].double() if k in s else zero for k in ("b_gate", "b_up", "b_down"))
    g, u = torch.mm(x, wg.t()) + bg, torch.mm(x, wu.t()) + bu
    sig = torch.sigmoid(g)
    act = g * sig
    y = s["scale"] * (torch.mm(act * u, wd.t()) + bd)
    if "residual" in s:
        y += s["residual"].double()
    if not s["train"]:
        return y
    dz = s["grad"].double() * s["scale"]
    da = torch.mm(dz, wd)
    dg, du = da * u * sig * (1 + g * (1 - sig)), da * act
    grads = {"x": torch.mm(dg, wg) + torch.mm(du, wu), "w_gate": torch.mm(dg.t(), x), "w_up": torch.mm(du.t(), x),
             "w_down": torch.mm(dz.t(), act * u), "residual": s["grad"].double()}
    if "b_gate" in s:
        grads.update(b_gate=dg.sum(0), b_up=du.sum(0), b_down=dz.sum(0))
    return (y, *(grads[k] for k in s["leaves"]))
