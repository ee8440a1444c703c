"""The gated feed-forward block as one operator, forward and backward (``gated_ffn``).

    out = residual + residual_scale * (silu(x Wg^T + bg) * (x Wu^T + bu)) Wd^T + bd scaled alike

It is the blocks' SwiGLU (mamba3/block.py:16-26) with the scaled residual that follows it
(mamba3/block.py:79-107): both projections, the activation and the product are one kernel, the down
projection with bias and residual another; single tokens, decode batches and long prompts run the
same call.  ``SwiGLU(..., fused=True)``, ``KulaMambaBlock`` / ``KulaMambaLM(..., fused_mlp=True)``
run their MLP through it.
"""

from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import _lib, ops


class _GatedFfn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_gate, w_up, w_down, b_gate, b_up, b_down, residual, scale):
        out, act, gu = ops.gated_ffn_fwd(x, w_gate, w_up, w_down, b_gate, b_up, b_down, residual, scale, True)
        ctx.save_for_backward(x, w_gate, w_up, w_down, b_gate, b_up, b_down, act, gu)
        ctx.scale = scale
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        x, w_gate, w_up, w_down, b_gate, b_up, b_down, act, gu = ctx.saved_tensors
        want = ctx.needs_input_grad
        grads = [None] * 7
        if any(want[:7]):
            grads = ops.gated_ffn_bwd(x, w_gate, w_up, w_down, b_gate, b_up, b_down, ctx.scale, act, gu,
                                      _lib._rows2d(dout, x.shape[1]), list(want[:7]))
        return (*grads, dout if want[7] else None, None)


def gated_ffn(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, w_down: torch.Tensor, *,
              b_gate: torch.Tensor | None = None, b_up: torch.Tensor | None = None,
              b_down: torch.Tensor | None = None, residual: torch.Tensor | None = None,
              residual_scale: float = 1.0) -> torch.Tensor:
    """residual + residual_scale * (act w_down^T + b_down), act = silu(x w_gate^T + b_gate) * (x w_up^T + b_up).

    x (..., d_model); w_gate, w_up (d_ff, d_model); w_down (d_model, d_ff), as nn.Linear stores them;
    b_gate and b_up (d_ff) come together, b_down (d_model) on its own; residual has x's shape.  All of
    one dtype (fp32, bf16 or fp16) on one CUDA device; under autocast every argument is cast to the
    autocast dtype first.  Any sizes and strides: operands that the copies cannot read in place
    (widths that are no multiple of 8, a last dimension with a stride, fp32) are laid out once per
    call.  Differentiable in every tensor argument; sums in fp32, and the activation (forward) and its
    two factors' gradients (backward) rounded to a 16-bit dtype once, as operands of the next products
    (fp16: relative to the largest incoming gradient, so that small ones keep their bits)."""
    if x.is_cuda and torch.is_autocast_enabled("cuda"):
        dt = torch.get_autocast_dtype("cuda")
        x, w_gate, w_up, w_down, b_gate, b_up, b_down, residual = [
            t if t is None or t.dtype == dt else t.to(dt)
            for t in (x, w_gate, w_up, w_down, b_gate, b_up, b_down, residual)]
    ts = [t for t in (x, w_gate, w_up, w_down, b_gate, b_up, b_down, residual) if t is not None]
    _lib._same_gpu("gated_ffn", ts)
    _lib._no_tangent("gated_ffn", ts)
    dt = x.dtype
    for t in ts:
        if t.dtype != dt:
            raise _lib.M3bError(f"gated_ffn: one dtype expected, got {[t.dtype for t in ts]}")
    _lib.dtype_code(dt)
    if x.dim() < 1 or w_gate.dim() != 2:
        raise ValueError("gated_ffn: x (..., d_model) and w_gate (d_ff, d_model) expected")
    f, d = w_gate.shape
    if x.shape[-1] != d or w_up.shape != (f, d) or w_down.shape != (d, f):
        raise ValueError(f"gated_ffn: x (..., {d}), w_up ({f}, {d}) and w_down ({d}, {f}) expected, got "
                         f"{tuple(x.shape)}, {tuple(w_up.shape)} and {tuple(w_down.shape)}")
    if d == 0 or f == 0:
        raise ValueError("gated_ffn: d_model and d_ff must be positive")
    if (b_gate is None) != (b_up is None):
        raise ValueError("gated_ffn: b_gate and b_up go together")
    if len(ts) > 4:
        for name, b, n in (("b_gate", b_gate, f), ("b_up", b_up, f), ("b_down", b_down, d)):
            if b is not None:
                if b.shape != (n,):
                    raise ValueError(f"gated_ffn: {name} ({n},) expected, got {tuple(b.shape)}")
        b_gate, b_up, b_down = [b if b is None else b.contiguous() for b in (b_gate, b_up, b_down)]
        if residual is not None and residual.shape != x.shape:
            raise ValueError(f"gated_ffn: residual must have x's shape {tuple(x.shape)}, got {tuple(residual.shape)}")
    x2 = _lib._rows2d(x, d)
    r2 = None if residual is None else _lib._rows2d(residual, d)
    w_gate, w_up, w_down = w_gate.contiguous(), w_up.contiguous(), w_down.contiguous()
    scale = float(residual_scale)
    if torch.is_grad_enabled() and any([t.requires_grad for t in ts]):
        args = [x2, w_gate, w_up, w_down, b_gate, b_up, b_down, r2]
        if torch.compiler.is_compiling():
            # one tensor in two places (x as its own residual) is one argument to the tracer, which then
            # loses one of its two gradients: views keep them apart
            args = [None if t is None else t.view(t.shape) for t in args]
        y = _GatedFfn.apply(*args, scale)
    else:
        y = ops.gated_ffn_fwd(x2, w_gate, w_up, w_down, b_gate, b_up, b_down, r2, scale, False)[0]
    return y if y.dim() == x.dim() else y.view(x.shape)
