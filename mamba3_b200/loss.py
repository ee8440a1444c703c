"""The language-model loss from the final hidden states (``linear_cross_entropy``).

KulaMambaLM's loss (mamba3/block.py:186-193) without the (tokens, vocab) logits: they are formed a
tile at a time on the tensor cores and reduced on the spot, and again in the backward pass, a piece
of the vocabulary at a time.  ``KulaMambaLM.forward(ids, labels, return_logits=False)`` runs it.
"""

from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import _lib, ops


class _LinearXent(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, target, ignore_index, reduction):
        loss, saved = ops.linear_xent_fwd(hidden, weight, target, ignore_index, reduction, True)
        ctx.save_for_backward(weight, saved)
        ctx.cfg = (hidden.shape[0], ignore_index, reduction)
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, dloss):
        weight, saved = ctx.saved_tensors
        rows, ignore_index, reduction = ctx.cfg
        dh, dw = ops.linear_xent_bwd(rows, weight, saved, dloss.float().contiguous(), ignore_index, reduction,
                                     ctx.needs_input_grad[0], ctx.needs_input_grad[1])
        return dh, dw, None, None, None


def linear_cross_entropy(hidden: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor, *,
                         ignore_index: int = -100, reduction: str = "mean") -> torch.Tensor:
    """Cross entropy of softmax(hidden weight^T) against `targets`, in fp32.

    hidden (..., d_model), weight (vocab, d_model), targets: integers of hidden's leading shape.
    Tokens whose target is `ignore_index` are left out: they cost no products, what their hidden
    states hold (NaN included) reaches no sum, and their gradient is zero.  reduction "mean" (over
    the kept tokens; NaN when there is none, with zero gradients), "sum", or "none" (the leading
    shape, 0 at ignored tokens).  hidden and weight share a dtype (fp32, bf16 or fp16); under
    autocast both are cast to the autocast dtype.  Differentiable in both.  The loss is fp32 in
    every dtype.  A target outside the vocabulary makes the loss and the gradients NaN and is
    reported by ``check_device_errors()``."""
    if hidden.is_cuda and torch.is_autocast_enabled("cuda"):
        dt = torch.get_autocast_dtype("cuda")
        hidden, weight = hidden.to(dt), weight.to(dt)
    _lib._same_gpu("linear_cross_entropy", (hidden, weight, targets))
    _lib._no_tangent("linear_cross_entropy", (hidden, weight))
    if hidden.dtype != weight.dtype:
        raise _lib.M3bError(f"linear_cross_entropy: one dtype expected, got {hidden.dtype} and {weight.dtype}")
    _lib.dtype_code(hidden.dtype)
    if reduction not in _lib.REDUCTIONS:
        raise ValueError(f"linear_cross_entropy: reduction 'mean', 'sum' or 'none', got {reduction!r}")
    if weight.dim() != 2 or hidden.dim() < 1 or hidden.shape[-1] != weight.shape[1]:
        raise ValueError(f"linear_cross_entropy: hidden (..., d_model) and weight (vocab, d_model) expected, got "
                         f"{tuple(hidden.shape)} and {tuple(weight.shape)}")
    if weight.shape[0] == 0 or weight.shape[1] == 0:
        raise ValueError("linear_cross_entropy: vocab and d_model must be positive")
    if targets.shape != hidden.shape[:-1]:
        raise ValueError(f"linear_cross_entropy: targets {tuple(hidden.shape[:-1])} expected, got {tuple(targets.shape)}")
    if targets.dtype not in (torch.int64, torch.int32, torch.int16, torch.uint8, torch.int8):
        raise ValueError(f"linear_cross_entropy: integer targets expected, got {targets.dtype}")
    h2 = _lib._rows2d(hidden, weight.shape[1])
    t1 = targets if targets.dim() == 1 else targets.reshape(-1)
    if t1.dtype != torch.int64:
        t1 = t1.to(torch.int64)
    t1 = t1.contiguous()
    w = weight.contiguous()
    if torch.is_grad_enabled() and (hidden.requires_grad or weight.requires_grad):
        loss = _LinearXent.apply(h2, w, t1, int(ignore_index), reduction)
    else:
        loss = ops.linear_xent_fwd(h2, w, t1, int(ignore_index), reduction, False)[0]
    return loss.view(targets.shape) if reduction == "none" else loss
