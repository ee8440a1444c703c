"""Global gradient norm and clipping over many tensors (``clip_grads``, ``clip_grad_norm_``).

    norm = (sum_i |g_i|^2)^(1/2);  out_i = g_i * min(1, max_norm / (norm + 1e-6))

The rule of torch.nn.utils.clip_grad_norm_, in two passes over all gradients at once: no launch per
tensor, no host synchronisation, the norm in fp32 or better whatever the gradients' types.
"""

from __future__ import annotations

import math
from typing import Iterable, Optional

import torch

from . import _lib


def _dense(t):
    """True when t's elements fill one run of memory in some order."""
    if t.is_contiguous():
        return True
    want = 1
    for size, stride in sorted(((n, s) for n, s in zip(t.shape, t.stride()) if n != 1), key=lambda x: x[1]):
        if stride != want:
            return False
        want *= size
    return True


@torch.no_grad()
def clip_grads(grads: Iterable[torch.Tensor], max_norm: float, norm_type: float = 2.0,
               out: Optional[Iterable[torch.Tensor]] = None) -> torch.Tensor:
    """Clip `grads` by their global norm; returns the norm before clipping (fp32, on their device).

    grads: dense tensors (fp32, bf16 or fp16, mixed as they come) on one CUDA device, no two of which
    share memory.  Without `out` they are clipped in place, and left unwritten when the norm is within
    max_norm.  With `out` (one tensor for each, of its shape and memory order; the dtypes may
    differ: the fp32 main gradients of a bf16 model, say) the clipped values go there.  max_norm may
    be math.inf (copies, or only the norm).  norm_type 2 or inf.  A norm that is not finite
    spreads as torch's rule has it: NaN makes every value NaN, infinity makes them 0 (inf itself NaN)."""
    gs = [grads] if isinstance(grads, torch.Tensor) else list(grads)
    if norm_type not in (2, 2.0, math.inf):
        raise ValueError(f"clip_grads: norm_type 2 or inf, got {norm_type}")
    max_norm = float(max_norm)
    if math.isnan(max_norm) or max_norm < 0:
        raise ValueError(f"clip_grads: max_norm must not be negative, got {max_norm}")
    os = gs if out is None else ([out] if isinstance(out, torch.Tensor) else list(out))
    if len(os) != len(gs):
        raise ValueError(f"clip_grads: {len(gs)} gradients and {len(os)} outputs")
    if not gs:
        return torch.zeros(())
    dev = gs[0].device
    for t in gs if out is None else gs + os:
        if t.device != dev or not t.is_cuda:
            raise _lib.M3bError(f"clip_grads: tensors on one CUDA device expected, got {dev} and {t.device}")
        if t.dtype not in _lib._DT:
            raise _lib.M3bError(f"unsupported dtype {t.dtype}")
        if not _dense(t):
            raise ValueError(f"clip_grads: dense tensors expected, got strides {t.stride()} of shape {tuple(t.shape)}")
    if out is not None:
        for g, o in zip(gs, os):
            if g.shape != o.shape or (g.stride() != o.stride() and not (g.is_contiguous() and o.is_contiguous())):
                raise ValueError("clip_grads: each output needs its gradient's shape and memory order")
            if g.numel() and g.data_ptr() == o.data_ptr() and g.dtype != o.dtype:
                raise ValueError("clip_grads: an output in its gradient's place needs its dtype")
    ptrs = [t.data_ptr() for t in os if t.numel()]
    if len(set(ptrs)) != len(ptrs):
        raise ValueError("clip_grads: the same tensor twice")
    return _lib.grad_clip(gs, os, max_norm, norm_type == math.inf, dev)


def clip_grad_norm_(parameters, max_norm: float, norm_type: float = 2.0,
                    error_if_nonfinite: bool = False) -> torch.Tensor:
    """torch.nn.utils.clip_grad_norm_ on `clip_grads`: clips the parameters' .grad in place and
    returns the norm.  error_if_nonfinite reads the norm on the host, after the gradients were
    clipped, and raises if it is not finite."""
    ps = [parameters] if isinstance(parameters, torch.Tensor) else list(parameters)
    grads = [p.grad for p in ps if p.grad is not None]
    if any(g.is_sparse for g in grads):
        raise ValueError("clip_grad_norm_: sparse gradients are not supported")
    norm = clip_grads(grads, max_norm, norm_type)
    if error_if_nonfinite and not math.isfinite(norm.item()):
        raise RuntimeError(f"The total norm of order {norm_type} for gradients from `parameters` is not finite")
    return norm
