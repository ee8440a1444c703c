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

# The methods themselves, for map(): with hundreds of tensors the host's time is in these calls.
_get_device, _data_ptr, _numel = torch.Tensor.get_device, torch.Tensor.data_ptr, torch.Tensor.numel
_is_contiguous, _dtype = torch.Tensor.is_contiguous, torch.Tensor.dtype.__get__


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


def clip_grads(grads: Iterable[torch.Tensor], max_norm: float, norm_type: float = 2.0,
               out: Optional[Iterable[torch.Tensor]] = None) -> torch.Tensor:
    """Clip `grads` by their global norm; returns the norm before clipping (fp32, on their device).

    grads: dense tensors (fp32, bf16 or fp16, mixed as they come) on one CUDA device, no two of which
    share memory.  Without `out` they are clipped in place, and left unwritten when the norm is within
    max_norm.  With `out` (one tensor for each, of its length and memory order; the dtypes may
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
    every = gs if os is gs else gs + os
    places = set(map(_get_device, every))
    if len(places) != 1 or -1 in places:
        raise _lib.M3bError(f"clip_grads: tensors on one CUDA device expected, got {sorted({str(t.device) for t in every})}")
    dtypes = list(map(_dtype, gs))
    out_dtypes = dtypes if os is gs else list(map(_dtype, os))
    for dt in {*dtypes, *out_dtypes}:
        _lib.dtype_code(dt)
    numel = list(map(_numel, gs))
    if not all(map(_is_contiguous, every)):
        for t in every:
            if not _dense(t):
                raise ValueError(f"clip_grads: dense tensors expected, got strides {t.stride()} of shape {tuple(t.shape)}")
        for g, o in zip(gs, os):
            if not (g.is_contiguous() and o.is_contiguous()) and (g.shape != o.shape or g.stride() != o.stride()):
                raise ValueError("clip_grads: each output needs its gradient's shape and memory order")
    ptrs = list(map(_data_ptr, gs))
    out_ptrs = ptrs
    full = 0 not in numel  # an empty tensor may have any address: it is in nobody's place
    if os is not gs:
        if numel != list(map(_numel, os)):
            raise ValueError("clip_grads: each output needs its gradient's length")
        out_ptrs = list(map(_data_ptr, os))
    written = out_ptrs if full else [p for p, n in zip(out_ptrs, numel) if n]
    places = set(written)
    if len(places) != len(written):
        raise ValueError("clip_grads: the same tensor twice")
    if os is not gs and not places.isdisjoint(ptrs):
        read = set(ptrs if full else (p for p, n in zip(ptrs, numel) if n))
        for n, p, q, a, b in zip(numel, ptrs, out_ptrs, dtypes, out_dtypes):
            if n and p == q and a != b:
                raise ValueError("clip_grads: an output in its gradient's place needs its dtype")
            if n and p != q and q in read:
                raise ValueError("clip_grads: an output in another gradient's place")
    norm = _lib.grad_clip(ptrs, numel, dtypes, out_ptrs, out_dtypes, max_norm, norm_type == math.inf, gs[0].device)
    torch.autograd.graph.increment_version(os)  # written by address: autograd must hear of it
    return norm


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
