"""Norm of the gradients of many parameters and clipping by it: one pass over the gradients for the norm, a second, which
returns at once below the limit, for the scaling; two launches for up to 1024 tensors of mixed types.  The reference has no
counterpart (CAME clips per tensor inside the step); `AdamW(max_grad_norm=...)` clips without the second pass."""
from __future__ import annotations

import math

import torch

from . import _host

_DTYPES = (torch.float32, torch.float16, torch.bfloat16)


def clip_grad_norm_(parameters, max_norm: float, norm_type: float = 2.0, error_if_nonfinite: bool = False) -> torch.Tensor:
    """Multiplies the gradients of `parameters` (a tensor or an iterable of tensors) in place by
    min(1, max_norm / (N + 1e-6)), N the 2-norm of all of them together, and returns N as a 0-dimensional fp32 tensor on
    their device, without waiting for it.  What `torch.nn.utils.clip_grad_norm_` does, sums in 64 bits; max_norm = inf leaves
    the gradients alone and gives N.  Gradients: float32, float16, bfloat16 (mixed if need be), any strides, all on one
    CUDA device, each listed once.  `error_if_nonfinite` waits for N and raises before anything is scaled."""
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError(f"max_norm must be >= 0, got {max_norm}")
    if float(norm_type) != 2.0:
        raise ValueError(f"came_b200 clips by the 2-norm, got norm_type={norm_type}")
    params = [parameters] if isinstance(parameters, torch.Tensor) else list(parameters)
    if error_if_nonfinite:
        norm = _clip(params, math.inf)
        if not math.isfinite(norm.item()):
            raise RuntimeError(f"the norm of the gradients is {norm.item()}, so that they cannot be clipped")
    return _clip(params, max_norm)


def _clip(params, max_norm):
    norm = _host.clip_grad_norm(params, max_norm, True)
    if norm is not None:
        return norm
    # something out of the ordinary: no gradients, strides with gaps, or what is refused
    grads = [p.grad for p in params if p.grad is not None]
    if not grads:
        return torch.zeros(())
    for g in grads:
        if g.layout != torch.strided:
            raise RuntimeError("clip_grad_norm_ does not support sparse gradients")
        if not g.is_cuda:
            raise RuntimeError(f"came_b200 clips CUDA tensors only (there is no CPU fallback); got a gradient on {g.device}")
        if g.device != grads[0].device:
            raise RuntimeError(f"clip_grad_norm_ needs all gradients on one device, got {grads[0].device} and {g.device}")
        if g.dtype not in _DTYPES:
            raise RuntimeError(f"came_b200 supports float32/float16/bfloat16 gradients, got {g.dtype}")
    full = [g for g in grads if g.numel()]
    if len({g.data_ptr() for g in full}) != len(full):
        raise ValueError("clip_grad_norm_: a gradient is listed twice")
    copies = [g.detach().contiguous() for g in grads]
    norm = _host.clip_grad_norm(copies, max_norm, False)
    if norm is None:
        raise RuntimeError("clip_grad_norm_: these gradients cannot be clipped")
    if not math.isinf(max_norm):
        for g, c in zip(grads, copies):
            if c.data_ptr() != g.data_ptr():
                g.detach().copy_(c)
    return norm
