"""Global gradient norm and clipping over many tensors, for training the
quaternion components or the LoRA factors of a model (hundreds of small
tensors a step): two kernel launches for all of them, nothing read back to the
host."""

from __future__ import annotations

import torch

from .mx import _ext

__all__ = ["clip_grad_norm"]


def clip_grad_norm(parameters, max_norm: float, error_if_nonfinite: bool = False) -> torch.Tensor:
    """Scale the gradients of ``parameters`` in place so that their global
    2-norm is at most ``max_norm``; return the norm before that (a float32
    scalar on their device).

    ``g <- g * min(1, max_norm / (norm + 1e-6))``.  ``parameters`` is a tensor
    or an iterable of tensors on one CUDA device; those without a gradient
    are skipped, one that comes up twice counts once.  Gradients may be
    float32, bfloat16 and float16 side by side; sums are kept in 64 bits in a
    fixed order.  An infinite ``max_norm`` gives the norm and leaves the
    gradients; otherwise a NaN norm makes every gradient NaN and an infinite
    one (past float32's range, too) zero, infinite ones NaN;
    ``error_if_nonfinite`` raises ``RuntimeError`` instead (the host then waits
    for the norm; the gradients are unchanged).  Gradients of different
    parameters must not overlap in memory; one that cannot be written in place
    is refused before any is scaled.
    """
    if isinstance(parameters, torch.Tensor):
        parameters = [parameters]
    return _ext().clip_grad_norm(parameters, float(max_norm), error_if_nonfinite)
