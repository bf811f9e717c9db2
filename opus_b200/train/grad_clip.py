"""Gradient clipping by the global norm (the optional clip of the training step, between backward and optimizer).

The call (but for foreach) and the result of torch.nn.utils.clip_grad_norm_, on
the package's kernels: one launch reads every gradient for the norm, one scales them, and
gradients within the bound are not written.
"""
from __future__ import annotations

from collections.abc import Iterable

import torch

from .. import ops


def clip_grad_norm_(parameters: torch.Tensor | Iterable[torch.Tensor], max_norm: float, norm_type: float = 2.0,
                    error_if_nonfinite: bool = False) -> torch.Tensor:
    """Clip the parameters' gradients in place so that their joint norm is at most max_norm; returns the norm they had.

    norm_type is 2 or inf.  Parameters without a gradient are skipped; one
    that is listed twice is refused (it would be scaled twice).
    error_if_nonfinite raises RuntimeError for a NaN or infinite norm and
    leaves the gradients as they are; it is the one case that waits for the
    device.
    """
    parameters = [parameters] if isinstance(parameters, torch.Tensor) else list(parameters)
    grads = [p.grad for p in parameters if p.grad is not None]
    if not error_if_nonfinite:
        return ops.clip_grads(grads, float(max_norm), float(norm_type))
    norm = ops.grad_norm(grads, float(norm_type))
    if not bool(torch.isfinite(norm)):
        raise RuntimeError(f"the gradients' norm of order {norm_type} is not finite, so they cannot be clipped")
    if grads:
        ops.scale_grads(grads, float(max_norm), norm)
    return norm
