"""Clipping of gradients by their global norm on MI355X HIP kernels.

Reference: src/ferrite/model/train.py:59-66, the first lines of adamw_update; :func:`~ferrite.kernels.adamw.fused_adamw_` holds
them for its own update. This is the step by itself, for another optimiser or for a look at the gradients before it
(csrc/clip.hip: ferrite_internal_clip).
"""

from __future__ import annotations

import math

import torch

from ferrite import _hip


def clip_grad_norm_(grads, max_norm: float) -> torch.Tensor:
    """Multiplies every tensor of ``grads`` by ``min(1, max_norm / (norm + 1e-6))`` in place and returns ``norm``, the square root of the
    sum of all their squares, before, as a 0-d f32 device tensor. No step waits for the host.

    ``grads``: float32 and bf16 tensors in any mixture and shape, empty ones too, on one device, each dense in memory (in any order of
    its dimensions); tensors that share memory raise RuntimeError, and so do ones that require a gradient outside of
    ``torch.no_grad()``. ``max_norm`` is 0 or more; ``math.inf`` only measures. Squares are added in 64 bits in a fixed order, the
    products are rounded once. Where the norm is not a finite float (a NaN or infinity among the gradients) they stay as they are."""
    grads = list(grads)
    if not grads:
        raise ValueError("no tensors")
    if not max_norm >= 0:
        raise ValueError(f"max_norm must be 0 or more; got {max_norm}")
    for g in grads:
        _hip.dtype_code(g.dtype)
    _hip.require_gpu(*grads)
    return _hip.native().clip_grad_norm(grads, float(max_norm))


def clip_grad_norm_reference(grads, max_norm: float) -> torch.Tensor:
    """The same in torch operations, in f64. Not used by the HIP path."""
    norm = torch.stack([g.double().square().sum() for g in grads]).sum().sqrt()
    if math.isfinite(float(norm.float())) and float(norm) + 1e-6 > max_norm:
        for g in grads:
            g.copy_(g.double() * (max_norm / (norm + 1e-6)))
    return norm.float()
