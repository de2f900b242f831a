"""Layer norm, with the residual add before it, on MI355X HIP kernels, with gradients.

The reference's model norms by RMS (src/ferrite/kernels/rmsnorm.py); this is the norm of models that centre their
rows and shift them, with :func:`~ferrite.kernels.rmsnorm.rmsnorm`'s interface. Kernels: csrc/layernorm.hip
(ferrite_internal_layernorm, ferrite_internal_layernorm_bwd), launched by csrc/native.cpp.
"""

from __future__ import annotations

import torch

from ferrite import _hip


def layernorm(x, weight, bias=None, *, residual=None, eps: float = 1e-5):
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last axis of ``x`` (float32 or bf16), in x's dtype.

    With ``residual`` given (x's shape and dtype), returns ``(h, y)`` where ``h = x + residual``, rounded to x's dtype, is the new
    residual stream and ``y`` the norm of that ``h``; otherwise returns ``y``. ``weight`` and ``bias`` [dim] share a dtype, float32 or
    bf16, dim is below 2^25. Statistics and sums are f32, those of the parameters' gradients in a fixed order. Differentiable in all
    four, once: a gradient taken with ``create_graph=True`` raises RuntimeError where it is itself differentiated. ``x`` and ``residual``
    get the same gradient tensor. Tensors that are not dense are copied first. A NaN or infinity makes NaN of its own row, and of the
    columns' parameter gradients."""
    if x.ndim < 1 or x.shape[-1] == 0:
        raise RuntimeError("layernorm needs a non-empty last dimension")
    dim = x.shape[-1]
    if weight.shape != (dim,) or bias is not None and bias.shape != (dim,):
        raise ValueError(f"weight and bias must have shape ({dim},), got {tuple(weight.shape)}"
                         + ("" if bias is None else f" and {tuple(bias.shape)}"))
    if bias is not None and bias.dtype != weight.dtype:
        raise ValueError(f"weight and bias must share a dtype; got {weight.dtype} and {bias.dtype}")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype):
        raise ValueError("residual must match x in shape and dtype")
    _hip.dtype_code(x.dtype)
    _hip.dtype_code(weight.dtype)
    _hip.require_gpu(x, weight, x if bias is None else bias, x if residual is None else residual)
    out = _hip.autograd().layernorm(x, weight, bias, residual, float(eps))
    return out[0] if residual is None else (out[0], out[1])


def layernorm_reference(x, weight, bias=None, *, residual=None, eps: float = 1e-5):
    """The same in torch operations, in f32 (f64 for float64 inputs). Not used by the HIP path."""
    work = torch.promote_types(x.dtype, torch.float32)
    h = x if residual is None else (x.to(work) + residual.to(work)).to(x.dtype)
    c = h.to(work) - h.to(work).mean(-1, keepdim=True)
    y = c * torch.rsqrt(c.square().mean(-1, keepdim=True) + eps) * weight.to(work)
    y = (y if bias is None else y + bias.to(work)).to(x.dtype)
    return y if residual is None else (h, y)
