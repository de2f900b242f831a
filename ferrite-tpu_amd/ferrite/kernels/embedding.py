"""Lookup of scaled table rows by token on MI355X HIP kernels, with the table's gradient.

Reference: src/ferrite/model/gpt.py:124-127 (``tok_emb[tokens]``) and its autodiff backward. The model's own embedding adds a
position table and has a kernel for vocabularies of up to 1024 tokens; this one takes any vocabulary, and models that scale
their embeddings. Kernels: csrc/embedding.hip (ferrite_internal_embedding, ferrite_internal_embedding_bwd).
"""

from __future__ import annotations

import torch

from ferrite import _hip
from ferrite.kernels._compat import to_torch_dtype


def embedding(tokens, table, *, scale: float = 1.0, padding_idx: int | None = None, dtype=None):
    """``table[tokens] * scale`` [..., dim] in ``dtype`` (default the table's) for int64 or int32 ``tokens`` [...] and a float32 or bf16
    ``table`` [vocab, dim]; the product is f32, rounded once.

    Differentiable in the table, once (RuntimeError where a gradient is differentiated again): equal tokens' rows are added in f32 in
    their order in ``tokens``, cut into pieces by their place among all rows, and rounded once; no atomics, so a call's result is the
    same every time. ``padding_idx`` (from 0 to vocab - 1) is looked up like any token and has no gradient. A token outside the table
    (a negative one too) gives a row of NaN and no gradient.
    Fewer than 2^27 tokens, vocab below 2^31 - 1, dim up to 4194240 (RuntimeError beyond). Tensors that are not dense are copied first."""
    if table.ndim != 2 or table.shape[0] < 1 or table.shape[1] < 1:
        raise ValueError(f"expected a table [vocab, dim]; got {tuple(table.shape)}")
    if tokens.dtype not in (torch.int64, torch.int32):
        raise ValueError(f"tokens must be int64 or int32; got {tokens.dtype}")
    if padding_idx is not None and not 0 <= padding_idx < table.shape[0]:
        raise ValueError(f"padding_idx must be from 0 to {table.shape[0] - 1}; got {padding_idx}")
    dtype = table.dtype if dtype is None else to_torch_dtype(dtype)
    _hip.dtype_code(table.dtype)
    _hip.dtype_code(dtype)
    _hip.require_gpu(tokens, table)
    return _hip.autograd().embedding(tokens, table, float(scale), -1 if padding_idx is None else int(padding_idx), dtype,
                                      False)


def embedding_reference(tokens, table, *, scale: float = 1.0, padding_idx: int | None = None, dtype=None):
    """The same in torch operations, in f32 (f64 for a float64 table), for tokens inside the table or not. Not used by the HIP path."""
    work = torch.promote_types(table.dtype, torch.float32)
    inside = (tokens >= 0) & (tokens < table.shape[0])
    rows = table.to(work)[torch.where(inside, tokens, 0).long()] * scale
    if padding_idx is not None:
        rows = torch.where((tokens == padding_idx)[..., None], rows.detach(), rows)
    rows = torch.where(inside[..., None], rows, torch.full_like(rows, float("nan")))
    return rows.to(table.dtype if dtype is None else to_torch_dtype(dtype))
