"""Attention of a tree of drafted tokens over a static KV cache on an MI355X HIP kernel.

The reference's decode step (src/ferrite/serving/engine.py:89-104, _cache_attention and _write_cache) attends one
token per sequence. Here a step runs up to 64 drafted tokens per sequence, several continuations
at once, over one reading of the cache (csrc/tree.hip: ferrite_internal_tree_attention), and writes their keys
and values behind the committed rows; :mod:`ferrite.kernels.drafts` then accepts and keeps some of them.
"""

from __future__ import annotations

import math

import torch

from ferrite import _hip

MAX_NODES = 64


def tree_attention(q, k_new, v_new, k_cache, v_cache, pos, parents, *, scale: float | None = None):
    """q [B, H, T, D], k_new, v_new [B, Hkv, T, D]; caches [B, Hkv, max_len, D] (updated in place at rows ``pos`` .. ``pos + T - 1``);
    pos int32 [B], parents int32 [B, T], T from 1 to 64, H a multiple of Hkv, D 64, 128 or 256. Returns [B, H, T, D] in q's
    dtype, token-major in memory (``.transpose(1, 2)`` of it is dense).

    Node t of a sequence hangs on node ``parents[b, t]`` < t, or on the committed tokens (-1). It sees the cache's rows
    0 .. pos - 1, its ancestors and itself. A node with any other parent, or that hangs on such a node, is absent (the
    padding of a smaller tree): nothing is written for it, nobody sees it and its output is zero. What a node does not see
    does not touch its output, NaN and infinities included. A sequence whose rows pos .. pos + T - 1 do not lie in the cache
    writes nothing and yields NaN. Scores and softmax are f32. There is no gradient (as for decode_attention). The caches
    must not overlap each other or the memory from the first element of q, k_new or v_new to its last: RuntimeError. B and H are
    at most 65535. q, k_new and v_new are read as they lie where rows are dense and start at 16-byte boundaries, else copied first."""
    if q.ndim != 4 or k_new.ndim != 4 or v_new.shape != k_new.shape or k_new.shape[0] != q.shape[0] \
            or k_new.shape[2:] != q.shape[2:] or k_new.shape[1] < 1 or q.shape[1] < 1 or q.shape[1] % k_new.shape[1]:
        raise ValueError(f"expected q as [B, H, T, D] and k_new, v_new as [B, Hkv, T, D] with H a multiple of Hkv; got "
                         f"{tuple(q.shape)}, {tuple(k_new.shape)}, {tuple(v_new.shape)}")
    b, h, t, d = q.shape
    hkv = k_new.shape[1]
    if not 1 <= t <= MAX_NODES:
        raise ValueError(f"a tree has 1 to {MAX_NODES} nodes; got {t}")
    if k_cache.ndim != 4 or k_cache.shape[:2] != (b, hkv) or k_cache.shape[3] != d or v_cache.shape != k_cache.shape:
        raise ValueError(f"expected caches [B, Hkv, max_len, D] matching k_new; got {tuple(k_cache.shape)}, {tuple(v_cache.shape)}")
    if not (q.dtype == k_new.dtype == v_new.dtype == k_cache.dtype == v_cache.dtype):
        raise ValueError("q, k_new, v_new and the caches must share a dtype")
    if not (k_cache.is_contiguous() and v_cache.is_contiguous()):
        raise ValueError("the caches must be contiguous (they are written in place)")
    if pos.shape != (b,) or parents.shape != (b, t):
        raise ValueError(f"expected pos [B] and parents [B, T]; got {tuple(pos.shape)} and {tuple(parents.shape)}")
    if pos.dtype != torch.int32 or parents.dtype != torch.int32:
        raise ValueError(f"pos and parents must be int32; got {pos.dtype} and {parents.dtype}")
    _hip.dtype_code(q.dtype)
    _hip.require_gpu(q, k_new, v_new, k_cache, v_cache, pos, parents)
    if scale is None:
        scale = 1.0 / math.sqrt(d)
    return _hip.native().tree_attention(q, k_new, v_new, k_cache, v_cache, pos, parents, float(scale))


def ancestors(parents: torch.Tensor) -> torch.Tensor:
    """Truth values [B, T, T]: whether node t sees node s (its ancestors and itself; nothing where t is absent)."""
    lines = []
    for ups in parents.tolist():
        sees = torch.zeros(len(ups), len(ups), dtype=torch.bool)
        for t, up in enumerate(ups):
            if up == -1:
                sees[t, t] = True
            elif 0 <= up < t and sees[up, up]:
                sees[t] = sees[up]
                sees[t, t] = True
        lines.append(sees)
    n = parents.shape[1]
    return (torch.stack(lines) if lines else torch.zeros(0, n, n, dtype=torch.bool)).to(parents.device)


def tree_attention_reference(q, k_new, v_new, k_cache, v_cache, pos, parents, *, scale: float | None = None):
    """The same in torch operations, in f32 (f64 for float64 inputs), sequence by sequence. Not used by the HIP path."""
    b, h, t, d = q.shape
    hkv, length = k_cache.shape[1:3]
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    work = torch.promote_types(q.dtype, torch.float32)
    out = torch.full((b, h, t, d), float("nan"), dtype=q.dtype, device=q.device)
    for i, (p, sees) in enumerate(zip(pos.tolist(), ancestors(parents))):
        if p < 0 or p + t > length:
            continue
        there = sees.diagonal().nonzero()[:, 0]
        k_cache[i, :, p + there] = k_new[i][:, there]
        v_cache[i, :, p + there] = v_new[i][:, there]
        out[i] = 0
        for node in there.tolist():
            rows = torch.cat([torch.arange(p, device=q.device), p + sees[node].nonzero()[:, 0]])
            keys = k_cache[i][:, rows].to(work).repeat_interleave(h // hkv, 0)
            values = v_cache[i][:, rows].to(work).repeat_interleave(h // hkv, 0)
            s = (keys * q[i][:, node, None].to(work)).sum(-1) * scale
            out[i][:, node] = (torch.softmax(s, -1)[..., None] * values).sum(1).to(q.dtype)
    return out
