"""The heads of a fused projection on an MI355X HIP kernel: split, and every query and key head
normed (RMS, a weight per element of the head) and rotated by its token's position, in one pass.

The reference splits the projection with transposes (src/ferrite/model/gpt.py:137) and has positions
in a learned table (gpt.py:124-127); it has no norm of the heads and no rotation. The kernel
(csrc/heads_rope.hip) reads the projection once and writes q, k and v as the attention kernels read
them, head-major; the backward kernel writes the projection's gradient in its own layout.
"""

from __future__ import annotations

import torch

from ferrite import _hip

MAX_HEAD_DIM = 512


def rope_tables(length: int, dim: int, *, base: float = 10000.0, device=None):
    """(cos, sin), f32 [length, dim // 2]: of the angle ``p * base ** (-2 i / dim)`` of position p and pair i,
    formed in 64 bits (an f32 angle of position 100,000 is off by up to 0.004)."""
    if dim < 2 or dim % 2 or length < 1:
        raise ValueError(f"expected an even number of rotated elements and at least one position; got {dim}, {length}")
    rate = base ** (-torch.arange(0, dim, 2, dtype=torch.float64, device=device) / dim)
    angle = torch.arange(length, dtype=torch.float64, device=device)[:, None] * rate
    return angle.cos().float(), angle.sin().float()


def _check(qkv, q_weight, k_weight, cos, sin, n_head, n_kv_head, positions) -> None:
    if n_head < 1 or n_kv_head < 1:
        raise ValueError(f"expected at least one query and one key head; got {n_head}, {n_kv_head}")
    if qkv.ndim != 3 or qkv.shape[2] % (n_head + 2 * n_kv_head) or qkv.shape[2] == 0:
        raise ValueError(f"expected qkv as [B, S, (n_head + 2 n_kv_head) * D]; got {tuple(qkv.shape)} for {n_head} query "
                         f"and {n_kv_head} key heads")
    d = qkv.shape[2] // (n_head + 2 * n_kv_head)
    if d % 2 or d > MAX_HEAD_DIM:
        raise ValueError(f"head_dim must be even and at most {MAX_HEAD_DIM}; got {d}")
    if q_weight.shape != (d,) or k_weight.shape != (d,):
        raise ValueError(f"expected weights [{d}]; got {tuple(q_weight.shape)} and {tuple(k_weight.shape)}")
    if q_weight.dtype != k_weight.dtype:
        raise ValueError("the two weights must share a dtype")
    if cos.ndim != 2 or sin.shape != cos.shape or not 1 <= cos.shape[1] <= d // 2 or cos.shape[0] < 1:
        raise ValueError(f"expected cos and sin as [positions, pairs] with 1 to {d // 2} pairs; got {tuple(cos.shape)} and "
                         f"{tuple(sin.shape)}")
    if cos.dtype != torch.float32 or sin.dtype != torch.float32:
        raise ValueError("cos and sin must be float32")
    if cos.requires_grad or sin.requires_grad:
        raise ValueError("the rotation has no gradient for cos and sin")
    if positions is None:
        if qkv.shape[1] > cos.shape[0]:
            raise ValueError(f"sequence {qkv.shape[1]} longer than the tables' {cos.shape[0]} positions")
    else:
        if positions.dtype != torch.int32:
            raise ValueError(f"positions must be int32; got {positions.dtype}")
        if positions.shape not in (qkv.shape[:2], qkv.shape[1:2]):
            raise ValueError(f"expected positions as [B, S] or [S]; got {tuple(positions.shape)} for {tuple(qkv.shape)}")


def qk_norm_rope(qkv, q_weight, k_weight, cos, sin, *, n_head: int, n_kv_head: int | None = None, positions=None,
                 eps: float = 1e-6, interleaved: bool = False):
    """(q [B, n_head, S, D], k, v [B, n_kv_head, S, D]), dense, of the projection ``qkv``
    [B, S, (n_head + 2 n_kv_head) * D] (columns ordered (q|k|v, head, dim), as model/gpt.py:137 splits them;
    ``n_kv_head`` defaults to ``n_head``), float32 or bfloat16.

    Every q and k head is divided by its root mean square (``eps`` added to the mean square) and multiplied by
    ``q_weight`` or ``k_weight`` [D]; then the pairs (i, i + pairs) of its first ``2 * pairs`` elements, or
    (2 i, 2 i + 1) when ``interleaved``, are rotated by the angles whose f32 ``cos`` and ``sin`` [positions,
    pairs] (:func:`rope_tables`) lie at the token's position: ``positions`` int32 [B, S] or [S], else 0..S-1. All of it
    in f32, rounded once. A position outside the tables gives NaN in its q and k rows. Head dims: even, up to 512.

    Differentiable in qkv and the weights, whose gradients are summed in f32 in a fixed order. A captured call that records
    a backward raises RuntimeError while a graph made outside the capture holds one of these as a leaf, and so does any call with a
    forward-mode tangent."""
    n_kv_head = n_head if n_kv_head is None else n_kv_head
    _check(qkv, q_weight, k_weight, cos, sin, n_head, n_kv_head, positions)
    _hip.dtype_code(qkv.dtype)
    _hip.dtype_code(q_weight.dtype)
    _hip.require_gpu(qkv, q_weight, k_weight, cos, sin, *(() if positions is None else (positions,)))
    return _hip.autograd().qk_norm_rope(qkv, q_weight, k_weight, cos, sin, positions, n_head, n_kv_head, float(eps),
                                        bool(interleaved))


def qk_norm_rope_reference(qkv, q_weight, k_weight, cos, sin, *, n_head: int, n_kv_head: int | None = None, positions=None,
                           eps: float = 1e-6, interleaved: bool = False):
    """The same in torch operations, in f32 (f64 for float64 inputs), differentiable. Not used by the HIP path."""
    n_kv_head = n_head if n_kv_head is None else n_kv_head
    b, s, w = qkv.shape
    d, pairs = w // (n_head + 2 * n_kv_head), cos.shape[1]
    work = torch.promote_types(qkv.dtype, torch.float32)
    at = torch.arange(s, device=qkv.device) if positions is None else positions.long()
    c, sn = cos.to(work)[at].unsqueeze(-2), sin.to(work)[at].unsqueeze(-2)  # [(B,) S, 1, pairs]
    x = qkv.reshape(b, s, n_head + 2 * n_kv_head, d)
    q, k, v = x.split([n_head, n_kv_head, n_kv_head], dim=2)

    def rotated(h, weight):
        h = h.to(work)
        u = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + eps) * weight.to(work)
        first = slice(0, 2 * pairs, 2) if interleaved else slice(0, pairs)
        second = slice(1, 2 * pairs, 2) if interleaved else slice(pairs, 2 * pairs)
        lo, hi = u[..., first], u[..., second]
        turned = (lo * c - hi * sn, hi * c + lo * sn)
        turned = torch.stack(turned, -1).flatten(-2) if interleaved else torch.cat(turned, -1)
        return torch.cat([turned, u[..., 2 * pairs:]], -1).to(qkv.dtype).transpose(1, 2)

    return rotated(q, q_weight), rotated(k, k_weight), v.transpose(1, 2)
