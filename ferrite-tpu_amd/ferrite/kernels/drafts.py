"""What follows a drafted step's attention, on MI355X HIP kernels: the drafted tokens that the model
itself would have taken, and the cache's rows of those put in order.

The reference's serving takes one token a step (src/ferrite/serving/engine.py:107-131, :181-203: argmax of the
step's logits); it drafts nothing. Here a step runs a tree of up to 64 drafted tokens per sequence:
:func:`~ferrite.kernels.tree_attention.tree_attention` attends it over the cache, :func:`accept_drafts`
walks it along the model's own choices, and :func:`compact_cache` moves the visited nodes' rows. Greedy
decoding of one token after another gives the same tokens. No step waits for the host, and all three
can be captured.
"""

from __future__ import annotations

import torch

from ferrite import _hip

MAX_NODES = 64


def _check_ints(name: str, t: torch.Tensor, shape, dtypes=(torch.int32,)) -> None:
    if t.shape != shape:
        raise ValueError(f"expected {name} as {list(shape)}; got {tuple(t.shape)}")
    if t.dtype not in dtypes:
        raise ValueError(f"{name} must be {' or '.join(str(d).replace('torch.', '') for d in dtypes)}; got {t.dtype}")


def accept_drafts(logits, tokens, parents):
    """(path int32 [B, T], count int32 [B], next_token int64 [B]) for the logits [B, T, V] of T drafted nodes (1 to 64) that
    hold ``tokens`` [B, T] and hang on ``parents`` int32 [B, T].

    Node 0 is the token that a sequence already has (parent -1). From it the walk goes to the child whose
    token is the argmax of the node's logits (of equal logits the lowest token, NaN above all, as
    torch.argmax; of equal children the lowest node) until there is none: ``path`` are the ``count`` nodes visited, -1
    behind them, and ``next_token`` the argmax at the last, which no draft held. A node whose parent is not -1 or an earlier
    node is absent: its logits are not read. Where node 0 is absent nothing is accepted: count 0, next_token -1. Logits that are
    not dense (a slice of a padded vocabulary) are copied first."""
    if logits.ndim != 3 or not 1 <= logits.shape[1] <= MAX_NODES or logits.shape[2] < 1:
        raise ValueError(f"expected logits as [B, T, V] with 1 to {MAX_NODES} nodes; got {tuple(logits.shape)}")
    _check_ints("tokens", tokens, logits.shape[:2], (torch.int64, torch.int32))
    _check_ints("parents", parents, logits.shape[:2])
    _hip.dtype_code(logits.dtype)
    _hip.require_gpu(logits, tokens, parents)
    return _hip.native().accept_drafts(logits, tokens, parents)


def compact_cache(k_cache, v_cache, pos, path, count) -> None:
    """Moves cache rows ``pos[b] + path[b, i]`` to ``pos[b] + i`` for i < ``count[b]``, in place, in every layer and head of the
    caches [B, H, max_len, D] or [layers, B, H, max_len, D]; pos [B], path [B, T] (1 to 64 entries) and count [B] are int32.

    A path goes up (path[b, i] > path[b, i - 1], from 0), as :func:`accept_drafts` gives it, so all rows move as if each were read
    before any was written. It ends at the first entry that does not, or whose row lies outside the cache; rows
    behind it stay as they are. Caches that overlap raise RuntimeError. Layers, B and H are at most 65535."""
    if k_cache.ndim not in (4, 5) or v_cache.shape != k_cache.shape:
        raise ValueError(f"expected caches [B, H, max_len, D] or [layers, B, H, max_len, D] of one shape; got "
                         f"{tuple(k_cache.shape)} and {tuple(v_cache.shape)}")
    if v_cache.dtype != k_cache.dtype:
        raise ValueError("the caches must share a dtype")
    if not (k_cache.is_contiguous() and v_cache.is_contiguous()):
        raise ValueError("the caches must be contiguous (they are written in place)")
    b = k_cache.shape[-4]
    if path.ndim != 2 or not 1 <= path.shape[1] <= MAX_NODES:
        raise ValueError(f"expected path as [B, T] with 1 to {MAX_NODES} entries; got {tuple(path.shape)}")
    _check_ints("path", path, (b, path.shape[1]))
    _check_ints("pos", pos, (b,))
    _check_ints("count", count, (b,))
    _hip.dtype_code(k_cache.dtype)
    _hip.require_gpu(k_cache, v_cache, pos, path, count)
    _hip.native().compact_cache(k_cache, v_cache, pos, path, count)


def accept_drafts_reference(logits, tokens, parents):
    """The same walk in Python over host copies."""
    wanted = torch.argmax(logits, dim=-1).tolist()
    paths, counts, following = [], [], []
    for want, toks, ups in zip(wanted, tokens.tolist(), parents.tolist()):
        path = [0] if ups[0] == -1 else []
        while path:
            at = path[-1]
            child = next((j for j in range(at + 1, len(ups)) if ups[j] == at and toks[j] == want[at]), None)
            if child is None:
                break
            path.append(child)
        paths.append(path + [-1] * (len(ups) - len(path)))
        counts.append(len(path))
        following.append(want[path[-1]] if path else -1)
    dev = logits.device
    shape = tuple(parents.shape)
    return (torch.tensor(paths, dtype=torch.int32, device=dev).reshape(shape),
            torch.tensor(counts, dtype=torch.int32, device=dev), torch.tensor(following, dtype=torch.int64, device=dev))


def compact_cache_reference(k_cache, v_cache, pos, path, count) -> None:
    """The same moves with torch indexing, in place."""
    for b, (p, line, n) in enumerate(zip(pos.tolist(), path.tolist(), count.tolist())):
        rows, last = [], -1
        for r in line[:max(n, 0)]:
            if p < 0 or r <= last or p + r >= k_cache.shape[-2]:
                break
            rows.append(p + r)
            last = r
        for c in (k_cache, v_cache):
            c.select(-4, b)[..., p:p + len(rows), :] = c.select(-4, b)[..., rows, :] if rows else c.select(-4, b)[..., :0, :]
