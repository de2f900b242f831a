"""The operators of a drafted step over the key-value cache, and the rotated heads that it and training
read: their plain forms in elementary torch operations, the calls of the library's kernels, and the cases
by which the two are measured.

    own                 False: `run` computes the plain forms; True: it calls the library
    listed()            the fixed cases
    draw(rng)           one more case from the same ranges
    prepare(case, seed) what a program has in hand before the call
    run(state)          one pass; returns its outputs
    work(case)          bytes and operations one pass cannot do without
    exact(case, seed)   the same outputs in 64 bits
"""

from __future__ import annotations

import math
import os
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
SIZE = {"bf16": 2, "f32": 4}
EPS = 1e-6


_calls = None


def _library():
    """The library's entry points, imported where its own kernels run, once."""
    global _calls
    if _calls is None:
        pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ferrite-tpu_amd")
        if pkg not in sys.path:
            sys.path.insert(0, pkg)
        from ferrite.kernels import drafts, qk_norm_rope, tree_attention

        _calls = (qk_norm_rope.qk_norm_rope, tree_attention.tree_attention, drafts.accept_drafts, drafts.compact_cache)
    return _calls


# ---------------------------------------------------------------- cases


def listed() -> list[dict]:
    return [
        # The heads of one decode token of the default model: the smallest call, one launch.
        _norm("norm_decode", 1, 1, 4, 4, 128, 128, "bf16", False, grad=False, positions=True),
        # The heads of a training step's layer (12 heads of 64, batch 8 x 1024), forward and backward.
        _norm("norm_train", 8, 1024, 12, 12, 64, 64, "bf16", False, grad=True, positions=False),
        # Prefill of one long prompt of ragged length with shared key heads.
        _norm("norm_prefill", 1, 8191, 32, 8, 128, 128, "bf16", False, grad=False, positions=False),
        # Training in float32: odd sizes, a head dim that fits no power of two, half of it rotated in adjacent pairs.
        _norm("norm_f32", 3, 1001, 5, 5, 80, 40, "f32", True, grad=True, positions=False),
        # A small tree over the serving default's cache for one user: latency.
        _tree("tree_small", 1, 4, 4, 8, 512, 128, "bf16", ragged=False),
        # Four drafts per sequence over the cache of the decode benchmark: the cache's bytes count.
        _tree("tree_long", 8, 32, 32, 4, 8192, 128, "bf16", ragged=False),
        # Wide trees of unequal sizes over shared key heads: 256 query rows for each cached row.
        _tree("tree_wide", 16, 32, 8, 64, 4096, 128, "bf16", ragged=True),
        # float32, ragged lengths, three query heads to a key head.
        _tree("tree_f32", 3, 6, 2, 13, 3001, 64, "f32", ragged=True),
        # Accepting a small draft over the byte vocabulary: latency.
        {"name": "accept_bytes", "kind": "accept", "b": 1, "t": 8, "v": 256, "dtype": "f32", "ragged": False},
        # A batch of trees over a large vocabulary of odd size.
        {"name": "accept_batch", "kind": "accept", "b": 16, "t": 32, "v": 50257, "dtype": "f32", "ragged": True},
        # The accepted rows of one user's tree, four layers.
        {"name": "compact_small", "kind": "compact", "layers": 4, "b": 1, "h": 4, "t": 8, "len": 512, "d": 128,
         "dtype": "bf16"},
        # The accepted rows of a batch in all layers of the 12-layer model.
        {"name": "compact_batch", "kind": "compact", "layers": 12, "b": 32, "h": 12, "t": 24, "len": 1024, "d": 64,
         "dtype": "bf16"},
    ]


def _norm(name, b, s, h, hkv, d, rot, dtype, interleaved, grad, positions) -> dict:
    return {"name": name, "kind": "norm", "b": b, "s": s, "h": h, "hkv": hkv, "d": d, "rot": rot, "dtype": dtype,
            "interleaved": interleaved, "grad": grad, "positions": positions}


def _tree(name, b, h, hkv, t, length, d, dtype, ragged) -> dict:
    return {"name": name, "kind": "tree", "b": b, "h": h, "hkv": hkv, "t": t, "len": length, "d": d, "dtype": dtype,
            "ragged": ragged}


def _log_int(rng, lo: int, hi: int) -> int:
    """An integer of [lo, hi], even over its logarithm."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng) -> dict:
    kind = rng.choice(["norm", "norm", "tree", "tree", "tree", "accept", "compact"])
    while True:
        case = globals()["_draw_" + kind](rng)
        case.pop("name", None)
        w = work(case)
        # No more than the largest listed cases; float32 products run at a sixteenth of bf16's rate.
        if w["bytes"] <= 6.7e8 and w["flops"] * (16 if case["dtype"] == "f32" else 1) <= 3.4e10 and _held(case) <= 1 << 31:
            return case


def _heads(rng) -> tuple[int, int]:
    hkv = _log_int(rng, 1, 16)
    return hkv * rng.choice([1, 1, 2, 3, 4, 8]), hkv


def _draw_norm(rng) -> dict:
    h, hkv = _heads(rng)
    d = rng.choice([32, 48, 64, 64, 80, 96, 128, 128, 128, 200, 256])
    rot = rng.choice([d, d, d, d // 4 * 2])
    s = 1 if rng.random() < 0.25 else _log_int(rng, 2, 8192)
    return _norm("", _log_int(rng, 1, 64), s, h, hkv, d, rot, "bf16" if rng.random() < 0.75 else "f32", rng.random() < 0.25,
                 grad=rng.random() < 0.5 and s > 1, positions=s == 1 or rng.random() < 0.3)


def _draw_tree(rng) -> dict:
    h, hkv = _heads(rng)
    t = _log_int(rng, 1, 64)
    return _tree("", _log_int(rng, 1, 32), h, hkv, t, _log_int(rng, 128, 16384), rng.choice([64, 128, 128, 256]),
                 "bf16" if rng.random() < 0.75 else "f32", ragged=rng.random() < 0.5)


def _draw_accept(rng) -> dict:
    return {"kind": "accept", "b": _log_int(rng, 1, 64), "t": _log_int(rng, 1, 64), "v": _log_int(rng, 100, 131072),
            "dtype": "f32" if rng.random() < 0.75 else "bf16", "ragged": rng.random() < 0.5}


def _draw_compact(rng) -> dict:
    t = _log_int(rng, 4, 64)
    return {"kind": "compact", "layers": _log_int(rng, 1, 32), "b": _log_int(rng, 1, 32), "h": _log_int(rng, 1, 16), "t": t,
            "len": _log_int(rng, 2 * t, 4096), "d": rng.choice([64, 128, 128, 256]),
            "dtype": "bf16" if rng.random() < 0.75 else "f32"}


def _held(case) -> int:
    """Bytes of a state's largest part."""
    if case["kind"] in ("tree", "compact"):
        return 2 * case.get("layers", 1) * case["b"] * case.get("hkv", case.get("h")) * case["len"] * case["d"] * SIZE[case["dtype"]]
    return 0


# ---------------------------------------------------------------- state


def _positions(case) -> list[int]:
    """Committed rows of each sequence: spread from a quarter of what the cache holds beside the drafts to all of it."""
    most = case["len"] - case["t"]
    return [most - (most * 3 // 4) * i // max(1, case["b"] - 1) for i in range(case["b"])]


def _nodes(case) -> list[int]:
    """Nodes of each sequence's tree: all, or spread from half of them up."""
    t, b = case["t"], case["b"]
    return [t - (t // 2) * i // max(1, b - 1) if case["ragged"] else t for i in range(b)]


def _counts(case) -> list[int]:
    """Accepted nodes of each sequence: from one to half of the drafted."""
    return [1 + i % (case["t"] // 2) if case["b"] > 1 else case["t"] // 2 for i in range(case["b"])]


def _trees(case, g):
    """Parents [B, T]: node 0 is the pending token, every other node hangs on one of the eight before it; nodes past a
    sequence's own number are absent (-2)."""
    b, t = case["b"], case["t"]
    sizes = torch.tensor(_nodes(case))[torch.randperm(b, generator=g)]
    idx = torch.arange(t)
    back = 1 + (torch.rand(b, t, generator=g).square() * idx.clamp(max=8)).long()
    parents = torch.where(idx > 0, (idx - back).clamp(min=0), -1)
    return torch.where(idx < sizes[:, None], parents, -2).int()


def prepare(case, seed):
    dev = torch.device("cuda:0")
    host = torch.Generator().manual_seed(seed)
    gen = torch.Generator(dev).manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape, dtype=dt, scale=1.0, loc=0.0):
        return torch.randn(*shape, generator=gen, device=dev, dtype=torch.float32).mul_(scale).add_(loc).to(dtype)

    if case["kind"] == "norm":
        b, s, h, hkv, d, rot = (case[k] for k in ("b", "s", "h", "hkv", "d", "rot"))
        rows = s if not case["positions"] else 8192 + s
        angle = (torch.arange(rows, dtype=torch.float64, device=dev)[:, None]
                 * 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=dev) / rot))
        st = {"case": case, "qkv": normal(b, s, (h + 2 * hkv) * d), "wq": normal(d, dtype=torch.float32, scale=0.1, loc=1.0),
              "wk": normal(d, dtype=torch.float32, scale=0.1, loc=1.0), "cos": angle.cos().float(), "sin": angle.sin().float(),
              "pos": None}
        if case["positions"]:  # sequences that stand at places of their own
            first = torch.randint(0, 8192, (b, 1), generator=host)
            st["pos"] = (first + torch.arange(s)).int().to(dev)
        if case["grad"]:
            st["leaves"] = [st[k].requires_grad_() for k in ("qkv", "wq", "wk")]
            st["grads"] = [normal(b, n, s, d) for n in (h, hkv, hkv)]
        return st
    if case["kind"] == "accept":
        b, t, v = case["b"], case["t"], case["v"]
        parents = _trees(case, host).to(dev)
        logits = normal(b, t, v, scale=2.0)
        # Drafts: two in three hold the token that the model wants after their parent.
        wanted = _first_max(logits).gather(1, parents.clamp(min=0).long())
        hit = (torch.rand(b, t, generator=host) < 0.67).to(dev)
        tokens = torch.where(hit, wanted, torch.randint(0, v, (b, t), generator=host).to(dev))
        return {"case": case, "logits": logits, "tokens": tokens, "parents": parents}
    order = torch.randperm(case["b"], generator=host)
    pos = torch.tensor(_positions(case))[order].int().to(dev)
    if case["kind"] == "compact":
        shape = (case["layers"], case["b"], case["h"], case["len"], case["d"])
        path = torch.full((case["b"], case["t"]), -1)
        counts = torch.tensor(_counts(case))[torch.randperm(case["b"], generator=host)]
        for i, n in enumerate(counts.tolist()):  # node 0, then nodes that each have to move
            path[i, :n] = torch.cat([torch.zeros(1, dtype=torch.long),
                                     2 + torch.randperm(case["t"] - 2, generator=host)[: n - 1].sort().values])
        return {"case": case, "k": normal(*shape), "v": normal(*shape), "pos": pos, "path": path.int().to(dev),
                "count": counts.int().to(dev)}
    b, h, hkv, t, d = (case[k] for k in ("b", "h", "hkv", "t", "d"))
    return {"case": case, "q": normal(b, h, t, d), "kn": normal(b, hkv, t, d), "vn": normal(b, hkv, t, d),
            "k": normal(b, hkv, case["len"], d), "v": normal(b, hkv, case["len"], d), "pos": pos,
            "parents": _trees(case, host).to(dev)}


# ---------------------------------------------------------------- one pass


def run(st):
    case = st["case"]
    if own:
        heads, attend, accept, compact = _library()
        if case["kind"] == "norm":
            out = heads(st["qkv"], st["wq"], st["wk"], st["cos"], st["sin"], n_head=case["h"], n_kv_head=case["hkv"],
                        positions=st["pos"], eps=EPS, interleaved=case["interleaved"])
            return [*out, *torch.autograd.grad(out, st["leaves"], st["grads"])] if case["grad"] else list(out)
        if case["kind"] == "tree":
            return [attend(st["q"], st["kn"], st["vn"], st["k"], st["v"], st["pos"], st["parents"]), st["k"], st["v"]]
        if case["kind"] == "accept":
            return list(accept(st["logits"], st["tokens"], st["parents"]))
        compact(st["k"], st["v"], st["pos"], st["path"], st["count"])
        return [st["k"], st["v"]]
    if case["kind"] == "norm":
        out = _plain_norm(st["qkv"], st["wq"], st["wk"], st["cos"], st["sin"], st["pos"], case)
        return [*out, *torch.autograd.grad(out, st["leaves"], st["grads"])] if case["grad"] else list(out)
    if case["kind"] == "tree":
        return [_plain_tree(st["q"], st["kn"], st["vn"], st["k"], st["v"], st["pos"], st["parents"]), st["k"], st["v"]]
    if case["kind"] == "accept":
        return _plain_accept(st["logits"], st["tokens"], st["parents"])
    _plain_compact(st["k"], st["v"], st["pos"], st["path"], st["count"])
    return [st["k"], st["v"]]


def _plain_norm(qkv, wq, wk, cos, sin, pos, case):
    b, s, _ = qkv.shape
    h, hkv, d, rot = case["h"], case["hkv"], case["d"], case["rot"]
    x = qkv.reshape(b, s, h + 2 * hkv, d)
    c, sn = (t[:s] if pos is None else t[pos.long()] for t in (cos, sin))
    c, sn = c[..., None, :], sn[..., None, :]  # [(B,) S, 1, rot / 2]

    def rotated(part, w):
        f = part.float()
        u = f * torch.rsqrt(f.square().mean(-1, keepdim=True) + EPS) * w
        if case["interleaved"]:
            lo, hi = u[..., 0:rot:2], u[..., 1:rot:2]
            y = torch.stack([lo * c - hi * sn, hi * c + lo * sn], -1).flatten(-2)
        else:
            lo, hi = u[..., : rot // 2], u[..., rot // 2:rot]
            y = torch.cat([lo * c - hi * sn, hi * c + lo * sn], -1)
        return torch.cat([y, u[..., rot:]], -1).to(qkv.dtype).transpose(1, 2).contiguous()

    return (rotated(x[:, :, :h], wq), rotated(x[:, :, h:h + hkv], wk), x[:, :, h + hkv:].transpose(1, 2).contiguous())


def _ancestors(parents):
    """[B, T, T] truth values: whether node s is node t or one of its ancestors, and [B, T]: whether node t is there, with
    every node that it hangs on."""
    b, t = parents.shape
    idx = torch.arange(t, device=parents.device)
    there = (parents >= -1) & (parents < idx)
    up = (parents[:, :, None] == idx) & there[:, :, None]
    reach = (up | torch.eye(t, dtype=torch.bool, device=parents.device)).float()
    for _ in range(6):  # up to 64 steps
        reach = (torch.matmul(reach, reach) > 0).float()
    reach = reach > 0
    return reach, ~(reach & ~there[:, None, :]).any(-1)


def _plain_tree(q, kn, vn, kc, vc, pos, parents):
    b, h, t, d = q.shape
    hkv, length = kc.shape[1:3]
    seq, node = torch.arange(b, device=q.device)[:, None], torch.arange(t, device=q.device)
    reach, there = _ancestors(parents)
    rows = pos.long()[:, None] + node  # [B, T]
    old_k, old_v = kc[seq, :, rows], vc[seq, :, rows]  # [B, T, Hkv, D]
    here = there[:, :, None, None]
    kc[seq, :, rows] = torch.where(here, kn.transpose(1, 2), old_k)
    vc[seq, :, rows] = torch.where(here, vn.transpose(1, 2), old_v)
    sees = (torch.arange(length, device=q.device) < pos[:, None])[:, None, :].expand(b, t, length).contiguous()
    sees = sees.scatter(2, rows[:, None, :].expand(b, t, t), reach & there[:, None, :])
    sees = (sees & there[:, :, None])[:, None, None]  # [B, 1, 1, T, L]
    s = torch.matmul(q.float().reshape(b, hkv, -1, d), kc.float().transpose(2, 3).contiguous()) / math.sqrt(d)
    s = s.reshape(b, hkv, h // hkv, t, length).masked_fill(~sees, -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True).clamp(min=-1e30))
    out = torch.matmul(p.reshape(b, hkv, -1, length), vc.float()).reshape(b, h, t, d)
    total = p.sum(-1).reshape(b, h, t, 1)
    return torch.where(total > 0, out / total, 0.0).to(q.dtype)


def _first_max(logits):
    """The lowest index of each row's largest value."""
    idx = torch.arange(logits.shape[-1], device=logits.device)
    return torch.where(logits == logits.amax(-1, keepdim=True), idx, logits.shape[-1]).amin(-1)


def _plain_accept(logits, tokens, parents):
    t = tokens.shape[1]
    idx = torch.arange(t, device=tokens.device)
    target = _first_max(logits)
    reach, there = _ancestors(parents)
    right = there & (parents >= 0) & (tokens == target.gather(1, parents.clamp(min=0).long()))
    twin = (parents[:, :, None] == parents[:, None, :]) & right[:, None, :] & (idx[None, :] < idx[:, None])
    right = right & ~twin.any(-1)  # of two children with one token the first
    right[:, 0] = there[:, 0]
    taken = there & ~(reach & ~right[:, None, :]).any(-1) & reach[:, :, 0]
    count = taken.sum(-1)
    path = torch.where(taken, idx, t).sort(-1).values
    last = torch.where(taken, idx, 0).amax(-1, keepdim=True)
    following = torch.where(count > 0, target.gather(1, last)[:, 0], -1)
    return [torch.where(path < t, path, -1).int(), count.int(), following]


def _plain_compact(k, v, pos, path, count):
    b, t = path.shape
    node = torch.arange(t, device=path.device)
    seq = torch.arange(b, device=path.device)[:, None]
    dst = pos.long()[:, None] + node
    src = torch.where(node < count[:, None], pos.long()[:, None] + path, dst)
    k[:, seq, :, dst] = k[:, seq, :, src]
    v[:, seq, :, dst] = v[:, seq, :, src]


# ---------------------------------------------------------------- floors


def work(case) -> dict:
    e = SIZE[case["dtype"]]
    if case["kind"] == "norm":
        values = case["b"] * case["s"] * (case["h"] + 2 * case["hkv"]) * case["d"]
        tables = case["s"] * case["rot"] * 4 * (case["b"] if case["positions"] else 1)
        both = 2 if case["grad"] else 1
        return {"bytes": both * (2 * values * e + tables), "flops": both * 10 * values}
    if case["kind"] == "tree":
        rows, new, d = sum(_positions(case)), case["b"] * case["t"], case["d"]
        return {"bytes": e * d * (2 * case["hkv"] * (rows + 2 * new) + 2 * case["h"] * new),
                "flops": 4 * case["h"] * d * sum(n * p for n, p in zip(_nodes(case), _positions(case)))}
    if case["kind"] == "accept":
        n = sum(_nodes(case)) * case["v"]
        return {"bytes": n * e, "flops": n}
    moved = sum(n - 1 for n in _counts(case))
    return {"bytes": max(64, 4 * case["layers"] * case["h"] * moved * case["d"] * e), "flops": 0}


# ---------------------------------------------------------------- 64 bits


def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "norm":
        return _exact_norm(st, case)
    if case["kind"] == "tree":
        return _exact_tree(st, case)
    if case["kind"] == "accept":
        return _exact_accept(st)
    k, v = st["k"], st["v"]
    for i, (p, n) in enumerate(zip(st["pos"].tolist(), st["count"].tolist())):
        for c in (k, v):
            c[:, i, :, p:p + n] = c[:, i, :, p + st["path"][i, :n].long()].clone()
    return [k, v]


def _exact_norm(st, case):
    b, s, h, hkv, d, rot = (case[k] for k in ("b", "s", "h", "hkv", "d", "rot"))
    half = rot // 2
    x = st["qkv"].detach().double().view(b, s, h + 2 * hkv, d).permute(0, 2, 1, 3)
    place = torch.arange(s, device=x.device).expand(b, s) if st["pos"] is None else st["pos"].long()
    # The rotation as complex products, of the pairs (i, i + rot / 2) or (2 i, 2 i + 1).
    turn = torch.complex(st["cos"].double(), st["sin"].double())[place][:, None]
    first = torch.arange(half, device=x.device) * (2 if case["interleaved"] else 1)
    second = first + (1 if case["interleaved"] else half)

    def turned(u, by):
        z = torch.complex(u[..., first], u[..., second]) * by
        y = u.clone()
        y[..., first], y[..., second] = z.real, z.imag
        return y

    out, dx, dws = [], [], []
    for i, (lo, hi) in enumerate(((0, h), (h, h + hkv))):
        part, w = x[:, lo:hi], (st["wq"], st["wk"])[i].detach().double()
        inv = (part.pow(2).sum(-1, keepdim=True) / d + EPS) ** -0.5
        out.append(turned(part * inv * w, turn))
        if case["grad"]:
            du = turned(st["grads"][i].double(), turn.conj())
            dws.append((du * part * inv).sum((0, 1, 2)))
            along = (du * w * part).sum(-1, keepdim=True) / d
            dx.append(inv * (du * w) - inv ** 3 * part * along)
    out.append(x[:, h + hkv:])
    if case["grad"]:
        dx.append(st["grads"][2].double())
        out += [torch.cat(dx, 1).permute(0, 2, 1, 3).reshape(b, s, -1), *dws]
    return out


def _exact_tree(st, case):
    b, h, t, d = st["q"].shape
    hkv, k, v = case["hkv"], st["k"], st["v"]
    out = torch.zeros(b, h, t, d, dtype=torch.float64, device=k.device)
    for i, (p, parents) in enumerate(zip(st["pos"].tolist(), st["parents"].tolist())):
        sees = [None] * t  # each node's own line of nodes
        for j, up in enumerate(parents):
            if up == -1:
                sees[j] = [j]
            elif 0 <= up < j and sees[up] is not None:
                sees[j] = sees[up] + [j]
        there = [j for j in range(t) if sees[j] is not None]
        if not there:
            continue
        rows = torch.tensor(there, device=k.device)
        k[i, :, p + rows], v[i, :, p + rows] = st["kn"][i][:, rows], st["vn"][i][:, rows]
        hidden = torch.ones(t, t, dtype=torch.bool)
        for j in there:
            hidden[j, sees[j]] = False
        hidden = hidden.to(k.device)
        for g in range(hkv):
            q = st["q"][i, g * (h // hkv):(g + 1) * (h // hkv)].double()  # [G, T, D]
            keys, values = k[i, g, :p + t].double(), v[i, g, :p + t].double()
            s = q @ keys.t() * d ** -0.5
            s[:, :, p:] = s[:, :, p:].masked_fill(hidden, -math.inf)
            out[i, g * (h // hkv):(g + 1) * (h // hkv)][:, rows] = torch.softmax(s[:, rows], -1) @ values
    return [out, k, v]


def _exact_accept(st):
    largest = st["logits"].double().amax(-1, keepdim=True)
    wanted = [[row.index(True) for row in rows] for rows in (st["logits"].double() == largest).tolist()]
    paths, counts, following = [], [], []
    for want, tokens, parents in zip(wanted, st["tokens"].tolist(), st["parents"].tolist()):
        path = [0] if parents[0] == -1 else []
        while path:
            child = [j for j in range(path[-1] + 1, len(parents)) if parents[j] == path[-1] and tokens[j] == want[path[-1]]]
            if not child:
                break
            path.append(child[0])
        paths.append(path + [-1] * (len(parents) - len(path)))
        counts.append(len(path))
        following.append(want[path[-1]] if path else -1)
    dev = st["tokens"].device
    return [torch.tensor(paths, dtype=torch.int32, device=dev), torch.tensor(counts, dtype=torch.int32, device=dev),
            torch.tensor(following, device=dev)]
