"""The operators of a layer-normed, biased transformer's training step around its attention: layer norm, a linear
layer with bias, activation and residual, the tokens' embedding, and the clipping of the gradients. Their plain
forms in elementary torch operations, the calls of the library's kernels, and the cases by which the two are measured.

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
EPS = 1e-5
GELU = (math.sqrt(2 / math.pi), 0.044715)

_calls = None


def _library():
    """The library's entry points, imported where its own kernels run, once."""
    global _calls
    if _calls is None:
        pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ferrite-tpu_amd")
        if pkg not in sys.path:
            sys.path.insert(0, pkg)
        from ferrite.kernels.clip import clip_grad_norm_
        from ferrite.kernels.embedding import embedding
        from ferrite.kernels.layernorm import layernorm
        from ferrite.kernels.matmul import linear

        _calls = (layernorm, linear, embedding, clip_grad_norm_)
    return _calls


# ---------------------------------------------------------------- cases


def listed() -> list[dict]:
    return [
        # The last norm of one decode token of the default model: the smallest call, one launch.
        _norm("norm_token", 1, 512, "bf16", residual=False, grad=False),
        # A training step's norm (12-layer model, batch 8 x 1024) with the residual add before it, forward and backward.
        _norm("norm_train", 8192, 768, "bf16", residual=True, grad=True),
        # Training in float32 at an odd width.
        _norm("norm_f32", 3001, 1003, "f32", residual=False, grad=True),
        # The MLP's first product of a decode step of eight users, default model: latency.
        _linear("linear_decode", 8, 512, 2048, "bf16", "gelu", bias=True, residual=False, grad=False),
        # The same layer of the default training step (batch 64 x 256), forward and backward.
        _linear("linear_train", 16384, 512, 2048, "bf16", "gelu", bias=True, residual=False, grad=True),
        # Prefill of 8192 tokens through a wide output projection that closes a residual branch.
        _linear("linear_wide", 8192, 4096, 4096, "bf16", "none", bias=True, residual=True, grad=False),
        # Training in float32 at ragged sizes.
        _linear("linear_f32", 2100, 1003, 515, "f32", "silu", bias=True, residual=True, grad=True),
        # A few bytes' embedding and its gradient: latency.
        _embed("embed_bytes", 1, 64, 256, 512, "bf16", grad=True, padded=False),
        # A training step's tokens over a vocabulary of 32768 (batch 8 x 1024), scaled, with the table's gradient.
        _embed("embed_train", 8, 1024, 32768, 768, "bf16", grad=True, padded=False),
        # float32, odd sizes, sequences padded behind their ends with a token that has no gradient.
        _embed("embed_f32", 3, 1001, 50257, 515, "f32", grad=True, padded=True),
        # The default model's float gradients, within the bound: nothing to scale.
        _clip("clip_default", 4, 512, 2048, 256, 256, "f32", over=False),
        # bf16 gradients of an eight-layer model over a vocabulary of 32768, over the bound.
        _clip("clip_model", 8, 768, 2048, 32768, 1024, "bf16", over=True),
    ]


def _norm(name, rows, dim, dtype, residual, grad) -> dict:
    return {"name": name, "kind": "norm", "rows": rows, "dim": dim, "dtype": dtype, "residual": residual, "grad": grad}


def _linear(name, m, k, n, dtype, act, bias, residual, grad) -> dict:
    return {"name": name, "kind": "linear", "m": m, "k": k, "n": n, "dtype": dtype, "act": act, "bias": bias,
            "residual": residual, "grad": grad}


def _embed(name, b, s, vocab, dim, dtype, grad, padded) -> dict:
    return {"name": name, "kind": "embed", "b": b, "s": s, "vocab": vocab, "dim": dim, "dtype": dtype, "grad": grad,
            "padded": padded}


def _clip(name, layers, d, f, vocab, seq, dtype, over) -> dict:
    return {"name": name, "kind": "clip", "layers": layers, "d": d, "f": f, "vocab": vocab, "seq": seq, "dtype": dtype,
            "over": over}


def _log_int(rng, lo: int, hi: int) -> int:
    """An integer of [lo, hi], even over its logarithm."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng) -> dict:
    kind = rng.choice(["norm", "norm", "linear", "linear", "linear", "embed", "embed", "clip"])
    while True:
        case = globals()["_draw_" + kind](rng)
        case.pop("name", None)
        w = work(case)
        # No more than the largest listed cases; float32 products run at a sixteenth of bf16's rate.
        if w["bytes"] <= 4.1e8 and w["flops"] * (16 if case["dtype"] == "f32" else 1) <= 2.76e11:
            return case


def _type(rng) -> str:
    return "bf16" if rng.random() < 0.75 else "f32"


def _width(rng, lo: int, hi: int) -> int:
    """A width as models have them, a multiple of 64, or any."""
    n = _log_int(rng, lo, hi)
    return n if rng.random() < 0.35 else max(lo, n // 64 * 64)


def _draw_norm(rng) -> dict:
    rows = _log_int(rng, 1, 64) if rng.random() < 0.3 else _log_int(rng, 64, 32768)
    return _norm("", rows, _width(rng, 64, 8192), _type(rng), rng.random() < 0.6, rng.random() < 0.6)


def _draw_linear(rng) -> dict:
    m = _log_int(rng, 1, 64) if rng.random() < 0.3 else _log_int(rng, 64, 16384)
    dtype, grad = _type(rng), rng.random() < 0.5
    # relu's slope jumps at 0: one sum of a million that rounding takes across it moves float32 gradients by 1e-3.
    acts = ["none", "gelu", "silu"] if grad and dtype == "f32" else ["none", "relu", "gelu", "silu"]
    return _linear("", m, _width(rng, 64, 4096), _width(rng, 64, 4096), dtype, rng.choice(acts), rng.random() < 0.8,
                   rng.random() < 0.4, grad)


def _draw_embed(rng) -> dict:
    return _embed("", _log_int(rng, 1, 32), _log_int(rng, 1, 2048), _log_int(rng, 256, 131072), _width(rng, 64, 4096),
                  _type(rng), rng.random() < 0.75, rng.random() < 0.4)


def _draw_clip(rng) -> dict:
    d = _width(rng, 64, 2048)
    return _clip("", rng.randint(1, 10), d, rng.choice([2, 4]) * d, _log_int(rng, 256, 50257), _log_int(rng, 64, 2048),
                 _type(rng), rng.random() < 0.6)


# ---------------------------------------------------------------- state


def _shapes(case) -> list[tuple]:
    """The shapes of a GPT's parameters, in the order of their names."""
    d, f = case["d"], case["f"]
    layer = [(d,), (d,), (d, f), (f, d), (d, d), (d, 3 * d)]
    return layer * case["layers"] + [(d,), (case["seq"], d), (case["vocab"], d)]


def _lengths(case) -> list[int]:
    """Tokens of each sequence before its padding: from a third to all of them."""
    b, s = case["b"], case["s"]
    return [s - (s * 2 // 3) * (i + 1) // b if case["padded"] else s for i in range(b)]


def prepare(case, seed):
    dev = torch.device("cuda:0")
    host = torch.Generator().manual_seed(seed)
    gen = torch.Generator(dev).manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0, loc=0.0, dtype=dt):
        return torch.randn(*shape, generator=gen, device=dev, dtype=torch.float32).mul_(scale).add_(loc).to(dtype)

    st = {"case": case}
    if case["kind"] == "norm":
        shape = (case["rows"], case["dim"])
        # Activations with channels of their own means and sizes, as residual streams have.
        own_size = normal(case["dim"], scale=0.5, dtype=torch.float32).exp()
        own_mean = normal(case["dim"], scale=0.5, dtype=torch.float32)
        st["x"] = (normal(*shape, dtype=torch.float32) * own_size + own_mean).to(dt)
        st["r"] = normal(*shape) if case["residual"] else None
        st["w"] = normal(case["dim"], scale=0.1, loc=1.0, dtype=torch.float32)
        st["b"] = normal(case["dim"], scale=0.1, dtype=torch.float32)
        outputs, names = (2 if case["residual"] else 1), ("x", "r", "w", "b")
        st["grads"] = [normal(*shape) for _ in range(outputs if case["grad"] else 0)]
    elif case["kind"] == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        st["x"], st["w"] = normal(m, k), normal(k, n, scale=1 / math.sqrt(k))
        st["b"] = normal(n, scale=0.5) if case["bias"] else None
        st["r"] = normal(m, n) if case["residual"] else None
        names = ("x", "w", "b", "r")
        st["grads"] = [normal(m, n)] if case["grad"] else []
    elif case["kind"] == "embed":
        b, s, v = case["b"], case["s"], case["vocab"]
        # Tokens as text has them: the k-th of the vocabulary about once in k.
        tokens = (float(v) ** torch.rand(b, s, generator=host, dtype=torch.float64)).long().clamp(1, v) - 1
        if case["padded"]:
            ends = torch.tensor(_lengths(case))[torch.randperm(b, generator=host)]
            tokens = torch.where(torch.arange(s) < ends[:, None], tokens, v - 1)
        st["pad"] = v - 1 if case["padded"] else None
        st["tokens"], st["table"] = tokens.to(dev), normal(v, case["dim"], scale=0.02)
        names = ("table",)
        st["grads"] = [normal(b, s, case["dim"])] if case["grad"] else []
    else:
        st["g"] = [normal(*shape, scale=1e-3) for shape in _shapes(case)]
        size = 1e-3 * math.sqrt(sum(math.prod(shape) for shape in _shapes(case)))  # about their norm
        st["most"] = size * (0.5 if case["over"] else 2.0)
        return st
    st["scale"] = math.sqrt(case["dim"]) if case["kind"] == "embed" else 1.0
    if case["grad"]:
        st["leaves"] = [st[k].requires_grad_() for k in names if st[k] is not None]
    return st


# ---------------------------------------------------------------- one pass


def run(st):
    case = st["case"]
    if case["kind"] == "clip":
        if case["over"]:
            st["most"] *= 1 - 2.0 ** -10  # clipped gradients lie at the bound: a lower one has them scaled at every pass
        if own:
            return [_library()[3](st["g"], st["most"]), *st["g"]]
        return [_plain_clip(st["g"], st["most"]), *st["g"]]
    if own:
        norm, linear, embed, _ = _library()
        if case["kind"] == "norm":
            out = norm(st["x"], st["w"], st["b"], residual=st["r"], eps=EPS)
        elif case["kind"] == "linear":
            out = linear(st["x"], st["w"], bias=st["b"], activation=None if case["act"] == "none" else case["act"],
                         residual=st["r"])
        else:
            out = embed(st["tokens"], st["table"], scale=st["scale"], padding_idx=st["pad"])
    elif case["kind"] == "norm":
        out = _plain_norm(st["x"], st["r"], st["w"], st["b"])
    elif case["kind"] == "linear":
        out = _plain_linear(st["x"], st["w"], st["b"], st["r"], case["act"])
    else:
        out = _plain_embed(st["tokens"], st["table"], st["scale"], st["pad"])
    out = list(out) if isinstance(out, tuple) else [out]
    return [*out, *torch.autograd.grad(out, st["leaves"], st["grads"])] if case["grad"] else out


def _plain_norm(x, r, w, b):
    """h = x + r in x's type, and h's rows less their mean, over their deviation, times w, plus b."""
    h = x if r is None else (x.float() + r.float()).to(x.dtype)
    f = h.float()
    c = f - f.mean(-1, keepdim=True)
    y = (c * torch.rsqrt(c.square().mean(-1, keepdim=True) + EPS) * w + b).to(x.dtype)
    return y if r is None else (h, y)


def _plain_linear(x, w, b, r, act):
    u = torch.matmul(x.float(), w.float())
    if b is not None:
        u = u + b.float()
    if act == "relu":
        u = torch.where(u > 0, u, 0.0)
    elif act == "gelu":
        u = 0.5 * u * (1 + torch.tanh(GELU[0] * (u + GELU[1] * u * u * u)))
    elif act == "silu":
        u = u / (1 + torch.exp(-u))
    return (u if r is None else u + r.float()).to(x.dtype)


def _plain_embed(tokens, table, scale, pad):
    f = table.float()
    if pad is not None:  # the padding's row is read and has no gradient
        rows = torch.arange(table.shape[0], device=table.device)[:, None]
        f = torch.where(rows == pad, f.detach(), f)
    return (f[tokens] * scale).to(table.dtype)


def _plain_clip(grads, most):
    norm = torch.sqrt(torch.stack([g.float().square().sum() for g in grads]).sum())
    factor = (most / (norm + 1e-6)).clamp(max=1.0)
    for g in grads:
        g.copy_(g.float() * factor)
    return norm


# ---------------------------------------------------------------- floors


def work(case) -> dict:
    e, grad = SIZE[case["dtype"]], case.get("grad", False)
    if case["kind"] == "norm":
        values = case["rows"] * case["dim"]
        streams = (4 if case["residual"] else 2) + (grad and (3 if case["residual"] else 2))  # dy (and dh) in, dx out
        return {"bytes": values * streams * e + 4 * case["dim"] * (4 if grad else 2), "flops": values * (16 if grad else 7)}
    if case["kind"] == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        values = m * k + k * n + m * n * (2 if case["residual"] else 1) + (n if case["bias"] else 0)
        more = m * n + m * k + k * n + (n if case["bias"] else 0) if grad else 0
        return {"bytes": e * (values + more), "flops": 2 * m * k * n * (3 if grad else 1)}
    if case["kind"] == "embed":
        rows, v, d = case["b"] * case["s"], case["vocab"], case["dim"]
        real = sum(_lengths(case))
        return {"bytes": 8 * rows + e * d * (min(v, rows) + rows + (real + v if grad else 0)),
                "flops": d * (rows + (real if grad else 0))}
    values = sum(math.prod(shape) for shape in _shapes(case))
    return {"bytes": values * e * (3 if case["over"] else 1), "flops": values * (3 if case["over"] else 2)}


# ---------------------------------------------------------------- 64 bits


def exact(case, seed):
    st = prepare(case, seed)
    with torch.no_grad():
        return globals()["_exact_" + case["kind"]](st, case)


def _exact_norm(st, case):
    x, w, b = st["x"], st["w"].double(), st["b"].double()
    # The residual stream is what is stored of the sum, in x's type.
    h = x.double() if st["r"] is None else (x.double() + st["r"].double()).to(x.dtype).double()
    centred = h - h.sum(-1, keepdim=True) / h.shape[1]
    rstd = ((centred * centred).sum(-1, keepdim=True) / h.shape[1] + EPS) ** -0.5
    unit = centred * rstd
    out = ([] if st["r"] is None else [h]) + [unit * w + b]
    if case["grad"]:
        dy = st["grads"][-1].double()
        g = dy * w
        dh = rstd * (g - g.mean(-1, keepdim=True) - unit * (g * unit).mean(-1, keepdim=True))
        if st["r"] is not None:
            dh = dh + st["grads"][0].double()
        out += [dh] * (1 if st["r"] is None else 2) + [(dy * unit).sum(0), dy.sum(0)]
    return out


def _exact_linear(st, case):
    x, w = st["x"].double(), st["w"].double()
    u = torch.mm(x, w) + (0.0 if st["b"] is None else st["b"].double())
    one = torch.ones_like(u)
    if case["act"] == "none":
        a, slope = u, one
    elif case["act"] == "relu":
        a, slope = u.clamp(min=0), (u > 0).double()
    else:
        # u times a sigmoid of z(u): z = u, or twice the tanh form's argument.
        z, dz = (u, one) if case["act"] == "silu" else (2 * GELU[0] * (u + GELU[1] * u ** 3),
                                                        2 * GELU[0] * (1 + 3 * GELU[1] * u ** 2))
        s = torch.sigmoid(z)
        a, slope = u * s, s + u * s * (1 - s) * dz
    out = [a if st["r"] is None else a + st["r"].double()]
    if case["grad"]:
        dy = st["grads"][0].double()
        du = dy * slope
        out += [torch.mm(du, w.t()), torch.mm(x.t(), du)]
        out += [] if st["b"] is None else [du.sum(0)]
        out += [] if st["r"] is None else [dy]
    return out


def _exact_embed(st, case):
    tokens, table = st["tokens"], st["table"].double()
    out = [table.index_select(0, tokens.reshape(-1)).reshape(*tokens.shape, -1) * st["scale"]]
    if case["grad"]:
        dy = st["grads"][0].double().reshape(-1, case["dim"])
        line = tokens.reshape(-1)
        if st["pad"] is not None:
            dy, line = dy[line != st["pad"]], line[line != st["pad"]]
        out.append(torch.zeros_like(table).index_put_((line,), dy * st["scale"], accumulate=True))
    return out


def _exact_clip(st, case):
    most = st["most"] * (1 - 2.0 ** -10 if case["over"] else 1.0)
    flat = [g.double().reshape(-1) for g in st["g"]]
    norm = math.sqrt(math.fsum(float(torch.dot(f, f)) for f in flat))
    factor = min(1.0, most / (norm + 1e-6))
    return [torch.tensor(norm, dtype=torch.float64), *(g.double() * factor for g in st["g"])]
