"""GPU tests of the operators of a layer-normed, biased transformer together: embedding with scale, layer norm, linear layers with
bias, activation and residual around the causal attention, and the clipping of all gradients, against the same step in 64 bits.

The step in f32 is held to the 64-bit one by 1e-4 of each gradient's norm: its sums of up to K products are off by at most
K u = 512 x 2^-24 = 3e-5 of the sum of their sizes, and by a thousandth of that as roundings go. In bf16 every tensor between two
operators is rounded, half a step 2^-8 of each value in one of 24 places in a row: 24 x 2^-8 = 0.094 of the norm if all erred alike."""

import math

import pytest
import torch

from ferrite.kernels.clip import clip_grad_norm_
from ferrite.kernels.embedding import embedding, embedding_reference
from ferrite.kernels.flash_attention import flash_attention
from ferrite.kernels.heads import merge_heads, split_heads
from ferrite.kernels.layernorm import layernorm, layernorm_reference
from ferrite.kernels.matmul import linear, linear_reference

pytestmark = pytest.mark.gpu

V, D, H, F, B, S = 2000, 128, 2, 512, 2, 128
PAD = 3


def _params(dev, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    mk = lambda *shape, scale: (scale * torch.randn(*shape, generator=g)).to(dev, dtype)
    p = {"tok": mk(V, D, scale=0.02)}
    for i in range(2):
        p |= {f"{i}.n1w": 1 + mk(D, scale=0.1), f"{i}.n1b": mk(D, scale=0.1), f"{i}.qkv": mk(D, 3 * D, scale=0.05),
              f"{i}.qkvb": mk(3 * D, scale=0.1), f"{i}.o": mk(D, D, scale=0.05), f"{i}.ob": mk(D, scale=0.1),
              f"{i}.n2w": 1 + mk(D, scale=0.1), f"{i}.n2b": mk(D, scale=0.1), f"{i}.w1": mk(D, F, scale=0.05),
              f"{i}.b1": mk(F, scale=0.1), f"{i}.w2": mk(F, D, scale=0.05), f"{i}.b2": mk(D, scale=0.1)}
    return {k: t.requires_grad_() for k, t in p.items()}


def _forward(p, tokens, kernels: bool):
    norm, lin, emb = (layernorm, linear, embedding) if kernels else (layernorm_reference, linear_reference, embedding_reference)
    h = emb(tokens, p["tok"], scale=math.sqrt(D), padding_idx=PAD)
    for i in range(2):
        w = lambda k: p[f"{i}.{k}"]
        qkv = lin(norm(h, w("n1w"), w("n1b")), w("qkv"), bias=w("qkvb"))
        if kernels:
            a = merge_heads(flash_attention(*split_heads(qkv, 3, H)))
        else:
            q, k, v = qkv.reshape(B, S, 3, H, D // H).permute(2, 0, 3, 1, 4)
            s = (q @ k.transpose(-1, -2)) / math.sqrt(D // H)
            s = s.masked_fill(torch.ones(S, S, device=s.device).triu(1).bool(), -math.inf)
            a = (torch.softmax(s, -1) @ v).transpose(1, 2).reshape(B, S, D)
        a = lin(a, w("o"), bias=w("ob"))
        h, y = norm(a, w("n2w"), w("n2b"), residual=h)  # the residual add of the norm
        h = lin(lin(y, w("w1"), bias=w("b1"), activation="gelu" if i else "silu"), w("w2"), bias=w("b2"), residual=h)  # and of the product
    return h


def _tokens(dev, seed=1):
    t = torch.randint(0, V, (B, S), generator=torch.Generator().manual_seed(seed))
    t[1, 90:] = PAD
    return t.to(dev)


def _step(p, tokens, dh, most, kernels=True):
    h = _forward(p, tokens, kernels)
    grads = list(torch.autograd.grad(h, list(p.values()), dh))
    if kernels:
        norm = clip_grad_norm_(grads, most)
    else:
        norm = torch.stack([g.square().sum() for g in grads]).sum().sqrt()
        grads = [g * min(1.0, most / (float(norm) + 1e-6)) for g in grads]
    return [h.detach(), norm, *grads]


@pytest.mark.parametrize("dtype,most,off", [(torch.float32, 1.0, 1e-4), (torch.float32, 1e9, 1e-4), (torch.bfloat16, 1.0, 0.094)])
def test_a_step_against_64_bits(dev, dtype, most, off):
    p, tokens = _params(dev, dtype), _tokens(dev)
    dh = torch.randn(B, S, D, generator=torch.Generator().manual_seed(2)).to(dev, dtype)
    got = _step(p, tokens, dh, most)
    want = _step({k: t.detach().double().requires_grad_() for k, t in p.items()}, tokens, dh.double(), most, kernels=False)
    for name, a, b in zip(["h", "norm", *p], got, want):
        assert float((a.double() - b).norm()) <= off * float(b.norm()), name
    grads = dict(zip(p, got[2:]))
    assert not grads["tok"][PAD].any()


def test_a_captured_step(dev):
    p, tokens = _params(dev, torch.bfloat16), _tokens(dev)
    dh = torch.randn(B, S, D, generator=torch.Generator().manual_seed(2)).to(dev, torch.bfloat16)
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _step(p, tokens, dh, 1.0)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _step(p, tokens, dh, 1.0)
    for k in range(3):
        tokens.copy_(_tokens(dev, 10 + k))
        with torch.no_grad():
            for t in p.values():
                t.add_(0.01 * torch.randn_like(t))
        graph.replay()
        want = _step(p, tokens, dh, 1.0)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_steps_of_two_threads(dev):
    """Two threads, a stream each, their own parameters: each finds what it finds alone."""
    from concurrent.futures import ThreadPoolExecutor

    runs = [(_params(dev, torch.bfloat16, seed), _tokens(dev, seed),
             torch.randn(B, S, D, generator=torch.Generator().manual_seed(seed)).to(dev, torch.bfloat16)) for seed in (4, 5)]
    want = [_step(*r, 1.0) for r in runs]
    torch.cuda.synchronize()

    def work(run):
        stream = torch.cuda.Stream(dev)
        with torch.cuda.stream(stream):
            out = [_step(*run, 1.0) for _ in range(5)]
        stream.synchronize()
        return out

    with ThreadPoolExecutor(2) as pool:
        for steps, w in zip(pool.map(work, runs), want):
            for out in steps:
                assert all(torch.equal(a, b) for a, b in zip(out, w))
