"""CPU tests of layer norm, the linear layer's epilogues, the embedding and gradient clipping: what they refuse, and their
references against torch."""

import pytest
import torch
import torch.nn.functional as F

from ferrite.kernels.clip import clip_grad_norm_, clip_grad_norm_reference
from ferrite.kernels.embedding import embedding, embedding_reference
from ferrite.kernels.layernorm import layernorm, layernorm_reference
from ferrite.kernels.matmul import linear, linear_reference


def test_layernorm_refuses():
    x, w, b = torch.randn(4, 8), torch.ones(8), torch.zeros(8)
    with pytest.raises(ValueError, match="shape"):
        layernorm(x, torch.ones(7))
    with pytest.raises(ValueError, match="shape"):
        layernorm(x, w, torch.zeros(9))
    with pytest.raises(ValueError, match="share a dtype"):
        layernorm(x, w, b.bfloat16())
    with pytest.raises(ValueError, match="residual"):
        layernorm(x, w, b, residual=x[:2])
    with pytest.raises(ValueError, match="residual"):
        layernorm(x, w, b, residual=x.bfloat16())
    with pytest.raises(ValueError, match="float32 or bfloat16"):
        layernorm(x.half(), w, b)
    with pytest.raises(ValueError, match="float32 or bfloat16"):
        layernorm(x, w.double(), b.double())
    with pytest.raises(RuntimeError, match="non-empty"):
        layernorm(torch.zeros(4, 0), torch.ones(0))
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        layernorm(x, w, b)


def test_layernorm_reference():
    g = torch.Generator().manual_seed(0)
    x, r = (torch.randn(3, 5, 40, generator=g, dtype=torch.float64, requires_grad=True) for _ in range(2))
    w, b = (torch.randn(40, generator=g, dtype=torch.float64, requires_grad=True) for _ in range(2))
    h, y = layernorm_reference(x, w, b, residual=r)
    assert torch.equal(h, x + r) and torch.allclose(y, F.layer_norm(h, (40,), w, b, 1e-5), rtol=1e-12, atol=1e-12)
    assert torch.allclose(layernorm_reference(x, w), F.layer_norm(x, (40,), w, None, 1e-5), rtol=1e-12, atol=1e-12)


def test_embedding_refuses():
    tokens, table = torch.zeros(4, dtype=torch.long), torch.ones(8, 16)
    with pytest.raises(ValueError, match="table"):
        embedding(tokens, torch.ones(8))
    with pytest.raises(ValueError, match="table"):
        embedding(tokens, torch.ones(0, 16))
    with pytest.raises(ValueError, match="int64 or int32"):
        embedding(tokens.float(), table)
    with pytest.raises(ValueError, match="int64 or int32"):
        embedding(tokens.short(), table)
    for pad in (-1, 8):
        with pytest.raises(ValueError, match="padding_idx"):
            embedding(tokens, table, padding_idx=pad)
    with pytest.raises(ValueError, match="float32 or bfloat16"):
        embedding(tokens, table.half())
    with pytest.raises(ValueError, match="float32 or bfloat16"):
        embedding(tokens, table, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        embedding(tokens, table)


def test_embedding_reference():
    g = torch.Generator().manual_seed(1)
    tokens, table = torch.randint(0, 9, (3, 20), generator=g), torch.randn(9, 6, generator=g, dtype=torch.float64, requires_grad=True)
    out = embedding_reference(tokens, table, scale=3.0, padding_idx=4)
    ref = F.embedding(tokens, table, padding_idx=4) * 3.0
    dy = torch.randn(out.shape, generator=g, dtype=torch.float64)
    assert torch.equal(out, ref)
    assert torch.allclose(torch.autograd.grad(out, table, dy)[0], torch.autograd.grad(ref, table, dy)[0], rtol=1e-12)
    tokens[0, 0], tokens[1, 1] = -1, 9
    out = embedding_reference(tokens, table.detach())
    assert bool(out[0, 0].isnan().all()) and bool(out[1, 1].isnan().all()) and int(out.isnan().sum()) == 12


def test_embedding_sizes_out_of_range():
    from ferrite import _hip

    lib = _hip.lib()
    assert lib.ferrite_internal_embedding_bwd_workspace(1 << 27, 8, 8) == -1
    assert lib.ferrite_internal_embedding_bwd_workspace(8, 4194241, 8) == -1
    assert lib.ferrite_internal_embedding_bwd_workspace(8, 8, 0x7fffffff) == -1
    assert lib.ferrite_internal_embedding_bwd_workspace(8, 0, 8) == -1
    assert lib.ferrite_internal_embedding_bwd_workspace(0, 8, 8) == 0
    assert lib.ferrite_internal_embedding_bwd_workspace(16384, 64, 50257) > 0
    assert lib.ferrite_internal_embedding_bwd(None, None, None, 1, 8, 8, -1, 1.0, 0, 1, 1, None, 0, None) == 1
    assert lib.ferrite_internal_embedding(None, None, None, 1, 8, 8, 1.0, 0, 1, 7, None) == 1


def test_clip_refuses():
    with pytest.raises(ValueError, match="no tensors"):
        clip_grad_norm_([], 1.0)
    for most in (-1.0, float("nan")):
        with pytest.raises(ValueError, match="max_norm"):
            clip_grad_norm_([torch.ones(3)], most)
    with pytest.raises(ValueError, match="float32 or bfloat16"):
        clip_grad_norm_([torch.ones(3), torch.ones(3).half()], 1.0)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        clip_grad_norm_([torch.ones(3)], 1.0)


def test_clip_reference():
    g = torch.Generator().manual_seed(2)
    grads = [torch.randn(n, generator=g) for n in (5, 70, 1)]
    params = [torch.nn.Parameter(torch.zeros_like(x)) for x in grads]
    for p, x in zip(params, grads):
        p.grad = x.clone()
    norm = torch.nn.utils.clip_grad_norm_(params, 2.0)
    assert torch.allclose(clip_grad_norm_reference(grads, 2.0), norm, rtol=1e-6)
    assert all(torch.allclose(x, p.grad, rtol=1e-6) for x, p in zip(grads, params))


def test_linear_refuses():
    x, w, b = torch.ones(4, 8), torch.ones(8, 6), torch.ones(6)
    with pytest.raises(ValueError, match="expected"):
        linear(x, torch.ones(7, 6), bias=b)
    with pytest.raises(ValueError, match="bias"):
        linear(x, w, bias=torch.ones(8))
    with pytest.raises(ValueError, match="activation"):
        linear(x, w, activation="tanh")
    with pytest.raises(ValueError, match="residual"):
        linear(x, w, residual=torch.ones(4, 8))
    with pytest.raises(ValueError, match="residual"):
        linear(x, w, residual=torch.ones(4, 6).bfloat16())
    for args in ((x.half(), w, b), (x, w.half(), b), (x, w, b.half())):
        with pytest.raises(ValueError, match="float32 or bfloat16"):
            linear(args[0], args[1], bias=args[2], activation="relu")
    with pytest.raises(RuntimeError, match="non-empty"):
        linear(torch.ones(4, 0), torch.ones(0, 6), bias=b)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        linear(x, w, bias=b)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        linear(x, w)


def test_linear_reference():
    g = torch.Generator().manual_seed(3)
    x, w, b, r = (torch.randn(*s, generator=g, dtype=torch.float64) for s in ((2, 3, 8), (8, 6), (6,), (2, 3, 6)))
    u = x @ w + b
    for act, ref in ((None, u), ("relu", u.clamp(min=0)), ("silu", u * torch.sigmoid(u)), ("gelu", F.gelu(u, approximate="tanh"))):
        assert torch.allclose(linear_reference(x, w, bias=b, activation=act, residual=r), ref + r, rtol=1e-12, atol=1e-12)


def test_linear_sizes_out_of_range():
    from ferrite import _hip

    lib = _hip.lib()
    assert lib.ferrite_internal_linear_workspace(None, None, None, 0, 8, 8, 1, 1) == -1
    assert lib.ferrite_internal_linear_workspace(None, None, None, 8, 1 << 31, 8, 1, 1) == -1
    assert lib.ferrite_internal_linear_workspace(None, None, None, 65, 64, 64, 1, 0) == -1  # a float weight of many rows
    assert lib.ferrite_internal_act_grad_workspace(4, 0) == -1
    assert lib.ferrite_internal_act_grad(None, None, None, None, 1, 8, 9, 1, 1, None, 0, None) == 1
    assert lib.ferrite_internal_layernorm_bwd_workspace(1, 0) == -1 and lib.ferrite_internal_layernorm_bwd_workspace(1, 1 << 25) == -1
    assert lib.ferrite_internal_clip_workspace(-1) == -1
    assert lib.ferrite_internal_clip(1, None, None, None, -1.0, None, None, 0, None) == 1
