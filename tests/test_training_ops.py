"""CPU tests of layer norm, the linear layer's epilogues, the embedding and gradient clipping: what they refuse, and their
references against torch."""

import pytest
import torch
import torch.nn.functional as F

from ferrite.kernels.layernorm import layernorm, layernorm_reference


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
