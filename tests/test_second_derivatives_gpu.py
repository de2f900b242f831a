"""GPU tests: layer norm, the linear layer's epilogue and the embedding are differentiable once. Their gradients under create_graph are those
without it, and what is computed from them cannot be differentiated: it raises instead of leaving a term out."""

import pytest
import torch

from ferrite.kernels.embedding import embedding
from ferrite.kernels.layernorm import layernorm
from ferrite.kernels.matmul import linear

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


def _call(what, dev, dtype):
    """Leaves, and the function of them."""
    g = torch.Generator().manual_seed(3)
    mk = lambda *shape: torch.randn(*shape, generator=g).to(dev, dtype).requires_grad_()
    if what == "embedding":
        tokens = torch.randint(0, 20, (30,), generator=g).to(dev)
        return [mk(20, 24)], lambda t: embedding(tokens, t, scale=2.0)
    if what == "layernorm":
        return [mk(9, 40), mk(40), mk(40)], layernorm
    if what == "layernorm, residual":
        return [mk(9, 40), mk(40), mk(40), mk(9, 40)], lambda x, w, b, r: layernorm(x, w, b, residual=r)[1]
    act = what.split()[1]
    return [mk(70, 16), mk(16, 24), mk(24)], lambda x, w, b: linear(x, w, bias=b, activation=None if act == "none" else act)


WHAT = ["embedding", "layernorm", "layernorm, residual", "linear none", "linear relu", "linear gelu", "linear silu"]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("what", WHAT)
def test_a_gradient_is_not_differentiated(dev, what, dtype):
    at, f = _call(what, dev, dtype)
    loss = lambda: f(*at).float().square().sum()  # a gradient that depends on the leaves arrives
    want = torch.autograd.grad(loss(), at)
    first = loss()
    got = torch.autograd.grad(first, at, create_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    for d in got:
        with pytest.raises(RuntimeError, match="differentiable once"):
            d.float().square().sum().backward(retain_graph=True)
        with pytest.raises(RuntimeError, match="differentiable once"):  # for leaves alone, beside a term that has its gradient
            torch.autograd.grad(first + d.float().square().sum(), at, retain_graph=True)
    assert all(t.grad is None for t in at)


@pytest.mark.parametrize("what", WHAT[1:])
def test_nor_is_one_of_a_constant_gradient(dev, what):
    at, f = _call(what, dev, F32)
    dy = torch.ones_like(f(*at))
    want = torch.autograd.grad(f(*at), at, dy)
    got = torch.autograd.grad(f(*at), at, dy, create_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(got[0].square().sum(), at)


def test_what_does_not_depend_on_the_inputs_has_no_graph(dev):
    at, f = _call("embedding", dev, F32)
    d, = torch.autograd.grad(f(*at).sum(), at, create_graph=True)  # the table's gradient is linear in what arrives, a constant here
    assert not d.requires_grad


def test_the_residuals_gradient_is_the_one_that_arrives(dev):
    (x, w, b), _ = _call("linear gelu", dev, F32)
    r = torch.randn(70, 24, device=dev, requires_grad=True)
    y = linear(x, w, bias=b, activation="gelu", residual=r)
    d, = torch.autograd.grad(y.square().sum(), r, create_graph=True)
    twice, = torch.autograd.grad(d.square().sum(), r)  # sum of (2 y)^2
    assert torch.equal(twice, 8 * y)


def test_gradients_kept_with_a_graph_train(dev):
    """backward(create_graph=True) and a step of an optimiser: what such a program does with first gradients alone."""
    at, f = _call("linear silu", dev, F32)
    f(*at).square().sum().backward(create_graph=True)
    want = torch.autograd.grad(f(*at).square().sum(), at)
    with torch.no_grad():
        for t, d in zip(at, want):
            assert torch.equal(t.grad, d)
            t.sub_(t.grad, alpha=0.1)
            t.grad = None
