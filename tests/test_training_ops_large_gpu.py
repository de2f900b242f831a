"""GPU tests of the training operators (layer norm, linear, embedding, clipping) on tensors of more than 2^31 elements: what lies behind
that many is computed as the same rows by themselves are. Everything before the last rows has a gradient of zero, so that sums over
all rows are those of the last."""

import pytest
import torch

from ferrite.kernels.clip import clip_grad_norm_
from ferrite.kernels.embedding import embedding
from ferrite.kernels.layernorm import layernorm, layernorm_reference
from ferrite.kernels.matmul import linear, linear_reference

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
LAST = 300  # rows that are looked at, at either end


@pytest.fixture(autouse=True)
def _give_back():
    yield
    torch.cuda.empty_cache()


def _near(a, b, off):
    a, b = a.detach().double(), b.detach().double()
    assert float((a - b).norm()) <= off * float(b.norm())


# Half a step of the output's type for each value and the f32 arithmetic before it, far below: 2^-8 in bf16, and 16 of 2^-24 in f32.
OFF = {BF16: 2.0**-8, F32: 2.0**-20}


@pytest.mark.parametrize("dim", [1024, 1003])
def test_layernorm(dev, dim):
    rows = (1 << 31) // dim + 2 * LAST
    x = torch.empty(rows, dim, device=dev, dtype=BF16).normal_(generator=torch.Generator(dev).manual_seed(dim)).requires_grad_()
    w, b = (torch.randn(dim, device=dev).requires_grad_() for _ in range(2))
    y = layernorm(x, w, b)
    for rs in (slice(0, LAST), slice(rows - LAST, rows)):
        _near(y[rs], layernorm_reference(x[rs].detach().double(), w.double(), b.double()), OFF[BF16])
    dy = torch.zeros_like(y)
    dy[-LAST:].normal_()
    got = torch.autograd.grad(y, (x, w, b), dy)
    assert not got[0][:LAST].any()
    xs = x[-LAST:].detach().double().requires_grad_()
    ws, bs = (t.detach().double().requires_grad_() for t in (w, b))
    want = torch.autograd.grad(layernorm_reference(xs, ws, bs), (xs, ws, bs), dy[-LAST:].double())
    _near(got[0][-LAST:], want[0], OFF[BF16])
    _near(got[1], want[1], 1e-5)  # the rows' f32 statistics and 300 products to a sum: some 20 of 2^-24
    _near(got[2], want[2], 1e-5)


@pytest.mark.parametrize("dtype,n,k", [(BF16, 32768, 64), (BF16, 32771, 33), (F32, 32768, 32), (F32, 32771, 19)])
def test_linear(dev, dtype, n, k):
    m = (1 << 31) // n + 2 * LAST
    g = torch.Generator(dev).manual_seed(n)
    x = torch.randn(m, k, device=dev, generator=g).to(dtype).requires_grad_()
    w = torch.randn(k, n, device=dev, generator=g).div_(k**0.5).to(dtype).requires_grad_()
    b = torch.randn(n, device=dev, generator=g).requires_grad_()
    r = torch.zeros(m, n, device=dev, dtype=dtype)
    r[-LAST:].normal_(generator=g)
    r.requires_grad_()
    y = linear(x, w, bias=b, activation="silu", residual=r)
    for rs in (slice(0, LAST), slice(m - LAST, m)):
        want = linear_reference(x[rs].detach().double(), w.detach().double(), bias=b.detach().double(), activation="silu",
                                residual=r[rs].detach().double())
        _near(y[rs], want, OFF[dtype])
    del want
    dy = torch.zeros_like(y)
    dy[-LAST:].normal_(generator=g)
    del y
    got = torch.autograd.grad(linear(x, w, bias=b, activation="silu", residual=r), (x, w, b, r), dy)
    xs, ws, bs = (t.detach().double().requires_grad_() for t in (x[-LAST:], w, b))
    out = linear_reference(xs, ws, bias=bs, activation="silu")
    want = torch.autograd.grad(out, (xs, ws, bs), dy[-LAST:].double())
    assert not got[0][:LAST].any() and torch.equal(got[3][-LAST:], dy[-LAST:])
    # the pre-activation's rounding, through a slope that changes by at most one half per unit of |u| < 8: 4 half steps; du's; the output's
    off = 6 * 2.0**-8 if dtype == BF16 else 1e-5
    _near(got[0][-LAST:], want[0], off)
    _near(got[1], want[1], off)
    _near(got[2], want[2], off)


@pytest.mark.parametrize("dim", [2048, 2043])
def test_embedding(dev, dim):
    """A table and an output of more than 2^31 elements each; every row of the table a constant of its own."""
    vocab = rows = (1 << 31) // dim + 2 * LAST
    g = torch.Generator(dev).manual_seed(dim)
    ids = (torch.arange(vocab, device=dev) % 251).to(BF16)  # whole numbers that bf16 holds
    table = ids[:, None].repeat(1, dim).requires_grad_()
    tokens = torch.randint(0, vocab, (rows,), device=dev, generator=g)
    tokens[-LAST:] = vocab - 1 - torch.arange(LAST, device=dev) // 3  # the table's last rows, three times each
    out = embedding(tokens, table, scale=2.0)
    assert torch.equal(out[:, 0], 2 * ids[tokens]) and torch.equal(out[:, -1], 2 * ids[tokens])
    dy = torch.zeros_like(out)
    dy[-LAST:] = 1.0
    dy[-LAST:, ::2] = 2.0
    del out
    d = torch.autograd.grad(embedding(tokens, table, scale=2.0), table, dy)[0]
    want = torch.full((dim,), 6.0, device=dev, dtype=BF16)
    want[::2] = 12.0
    assert bool((d[-(LAST // 3):] == want).all()) and not d[:LAST].any() and float(d[:, 0].float().sum()) == 12.0 * (LAST // 3)


def test_clip(dev):
    n = (1 << 31) + 70001
    big = torch.zeros(n + 1, device=dev, dtype=BF16)[1:]
    big[-1000:] = 3.0
    big[:1000] = 4.0
    small = torch.zeros(5, device=dev)
    norm = clip_grad_norm_([small, big], 15.0)
    exact = (1000 * 25.0) ** 0.5
    assert abs(float(norm) - exact) <= 2.0**-23 * exact
    factor = 15.0 / exact
    for part, v in ((big[-1000:], 3.0), (big[:1000], 4.0)):
        assert bool(((part.double() - v * factor).abs() <= 1.01 * 2.0**-8 * v * factor).all())
    assert not big[1000:-1000].any()
