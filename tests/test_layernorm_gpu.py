"""GPU tests of layer norm (csrc/layernorm.hip), forward and backward, against the formulas in 64 bits.

Tolerances, in units u = 2^-24 of f32's half step, before the output's own rounding. S is the most additions in a row that a sum over
a row takes: 32 in a lane, 6 in a wave, 8 over waves (48 allowed; in the sweeps dim / 256 and 16). The mean is corrected by the mean of the
differences, so a difference c is off by 2 u |c| + (S - 1) u mean|c|. Their squares' sum is within S + 4, the inverse deviation within
half of that and 4: 30 u at S = 48. A normed value n = c / deviation is then within (S / 2 + 10) |n| + S (as mean|c| is at most
the deviation), y = n w + b adds a product and a sum. A gradient's means of g = dy w and of g n carry S and n's own error: K = S + 90 of
each of its terms. A parameter's gradient is summed over rows of a group, 4 groups, 32 partial rows of a wave and 16 waves, 256 partial rows in
all or up to 512 to 1024 columns: rows / 2048 of a group to 1024 columns where there are rows for that, rows / 1024 to 2048, rows / 256
beyond and in the sweeps, where a wave has 16 partial rows and there are no groups. 64 and rows / 2048 hold for every case of `_check`."""

import pytest
import torch

from ferrite.kernels.layernorm import layernorm, layernorm_reference

pytestmark = pytest.mark.gpu

U = 2.0**-24
HALF = {torch.bfloat16: 2.0**-8, torch.float32: 2.0**-24}
BF16, F32 = torch.bfloat16, torch.float32
EPS = 1e-5


def _inputs(dev, rows, dim, dtype, wdtype, residual, bias, seed=0, loc=0.0):
    g = torch.Generator().manual_seed(seed)
    mk = lambda *shape: torch.randn(*shape, generator=g)
    x = (loc + mk(rows, dim) * (0.5 + torch.rand(dim, generator=g))).to(dev, dtype)
    r = mk(rows, dim).to(dev, dtype) if residual else None
    w, b = (1 + 0.3 * mk(dim)).to(dev, wdtype), (0.3 * mk(dim)).to(dev, wdtype) if bias else None
    dy, dh = mk(rows, dim).to(dev, dtype), mk(rows, dim).to(dev, dtype) if residual else None
    return x, r, w, b, dy, dh


def _swept(dim):
    return dim < 8 or dim > 16384


def _parts(x, r, w, eps):
    h = x if r is None else (x.float() + r.float()).to(x.dtype)
    c = h.double() - h.double().mean(-1, keepdim=True)
    rs = (c.square().mean(-1, keepdim=True) + eps).rsqrt()
    return h, c * rs, rs, w.double()


def _check(x, r, w, b, dy, dh, outs, grads, eps=EPS):
    h, n, rs, wd = _parts(x, r, w, eps)
    rows, dim = x.shape
    s = dim / 256 + 16 if _swept(dim) else 48
    bd = 0.0 if b is None else b.double()
    y = outs[-1]
    if r is not None:
        assert torch.equal(outs[0], h)
    ref = n * wd + bd
    off_n = (s / 2 + 11) * n.abs() + s
    tol = U * (off_n * wd.abs() + (n * wd).abs() + 2 * ref.abs()) + HALF[y.dtype] * ref.abs() * 1.01 + 1e-38
    assert y.dtype == x.dtype and bool(((y.double() - ref).abs() <= tol).all())
    if grads is None:
        return
    dx, dw, db = grads["x"], grads["w"], grads.get("b")
    dyd = dy.double()
    g = dyd * wd
    mg, mgn = g.mean(-1, keepdim=True), (g * n).mean(-1, keepdim=True)
    ref = rs * (g - mg - n * mgn) + (0.0 if dh is None else dh.double())
    mag, magn = g.abs().mean(-1, keepdim=True), (g * n).abs().mean(-1, keepdim=True)
    tol = U * (s + 90) * rs * (g.abs() + mag + n.abs() * (magn + mag) + magn) + (2 * U + 1.01 * HALF[dx.dtype]) * ref.abs() + 1e-38
    assert bool(((dx.double() - ref).abs() <= tol).all())
    if r is not None:
        assert torch.equal(grads["r"], dx)
    k = 64 + rows / 2048
    mean = (h.double().mean(-1, keepdim=True).abs() * rs) if _swept(dim) else 0.0  # room for a mean as it is stored, which the sweeps do without
    ref = (dyd * n).sum(0)
    tol = U * (dyd.abs() * (off_n + 2 * mean + k * n.abs())).sum(0) + 1.01 * HALF[dw.dtype] * ref.abs() + 1e-38
    assert dw.dtype == w.dtype and bool(((dw.double() - ref).abs() <= tol).all())
    if db is not None:
        ref = dyd.sum(0)
        tol = U * k * dyd.abs().sum(0) + 1.01 * HALF[db.dtype] * ref.abs() + 1e-38
        assert bool(((db.double() - ref).abs() <= tol).all())


def _run(x, r, w, b, dy, dh, eps=EPS):
    """Outputs and the gradients of all inputs, by name."""
    leaves = {k: t.detach().requires_grad_() for k, t in (("x", x), ("r", r), ("w", w), ("b", b)) if t is not None}
    out = layernorm(leaves["x"], leaves["w"], leaves.get("b"), residual=leaves.get("r"), eps=eps)
    outs = list(out) if r is not None else [out]
    grads = torch.autograd.grad(outs, list(leaves.values()), [dh, dy] if r is not None else [dy])
    return [o.detach() for o in outs], dict(zip(leaves, grads))


DIMS = [1, 2, 7, 8, 9, 15, 64, 77, 512, 513, 768, 1003, 1024, 1025, 2047, 2048, 2049, 4096, 4100, 5000, 8192, 8193, 16384, 16385]


@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("dtype,wdtype,residual,bias", [(BF16, F32, True, True), (BF16, BF16, False, False),
                                                        (F32, F32, True, False), (F32, BF16, False, True)])
def test_forward_and_backward(dev, dim, dtype, wdtype, residual, bias):
    for rows in (1, 5, 67):
        args = _inputs(dev, rows, dim, dtype, wdtype, residual, bias, seed=dim + rows)
        outs, grads = _run(*args)
        _check(*args, outs, grads)
        with torch.no_grad():
            plain = layernorm(args[0], args[2], args[3], residual=args[1], eps=EPS)
        for a, o in zip(plain if residual else [plain], outs):
            assert torch.equal(a, o)  # the call that records nothing gives the same bits


@pytest.mark.parametrize("rows,dim,dtype", [(8192, 768, BF16), (3001, 1003, F32), (20000, 130, BF16), (2500, 3000, F32)])
def test_many_rows(dev, rows, dim, dtype):
    args = _inputs(dev, rows, dim, dtype, F32, True, True, seed=3)
    outs, grads = _run(*args)
    _check(*args, outs, grads)
    again = _run(*args)
    assert all(torch.equal(grads[k], again[1][k]) for k in grads)  # sums in a fixed order


@pytest.mark.parametrize("dim", [8, 100, 768, 3000])
def test_a_mean_far_from_zero_keeps_precision(dev, dim):
    args = _inputs(dev, 9, dim, F32, F32, False, True, seed=5, loc=1e4)
    outs, grads = _run(*args)
    _check(*args, outs, grads)


@pytest.mark.parametrize("dim", [3, 96, 1003, 5000])
def test_rows_without_deviation(dev, dim):
    x = torch.full((4, dim), 3.25, device=dev)
    w, b = torch.randn(dim, device=dev), torch.randn(dim, device=dev)
    # dim equal values: their sum is rounded, the corrected mean is not off by more than its half step
    y = layernorm(x, w, b, eps=1e-5)
    assert bool(((y - b).abs() <= 3.25 * 2.0**-23 * 1e-5**-0.5 * w.abs() + U * b.abs() * 2).all())


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("dim", [5, 77, 768, 4100])
def test_a_bad_row_stays_alone(dev, dtype, dim):
    args = _inputs(dev, 11, dim, dtype, F32, True, True, seed=7)
    good, _ = _run(*args)
    x = args[0].clone()
    x[3, dim // 2] = float("nan")
    x[7, 0] = float("inf")
    bad, grads = _run(x, *args[1:])
    keep = torch.tensor([i not in (3, 7) for i in range(11)], device=dev)
    for a, b in zip(good, bad):
        assert torch.equal(a[keep], b[keep])
    assert bool(bad[1][~keep].isnan().all()) and bool(grads["w"].isnan().all()) and bool(grads["x"][keep].isfinite().all())
    assert bool(grads["b"].isfinite().all())


def test_layouts_and_leading_dimensions(dev):
    x0 = torch.randn(3, 50, 2, 130, device=dev, dtype=BF16)
    w, b = torch.randn(130, device=dev), torch.randn(130, device=dev)
    for x in (x0, x0.transpose(0, 1), x0[:, ::2], x0[..., 1:], x0[..., :1, :]):
        wx, bx = w[:x.shape[-1]], b[:x.shape[-1]]
        ref = layernorm(x.contiguous(), wx.contiguous(), bx.contiguous())
        assert torch.equal(layernorm(x, wx, bx), ref) and ref.shape == x.shape
    flat = torch.randn(7 * 96 + 1, device=dev)
    x = flat[1:].view(7, 96)  # rows that start between 16-byte boundaries
    wide = torch.randn(97, device=dev)
    assert torch.equal(layernorm(x, wide[1:], wide[:96]), layernorm(x.clone(), wide[1:].clone(), wide[:96].clone()))


def test_one_row_and_one_tensor_twice(dev):
    x, w, b = (torch.randn(96, device=dev, requires_grad=True) for _ in range(3))
    y = layernorm(x, w, b)
    assert y.shape == (96,) and torch.equal(y, layernorm(x[None], w, b)[0])
    h, y = layernorm(x, w, residual=x)  # both inputs' gradients meet in one leaf
    g = torch.randn(96, device=dev)
    dx, = torch.autograd.grad(y, x, g)
    x2 = (x.detach() * 2).requires_grad_()
    assert torch.equal(h, x2) and torch.equal(dx, 2 * torch.autograd.grad(layernorm(x2, w), x2, g)[0])


def test_nothing_to_norm(dev):
    w, b = torch.ones(64, device=dev, requires_grad=True), torch.ones(64, device=dev, requires_grad=True)
    x = torch.zeros(0, 64, device=dev, requires_grad=True)
    y = layernorm(x, w, b)
    assert y.shape == (0, 64)
    dx, dw, db = torch.autograd.grad(y.sum(), (x, w, b))
    assert dx.shape == (0, 64) and not dw.any() and not db.any()


def test_one_output_used(dev):
    args = _inputs(dev, 33, 200, F32, F32, True, True, seed=9)
    x, r, w, b = (t.clone().requires_grad_() for t in args[:4])
    h, y = layernorm(x, w, b, residual=r)
    dx, = torch.autograd.grad(y, x, args[4], retain_graph=True)
    ref = _run(*args[:4], args[4], torch.zeros_like(args[4]))[1]["x"]
    assert torch.equal(dx, ref)
    only_h = torch.autograd.grad(h, (x, r, w, b), args[5])
    assert torch.equal(only_h[0], args[5]) and not only_h[2].any() and not only_h[3].any()


def test_the_gradient_against_differences(dev):
    """Along a direction, in 64 bits through the reference: (f(x + t v) - f(x - t v)) / 2 t, off by O(t^2)."""
    args = _inputs(dev, 6, 40, F32, F32, False, True, seed=11)
    _, grads = _run(*args)
    g = torch.Generator().manual_seed(1)
    x, w, b, dy = (t.double() for t in (args[0], args[2], args[3], args[4]))
    v = [torch.randn(t.shape, generator=g, dtype=torch.float64).to(dev) for t in (x, w, b)]
    t = 1e-4
    f = lambda s: (layernorm_reference(x + s * v[0], w + s * v[1], b + s * v[2]) * dy).sum()
    slope = (f(t) - f(-t)) / (2 * t)
    mine = sum((grads[k].double() * d).sum() for k, d in zip("xwb", v))
    assert abs(float(slope - mine)) <= 1e-5 * sum(float((grads[k].double() * d).abs().sum()) for k, d in zip("xwb", v))


def test_another_stream_and_a_captured_step(dev):
    args = _inputs(dev, 300, 768, BF16, F32, True, True, seed=13)
    ref, ref_grads = _run(*args)
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        outs, grads = _run(*args)
        leaves = [t.clone().requires_grad_() for t in args[:4]]

        def step():
            out = layernorm(leaves[0], leaves[2], leaves[3], residual=leaves[1])
            return [*out, *torch.autograd.grad(out, leaves, [args[5], args[4]])]

        step()
    side.synchronize()
    assert torch.equal(outs[1], ref[1]) and all(torch.equal(grads[k], ref_grads[k]) for k in grads)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for k in range(3):
        with torch.no_grad():
            leaves[0].copy_(args[0] * (1 + k))
        graph.replay()
        want, want_grads = _run(leaves[0].detach(), *args[1:])
        torch.cuda.synchronize()
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
        assert all(torch.equal(a, want_grads[n]) for a, n in zip(out[2:], "xrwb"))


def test_capture_refuses_leaves_that_an_eager_graph_holds(dev):
    x, w = torch.randn(4, 64, device=dev, requires_grad=True), torch.ones(64, device=dev, requires_grad=True)
    held = layernorm(x, w)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="holds one of its leaves"):
        with torch.cuda.graph(graph):
            layernorm(x, w)
    del held


def test_forward_mode_is_refused(dev):
    import torch.autograd.forward_ad as fwd

    x, w = torch.randn(4, 64, device=dev), torch.randn(64, device=dev)
    with fwd.dual_level(), pytest.raises((RuntimeError, NotImplementedError)):
        layernorm(x, fwd.make_dual(w, torch.ones_like(w)))


@pytest.mark.parametrize("dim", [2, 3, 7, 16385, 20000])
@pytest.mark.parametrize("rows", [9, 700])
@pytest.mark.parametrize("residual", [False, True])
def test_a_mean_far_from_zero_keeps_precision_in_the_sweeps(dev, dim, rows, residual):
    """Rows of fewer than 8 and of more than 16384 elements: the weight's gradient takes the normed values of the forward, without a
    term for the mean's rounding, which at a mean of 10^4 deviations is up to 2^-11 of one: 8192 u."""
    x, r, w, b, dy, dh = args = _inputs(dev, rows, dim, F32, F32, residual, True, seed=15, loc=1e4)
    outs, grads = _run(*args)
    _check(*args, outs, grads)
    _, n, _, _ = _parts(x, r, w, EPS)
    s = dim / 256 + 16
    dyd, ref = dy.double(), (dy.double() * n).sum(0)
    tol = U * (dyd.abs() * ((s / 2 + 11) * n.abs() + s + (64 + rows / 256) * n.abs())).sum(0) + 1.01 * HALF[F32] * ref.abs() + 1e-38
    assert bool(((grads["w"].double() - ref).abs() <= tol).all())


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_only_the_residual_stream_used(dev, dtype):
    """h's own gradient passes as it is, from rows with a NaN or an infinity too, and the parameters get none."""
    args = _inputs(dev, 33, 200, dtype, F32, True, True, seed=17)
    x, r, w, b = (t.clone().requires_grad_() for t in args[:4])
    with torch.no_grad():
        x[3, 5], x[7, 0] = float("nan"), float("inf")
    h, _ = layernorm(x, w, b, residual=r)
    dx, dr, dw, db = torch.autograd.grad(h, (x, r, w, b), args[5])
    assert torch.equal(dx, args[5]) and torch.equal(dr, args[5]) and not dw.any() and not db.any()


@pytest.mark.parametrize("scale", [1e-18, 1e-19, 1e-20])
@pytest.mark.parametrize("dim", [5, 96, 1003, 3000, 16385])
def test_deviations_whose_squares_are_subnormal(dev, dim, scale):
    """With eps = 0 the variance may lie below the normal floats. Its squares and their mean are each rounded to a multiple of 2^-149 there, so
    it is off by at most that, and the inverse deviation by half of 2^-149 / var (all of it allowed) beside the usual."""
    x, _, w, _, dy, _ = _inputs(dev, 7, dim, F32, F32, False, False, seed=19)
    x = (x * scale).requires_grad_()
    w.requires_grad_()
    y = layernorm(x, w, eps=0.0)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    _, n, rs, wd = _parts(x.detach(), None, w.detach(), 0.0)
    s = dim / 256 + 16 if _swept(dim) else 48
    more = 2.0**-149 * rs.square()
    tol = U * ((s / 2 + 11) * n.abs() + s + 2 * n.abs()) * wd.abs() + more * (n * wd).abs() + U * (n * wd).abs()
    assert bool(((y.detach().double() - n * wd).abs() <= tol).all())
    g = dy.double() * wd
    ref = rs * (g - g.mean(-1, keepdim=True) - n * (g * n).mean(-1, keepdim=True))
    off = (U * (s + 90) + more) * 3 * rs * (g.abs() + g.abs().mean(-1, keepdim=True) + n.abs() * (g * n).abs().mean(-1, keepdim=True))
    off = off + (U * (s + 90)) * rs * (n.abs() * g.abs().mean(-1, keepdim=True) + (g * n).abs().mean(-1, keepdim=True))
    assert bool(((dx.double() - ref).abs() <= off).all())
    ref = (dy.double() * n).sum(0)
    off = (dy.double().abs() * (U * ((s / 2 + 11) * n.abs() + s + 64 * n.abs()) + more * n.abs())).sum(0) + U * 1.01 * ref.abs()
    assert bool(((dw.double() - ref).abs() <= off).all())
