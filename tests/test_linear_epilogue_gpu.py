"""GPU tests of the linear layer with bias, activation and residual (csrc/matmul.hip, skinny.hip, linear.hip), against 64 bits.

Tolerances. A sum of K products in f32 is off by at most (K + 20) u of the sum of their sizes, u = 2^-24, in any order (20 for the
bias and the joining of parts). The activations' slopes are at most 1.13, their curvature at most 0.8; their own evaluation (an exp2, a
reciprocal, the argument's roundings) takes 8 u (1 + |y|). The output is rounded once: half a step of its type. The backward's slope
is that of the pre-activation rounded to x's type: off by 0.8 of half a step of u and of u's own error, and 10 u; of relu, by 1 where
u's error reaches across 0. du is rounded to x's type before the products, and not before the bias's sums, which add at most 64
rows of a lane, 8 lanes, 32 partial rows and 16 waves (120)."""

import pytest
import torch

from ferrite.kernels.matmul import linear, linear_reference

pytestmark = pytest.mark.gpu

U = 2.0**-24
HALF = {torch.bfloat16: 2.0**-8, torch.float32: 2.0**-24}
BF16, F32 = torch.bfloat16, torch.float32


def _inputs(dev, m, k, n, dtype, wdtype, bdtype, bias, residual, seed=0):
    g = torch.Generator().manual_seed(seed)
    mk = lambda *shape: torch.randn(*shape, generator=g)
    return (mk(m, k).to(dev, dtype), (mk(k, n) * k**-0.5).to(dev, wdtype), (0.5 * mk(n)).to(dev, bdtype) if bias else None,
            mk(m, n).to(dev, dtype) if residual else None, mk(m, n).to(dev, dtype))


def _act(u, act):
    """The activation of f64 u and its slope, from the formulas."""
    if act is None:
        return u, torch.ones_like(u)
    if act == "relu":
        return u.clamp(min=0), (u > 0).double()
    z, dz = (u, torch.ones_like(u)) if act == "silu" else (2 * (2 / torch.pi) ** 0.5 * (u + 0.044715 * u**3),
                                                           2 * (2 / torch.pi) ** 0.5 * (1 + 3 * 0.044715 * u**2))
    s = torch.sigmoid(z)
    return u * s, s + u * s * (1 - s) * dz


def _check(x, w, b, r, dy, act, out, grads):
    dt = x.dtype
    xd, wd = x.double(), w.to(dt).double()
    m, k = x.shape
    n = w.shape[1]
    u = xd @ wd
    size = xd.abs() @ wd.abs()
    if b is not None:
        u, size = u + b.double(), size + b.double().abs()
    y, slope = _act(u, act)
    ref = y if r is None else y + r.double()
    off = U * (k + 20) * size
    tol = 1.13 * off + 8 * U * (1 + y.abs()) + 2 * U * ref.abs() + 1.01 * HALF[dt] * ref.abs()
    assert out.shape == ref.shape and out.dtype == dt and bool(((out.double() - ref).abs() <= tol).all())
    if grads is None:
        return
    dyd = dy.double()
    du = dyd * slope
    near = (u.abs() <= off).double() if act == "relu" else 0.8 * (HALF[dt] * u.abs() + off) + 10 * U
    off_du = torch.zeros_like(du) if act is None else dyd.abs() * near + 2 * U * du.abs()
    rounded = off_du if act is None else off_du + 1.01 * HALF[dt] * (du.abs() + off_du)
    dx, dw = du @ wd.t(), xd.t() @ du
    tol = rounded @ wd.abs().t() + U * (n + 20) * (du.abs() @ wd.abs().t()) + 1.01 * HALF[dt] * dx.abs()
    assert grads["x"].dtype == dt and bool(((grads["x"].double() - dx).abs() <= tol).all())
    tol = xd.abs().t() @ rounded + U * (m + 20) * (xd.abs().t() @ du.abs()) + 1.01 * HALF[w.dtype] * dw.abs()
    assert grads["w"].dtype == w.dtype and bool(((grads["w"].double() - dw).abs() <= tol).all())
    if b is not None:
        db = du.sum(0)
        tol = off_du.sum(0) + U * 120 * du.abs().sum(0) + 1.01 * HALF[b.dtype] * db.abs()
        assert grads["b"].dtype == b.dtype and bool(((grads["b"].double() - db).abs() <= tol).all())
    if r is not None:
        assert torch.equal(grads["r"], dy)


def _run(x, w, b, r, dy, act):
    leaves = {k: t.detach().requires_grad_() for k, t in (("x", x), ("w", w), ("b", b), ("r", r)) if t is not None}
    out = linear(leaves["x"], leaves["w"], bias=leaves.get("b"), activation=act, residual=leaves.get("r"))
    return out.detach(), dict(zip(leaves, torch.autograd.grad(out, list(leaves.values()), dy)))


# m, k, n in bf16, by the kernel that the forward's product takes
SIZES_BF16 = [
    (1, 512, 2048), (8, 512, 2048), (3, 1, 1), (8, 513, 100), (33, 1000, 77), (64, 4096, 256), (40, 2048, 264),  # few rows; K cut
    (300, 128, 512), (257, 64, 264), (16384, 64, 256), (16384, 64, 1024), (300, 1088, 512),  # 256- and 128-row tiles; K cut
    (16384, 72, 256), (16384, 72, 1024), (300, 1096, 512),  # ragged K
    (700, 333, 519), (2100, 250, 515), (70, 1500, 9),  # packed operands, rows at odd places
    (300, 200, 512), (65, 30, 7), (70, 64, 130), (100, 8, 8),  # products that leave in f32
]
SIZES_F32 = [(1, 7, 3), (5, 512, 64), (64, 100, 515), (300, 512, 100), (1000, 1003, 515), (2048, 64, 2048), (100, 2048, 70)]


@pytest.mark.parametrize("m,k,n", SIZES_BF16)
@pytest.mark.parametrize("act,wdtype,bdtype,bias,residual", [("gelu", BF16, BF16, True, False), ("silu", F32, F32, True, True),
                                                             ("relu", BF16, F32, False, True), (None, BF16, BF16, True, True)])
def test_bf16(dev, m, k, n, act, wdtype, bdtype, bias, residual):
    x, w, b, r, dy = _inputs(dev, m, k, n, BF16, wdtype, bdtype, bias, residual, seed=m + k + n)
    out, grads = _run(x, w, b, r, dy, act)
    _check(x, w, b, r, dy, act, out, grads)
    with torch.no_grad():
        _check(x, w, b, r, dy, act, linear(x, w, bias=b, activation=act, residual=r), None)
    if bias:
        assert torch.equal(grads["b"], _run(x, w, b, r, dy, act)[1]["b"])  # sums in a fixed order


@pytest.mark.parametrize("m,k,n", SIZES_F32)
@pytest.mark.parametrize("act,wdtype,bias,residual", [("gelu", F32, True, False), ("silu", BF16, True, True),
                                                      ("relu", F32, False, True), (None, F32, True, False)])
def test_f32(dev, m, k, n, act, wdtype, bias, residual):
    x, w, b, r, dy = _inputs(dev, m, k, n, F32, wdtype, F32, bias, residual, seed=m + k + n)
    out, grads = _run(x, w, b, r, dy, act)
    _check(x, w, b, r, dy, act, out, grads)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows,cols", [(1, 1), (9, 7), (1000, 8), (5000, 9), (70000, 24), (63, 4100), (8192, 768), (3, 20000)])
def test_bias_gradient_of_many_rows(dev, dtype, rows, cols):
    """Alone, with a narrow product: what every row adds to a column."""
    x, w, b, _, dy = _inputs(dev, rows, 8, cols, dtype, dtype, F32, True, False, seed=rows)
    _, grads = _run(x, w, b, None, dy, None)
    ref, size = dy.double().sum(0), dy.double().abs().sum(0)
    most = 120 if rows <= 65536 else 120 + rows / 1024
    assert bool(((grads["b"].double() - ref).abs() <= U * most * size).all())


@pytest.mark.parametrize("act", ["relu", "gelu", "silu"])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_far_and_bad_values(dev, act, dtype):
    """One product of one element: u = x w over the whole range, NaN and infinities among it."""
    x = torch.tensor([0.0, -0.0, 1e-30, -1e-30, 30.0, -30.0, 200.0, -200.0, 1e15, -1e15, 3e38, -3e38, float("inf"), float("nan")],
                     device=dev).to(dtype)[:, None]
    w, dy = torch.ones(1, 1, device=dev, dtype=dtype), torch.ones(14, 1, device=dev, dtype=dtype)
    b = torch.zeros(1, device=dev)
    out, grads = _run(x, w, b, None, dy, act)
    y, slope = _act(x.double(), act)
    y = torch.where(x.double() < -1e3, torch.zeros_like(y), y)  # the formula's u times 0
    y, slope = (torch.where(x.double().isinf(), t, v) for t, v in ((x.double(), y), (torch.ones_like(y), torch.where(
        x.double().abs() > 1e3, (x.double() > 0).double(), slope))))
    good = ~x.isnan()
    assert bool(out[~good].isnan().all())
    assert torch.allclose(out[good].double(), y[good], rtol=2 * HALF[dtype] + 1e-6, atol=1e-11)
    assert torch.allclose(grads["x"][good].double(), slope[good], rtol=2 * HALF[dtype] + 1e-6, atol=1e-11)


@pytest.mark.parametrize("m,k,n", [(40, 96, 64), (300, 128, 512), (300, 333, 519)])
def test_a_bad_row_stays_alone(dev, m, k, n):
    x, w, b, r, dy = _inputs(dev, m, k, n, BF16, BF16, F32, True, True)
    good, _ = _run(x, w, b, r, dy, "gelu")
    x2, r2 = x.clone(), r.clone()
    x2[m // 2, k // 3] = float("nan")
    r2[m // 3, n // 2] = float("inf")
    bad, _ = _run(x2, w, b, r2, dy, "gelu")
    same = torch.ones(m, n, dtype=torch.bool, device=dev)
    same[m // 2] = False
    same[m // 3, n // 2] = False
    assert torch.equal(good[same], bad[same]) and bool(bad[m // 2].isnan().all()) and bool(bad[m // 3, n // 2].isinf())


def test_layouts_and_leading_dimensions(dev):
    x, w, b, r, _ = _inputs(dev, 84, 130, 72, BF16, BF16, F32, True, True, seed=1)
    ref = linear(x, w, bias=b, activation="silu", residual=r)
    views = linear(x.t().contiguous().t().view(7, 12, 130), w.t().contiguous().t(), bias=b.repeat(2)[72:], activation="silu",
                   residual=r.view(7, 12, 72))
    assert views.shape == (7, 12, 72) and torch.equal(views.reshape(84, 72), ref)
    room = torch.zeros(84 * 72 + 84 * 130 + 5, device=dev, dtype=BF16)
    x1, r1 = room[1:1 + 84 * 130].view(84, 130), room[3 + 84 * 130:3 + 84 * 202].view(84, 72)  # rows at odd elements
    x1.copy_(x)
    r1.copy_(r)
    assert torch.allclose(linear(x1, w, bias=b, activation="silu", residual=r1).float(), ref.float(), rtol=2**-7, atol=2**-7)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_one_row_and_shared_inputs(dev, dtype):
    x, w, b, r, dy = _inputs(dev, 1, 64, 64, dtype, dtype, F32, True, True, seed=2)
    one = linear(x[0], w, bias=b, activation="gelu", residual=r[0])
    assert one.shape == (64,) and torch.equal(one, linear(x, w, bias=b, activation="gelu", residual=r)[0])
    leaf = x.clone().requires_grad_()  # the residual is the input
    y = linear(leaf, w, bias=b.expand(64), residual=leaf)
    got, = torch.autograd.grad(y, leaf, dy)
    a, c = (x.clone().requires_grad_() for _ in range(2))
    parts = torch.autograd.grad(linear(a, w, bias=b, residual=c), (a, c), dy)
    assert torch.equal(got, parts[0] + parts[1])


def test_nothing_to_multiply(dev):
    w, b = torch.randn(16, 24, device=dev, requires_grad=True), torch.randn(24, device=dev, requires_grad=True)
    x = torch.zeros(0, 16, device=dev, requires_grad=True)
    out = linear(x, w, bias=b, activation="gelu")
    assert out.shape == (0, 24)
    dx, dw, db = torch.autograd.grad(out.sum(), (x, w, b))
    assert dx.shape == (0, 16) and not dw.any() and not db.any()
    assert linear(torch.zeros(5, 16, device=dev), torch.zeros(16, 0, device=dev), activation="relu").shape == (5, 0)


def test_plain_products_are_as_they_were(dev):
    for m, k, n in ((8, 512, 2048), (300, 128, 512), (700, 333, 519)):
        x, w, _, _, _ = _inputs(dev, m, k, n, BF16, BF16, F32, False, False)
        assert torch.equal(linear(x, w), linear(x, w, bias=torch.zeros(n, device=dev)))


def test_the_gradient_against_differences(dev):
    x, w, b, r, dy = _inputs(dev, 9, 33, 21, F32, F32, F32, True, True, seed=4)
    g = torch.Generator().manual_seed(2)
    for act in (None, "gelu", "silu"):
        _, grads = _run(x, w, b, r, dy, act)
        at = [t.double() for t in (x, w, b, r)]
        v = [torch.randn(t.shape, generator=g, dtype=torch.float64).to(dev) for t in at]
        f = lambda s: (linear_reference(at[0] + s * v[0], at[1] + s * v[1], bias=at[2] + s * v[2], activation=act,
                                        residual=at[3] + s * v[3]) * dy.double()).sum()
        slope = (f(1e-4) - f(-1e-4)) / 2e-4
        parts = [(grads[k].double() * d) for k, d in zip("xwbr", v)]
        assert abs(float(slope - sum(p.sum() for p in parts))) <= 1e-5 * sum(float(p.abs().sum()) for p in parts)


@pytest.mark.parametrize("m,k,n,act,dtype", [(8, 512, 256, "gelu", BF16), (300, 1088, 512, "silu", BF16), (300, 333, 519, "relu", BF16),
                                             (130, 200, 90, "gelu", F32)])
def test_another_stream_and_a_captured_step(dev, m, k, n, act, dtype):
    x, w, b, r, dy = _inputs(dev, m, k, n, dtype, dtype, F32, True, True, seed=6)
    ref, ref_grads = _run(x, w, b, r, dy, act)
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out, grads = _run(x, w, b, r, dy, act)
        leaves = [t.clone().requires_grad_() for t in (x, w, b, r)]

        def step():
            y = linear(leaves[0], leaves[1], bias=leaves[2], activation=act, residual=leaves[3])
            return [y, *torch.autograd.grad(y, leaves, dy)]

        step()
    side.synchronize()
    assert torch.equal(out, ref) and all(torch.equal(grads[i], ref_grads[i]) for i in grads)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for i in range(3):
        with torch.no_grad():
            leaves[0].copy_(x * (i + 1))
            leaves[3].copy_(r * (1 - i))
        graph.replay()
        want, want_grads = _run(leaves[0].detach(), w, b, leaves[3].detach(), dy, act)
        torch.cuda.synchronize()
        assert torch.equal(got[0], want) and all(torch.equal(a, want_grads[i]) for a, i in zip(got[1:], "xwbr"))


def test_overlapping_outputs_are_refused_at_the_entry_point(dev):
    from ferrite import _hip

    x, w = torch.randn(8, 16, device=dev), torch.randn(16, 8, device=dev)
    out = torch.empty(2, 8, 8, device=dev)
    lib = _hip.lib()
    call = lambda res, aux: lib.ferrite_internal_linear(x.data_ptr(), w.data_ptr(), None, res, out.data_ptr(), aux, 8, 8, 16, _hip.F32,
                                                        _hip.F32, _hip.F32, 0, None, 0, _hip.stream_of(x))
    assert call(out.data_ptr(), None) != _hip.OK and "overlap" in _hip.last_error()
    assert call(None, out.data_ptr() + 128) != _hip.OK
    assert call(out[1].data_ptr(), out[1].data_ptr()) != _hip.OK


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_gradients_that_are_asked_for(dev, dtype):
    x, w, b, r, dy = _inputs(dev, 70, 96, 40, dtype, dtype, F32, True, True, seed=8)
    _, full = _run(x, w, b, r, dy, "silu")
    for wanted in ("x", "w", "b", "r", "xb", "wr"):
        leaves = {k: t.detach().requires_grad_(k in wanted) for k, t in zip("xwbr", (x, w, b, r))}
        y = linear(leaves["x"], leaves["w"], bias=leaves["b"], activation="silu", residual=leaves["r"])
        got = torch.autograd.grad(y, [leaves[k] for k in wanted], dy)
        assert all(torch.equal(g, full[k]) for g, k in zip(got, wanted))
    leaves = {k: t.detach().requires_grad_() for k, t in zip("xwbr", (x, w, b, r))}  # all record, one is asked for
    y = linear(leaves["x"], leaves["w"], bias=leaves["b"], activation="silu", residual=leaves["r"])
    assert torch.equal(torch.autograd.grad(y, leaves["w"], dy)[0], full["w"])


def test_capture_refuses_leaves_that_an_eager_graph_holds(dev):
    x, w = torch.randn(4, 64, device=dev, requires_grad=True), torch.randn(64, 8, device=dev, requires_grad=True)
    held = linear(x, w, activation="relu")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="holds one of its leaves"):
        with torch.cuda.graph(graph):
            linear(x, w, activation="relu")
    del held


def test_forward_mode_is_refused(dev):
    import torch.autograd.forward_ad as fwd

    x, w = torch.randn(4, 64, device=dev), torch.randn(64, 8, device=dev)
    with fwd.dual_level(), pytest.raises((RuntimeError, NotImplementedError)):
        linear(fwd.make_dual(x, torch.ones_like(x)), w, activation="relu")


def test_bias_gradient_tall_and_wide(dev):
    """Dense rows of 16400 columns, 65536 of them: 64 rows to a lane there too."""
    rows, cols = 65536, 16400
    g = torch.Generator(dev).manual_seed(5)
    x, w, b = (torch.randn(*s, device=dev, generator=g).to(BF16) for s in ((rows, 8), (8, cols), (cols,)))
    dy = torch.randn(rows, cols, device=dev, generator=g, dtype=BF16)
    _, grads = _run(x, w, b.float(), None, dy, None)
    for part in torch.arange(cols, device=dev).split(2050):
        d = dy[:, part].double()
        assert bool(((grads["b"][part].double() - d.sum(0)).abs() <= U * 121 * d.abs().sum(0)).all())


def test_bias_gradient_of_one_value_in_every_row(dev):
    """At 524296 columns, more than the grid has workgroups for. The value's roundings all point one way where a sum passes 512: in one
    line of 1024 rows they make 256 u of the sum, and of 64 rows next to nothing."""
    from ferrite import _hip

    rows, cols, value = 8192, 524296, 1 + 2.0**-15 - 2.0**-23
    lib = _hip.lib()
    dy, db = torch.full((rows, cols), value, device=dev), torch.empty(cols, device=dev)
    ws = torch.empty(lib.ferrite_internal_act_grad_workspace(rows, cols) + 16, dtype=torch.uint8, device=dev)
    rc = lib.ferrite_internal_act_grad(dy.data_ptr(), None, None, db.data_ptr(), rows, cols, 0, _hip.F32, _hip.F32, ws.data_ptr(),
                                       ws.numel(), _hip.stream_of(dy))
    assert rc == _hip.OK
    assert float((db.double() - rows * value).abs().max()) <= U * 121 * rows * value


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_silu_slope_far_below_zero(dev, dtype):
    """s + u s (1 - s) at u = x to its own precision while s is a normal float: 2 |u| u = 2^-24 for the exponent's two roundings, and 16 for
    the rest. Below that it goes on to zero."""
    x = torch.cat([torch.linspace(-86.0, -40.0, 93), torch.tensor([-88.0, -90.0, -100.0, -128.0, -200.0, -1e4, -3e38])]).to(dev, dtype)[:, None]
    w, dy = torch.ones(1, 1, device=dev, dtype=dtype), torch.ones(100, 1, device=dev, dtype=dtype)
    _, grads = _run(x, w, torch.zeros(1, device=dev), None, dy, "silu")
    xd = x.double()
    s = torch.sigmoid(xd)
    slope = s + xd * s * (1 - s)
    tol = U * (2 * xd.abs() + 16) * slope.abs() + 1.01 * HALF[dtype] * slope.abs() + torch.where(xd < -87, 1.5e-36, 0.0)
    assert bool(((grads["x"].double() - slope).abs()[:93] <= tol[:93]).all())
    assert bool((grads["x"].double()[93:].abs() <= 1.1e-36).all())
