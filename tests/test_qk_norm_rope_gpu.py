"""GPU tests of the heads' split, norm and rotation (csrc/heads_rope.hip), forward and backward, against
the same formulas in 64 bits (qk_norm_rope_reference on float64 copies of the inputs).

Tolerances, in units u = 2^-24 of f32's half step, before the output's own rounding (half a step of its
type). A lane adds at most 16 squares (or 8), the group's sum 6 more: 22 u in the mean square, 11 in its
root, and 5 for the division, the added eps and the rsqrt: r is within 16 u. A rotated value lo c - hi s
adds two products and a sum: 20 u (|lo| + |hi|). A gradient adds the same 20 u to r |w| (|g_lo| + |g_hi|)
(24 allowed), and its mean term 22 u for the sum, 3 * 16 for r^3 and a few for the products: 80 u of
r^3 |x| mean|du w x|. A weight's gradient is summed over at most 128 additions in a row (per lane, group,
wave and slice) of terms within 24 u."""

import pytest
import torch

from ferrite.kernels.flash_attention import flash_attention
from ferrite.kernels.heads import split_heads
from ferrite.kernels.qk_norm_rope import qk_norm_rope, qk_norm_rope_reference, rope_tables

pytestmark = pytest.mark.gpu

U = 2.0**-24
HALF = {torch.bfloat16: 2.0**-8, torch.float32: 2.0**-24}
BF16, F32 = torch.bfloat16, torch.float32


def _inputs(dev, b, s, h, hkv, d, rot, dtype, wdtype=F32, rows=None, seed=0):
    g = torch.Generator().manual_seed(seed)
    mk = lambda *shape: torch.randn(*shape, generator=g)
    qkv = mk(b, s, (h + 2 * hkv) * d).to(dev, dtype)
    wq, wk = ((1 + 0.2 * mk(d)).to(dev, wdtype) for _ in range(2))
    cos, sin = rope_tables(rows or max(s, 1), rot, device=dev)
    return qkv, wq, wk, cos, sin


def _exact(qkv, wq, wk, cos, sin, **kw):
    return qk_norm_rope_reference(qkv.double(), wq.double(), wk.double(), cos.double(), sin.double(), **kw)


def _sizes(h, d, rot, inter):
    """[.., S, D] absolute sums |lo| + |hi| of each rotated element's pair, of a head-major tensor."""
    a = h.abs().clone()
    first = slice(0, rot, 2) if inter else slice(0, rot // 2)
    second = slice(1, rot, 2) if inter else slice(rot // 2, rot)
    both = a[..., first] + a[..., second]
    a[..., first], a[..., second] = both, both
    return a


def _check_forward(out, qkv, wq, wk, cos, sin, h, hkv, inter, positions=None, eps=1e-6):
    kw = dict(n_head=h, n_kv_head=hkv, positions=positions, eps=eps, interleaved=inter)
    ref = _exact(qkv, wq, wk, cos, sin, **kw)
    flat = _exact(qkv, wq, wk, torch.ones_like(cos), torch.zeros_like(sin), **kw)  # normed, not rotated
    for o, r, n in zip(out[:2], ref[:2], flat[:2]):
        assert o.shape == r.shape and o.dtype == qkv.dtype and o.is_contiguous()
        tol = 20 * U * _sizes(n, n.shape[-1], 2 * cos.shape[1], inter) + HALF[o.dtype] * r.abs() * 1.01
        assert bool(((o.double() - r).abs() <= tol).all())
    assert out[2].is_contiguous() and torch.equal(out[2].double(), ref[2])


CASES = [
    # b, s, h, hkv, d, rot, dtype, interleaved
    (1, 1, 4, 4, 128, 128, BF16, False),
    (2, 37, 3, 1, 64, 64, BF16, False),
    (2, 130, 12, 12, 64, 64, BF16, True),
    (1, 65, 8, 2, 128, 64, BF16, False),
    (3, 33, 5, 5, 80, 40, BF16, False),    # units that fill no power of two; the rotated part no whole vectors: by elements
    (3, 33, 5, 5, 80, 32, BF16, False),    # the same heads in vectors
    (1, 19, 2, 2, 256, 256, BF16, False),
    (1, 9, 2, 1, 512, 256, BF16, True),
    (2, 11, 1, 1, 32, 16, BF16, True),
    (2, 100, 3, 3, 96, 96, F32, False),
    (3, 101, 5, 5, 80, 40, F32, True),
    (1, 7, 2, 2, 512, 512, F32, False),
    (2, 13, 2, 1, 10, 6, F32, True),       # by elements
    (2, 13, 2, 1, 2, 2, F32, False),
    (1, 21, 3, 1, 130, 130, BF16, False),  # by elements, over 128
    (1, 5, 1, 1, 258, 4, F32, False),
    (9, 700, 7, 3, 64, 64, BF16, False),   # two heads to a wave
    (4, 701, 9, 5, 8, 8, F32, False),
]


@pytest.mark.parametrize("b,s,h,hkv,d,rot,dtype,inter", CASES)
def test_forward_and_gradients(dev, b, s, h, hkv, d, rot, dtype, inter):
    qkv, wq, wk, cos, sin = _inputs(dev, b, s, h, hkv, d, rot, dtype, seed=s + d)
    leaves = [t.clone().requires_grad_() for t in (qkv, wq, wk)]
    out = qk_norm_rope(*leaves, cos, sin, n_head=h, n_kv_head=hkv, interleaved=inter)
    _check_forward(out, qkv, wq, wk, cos, sin, h, hkv, inter)
    g = torch.Generator().manual_seed(1)
    grads = [torch.randn(t.shape, generator=g).to(dev, dtype) for t in out]
    got = torch.autograd.grad(out, leaves, grads)
    again = torch.autograd.grad(qk_norm_rope(*leaves, cos, sin, n_head=h, n_kv_head=hkv, interleaved=inter), leaves, grads)
    assert all(torch.equal(x, y) for x, y in zip(got, again))
    ref_leaves = [t.double().requires_grad_() for t in (qkv, wq, wk)]
    ref_out = qk_norm_rope_reference(*ref_leaves, cos.double(), sin.double(), n_head=h, n_kv_head=hkv, interleaved=inter)
    ref = torch.autograd.grad(ref_out, ref_leaves, [t.double() for t in grads])
    _check_gradients(got, ref, grads, qkv, wq, wk, h, hkv, rot, inter)


def _check_gradients(got, ref, grads, qkv, wq, wk, h, hkv, rot, inter, eps=1e-6):
    b, s, _ = qkv.shape
    d = wq.shape[0]
    x = qkv.double().reshape(b, s, h + 2 * hkv, d)
    r = torch.rsqrt(x.square().mean(-1, keepdim=True) + eps)
    w = torch.cat([wq.double().expand(h, d), wk.double().expand(hkv, d), torch.zeros(hkv, d, device=x.device)])
    gs = torch.cat([_sizes(t.double(), d, rot, inter) for t in grads], 1).transpose(1, 2)  # [B, S, heads, D]
    direct = r * w.abs() * gs
    mean = (gs * w.abs() * x.abs()).mean(-1, keepdim=True)
    rd = ref[0].reshape(x.shape)
    tol = U * (24 * direct + 80 * r**3 * x.abs() * mean) + HALF[qkv.dtype] * rd.abs() * 1.01
    assert got[0].dtype == qkv.dtype
    assert bool(((got[0].double().reshape(x.shape) - rd).abs() <= tol).all())
    terms = (gs * x.abs() * r).sum((0, 1))  # [heads, D]
    for o, e, t in ((got[1], ref[1], terms[:h]), (got[2], ref[2], terms[h:h + hkv])):
        assert bool(((o.double() - e).abs() <= 152 * U * t.sum(0) + HALF[o.dtype] * e.abs() * 1.01).all())


@pytest.mark.parametrize("dtype,wdtype", [(BF16, BF16), (F32, BF16), (BF16, F32)])
def test_positions_strides_and_weight_types(dev, dtype, wdtype):
    """Views that a program has: columns of a wider row, every second token, sequences that overlap in nothing but
    their order, an address off 16 bytes; positions per sequence and per token."""
    b, s, h, hkv, d, rot = 3, 17, 4, 2, 64, 32
    width = (h + 2 * hkv) * d
    big, wq, wk, cos, sin = _inputs(dev, b, 2 * s, h, hkv, d + 3, rot, dtype, wdtype, rows=900)
    wq, wk = wq[:d], wk[3:]
    views = [big[:, ::2, 8:8 + width], big[:, 1::2, 1:1 + width], big.transpose(0, 1)[:b, :3, :width],
             big[..., :width].flip(0)[:, :s], big[:1, :s, :width].expand(b, s, width)]
    for i, view in enumerate(views):
        n = view.shape[1]
        pos = torch.randint(0, 900, (view.shape[0], n), generator=torch.Generator().manual_seed(i)).int().to(dev)
        for p in (pos, pos[0], pos.t().contiguous().t()):
            leaves = [view.detach(), wq.detach().requires_grad_(), wk.detach().requires_grad_()]
            out = qk_norm_rope(*leaves, cos, sin, n_head=h, n_kv_head=hkv, positions=p)
            full = p.expand(view.shape[0], n)
            _check_forward([t.detach() for t in out], view.contiguous(), wq, wk, cos, sin, h, hkv, False, full)
        dense = view.clone().requires_grad_()
        via = view.detach().requires_grad_()
        grads = [torch.randn_like(t) for t in out]
        a = torch.autograd.grad(qk_norm_rope(via, wq, wk, cos, sin, n_head=h, n_kv_head=hkv, positions=pos), via, grads)
        e = torch.autograd.grad(qk_norm_rope(dense, wq, wk, cos, sin, n_head=h, n_kv_head=hkv, positions=pos), dense, grads)
        assert torch.allclose(a[0].float(), e[0].float(), rtol=2 * HALF[dtype] * 2, atol=1e-5)


def test_positions_outside_the_tables(dev):
    qkv, wq, wk, cos, sin = _inputs(dev, 2, 6, 2, 1, 64, 64, F32, rows=10)
    pos = torch.tensor([[0, 9, 10, -1, 3, 2**31 - 1], [1, 2, 3, 4, 5, -(2**31)]], dtype=torch.int32, device=dev)
    q, k, v = qk_norm_rope(qkv, wq, wk, cos, sin, n_head=2, n_kv_head=1, positions=pos)
    bad = ((pos < 0) | (pos >= 10))[:, None, :, None]
    for t in (q, k):
        assert torch.equal(torch.isnan(t), bad.expand_as(t))
    ok = qk_norm_rope(qkv, wq, wk, cos, sin, n_head=2, n_kv_head=1, positions=pos.clamp(0, 9))
    for t, r in zip((q, k, v), ok):
        assert torch.equal(torch.where(bad, 0.0, t) if t is not v else t, torch.where(bad, 0.0, r) if t is not v else r)


def test_partial_and_broadcast_gradients(dev):
    """Outputs that nothing reads, gradients that are expanded or strided."""
    qkv, wq, wk, cos, sin = _inputs(dev, 2, 40, 4, 2, 64, 64, BF16)
    leaves = [t.requires_grad_() for t in (qkv, wq, wk)]
    kw = dict(n_head=4, n_kv_head=2)
    zero = [torch.zeros(2, n, 40, 64, device=dev, dtype=BF16) for n in (4, 2, 2)]
    one = torch.randn(2, 4, 40, 64, device=dev).to(BF16)
    for i, g in ((0, one), (1, one[:, :2]), (2, one[:, :2]), (0, one[:, :1].expand(2, 4, 40, 64)),
                 (1, torch.ones((), device=dev, dtype=BF16).expand(2, 2, 40, 64)), (2, one.transpose(0, 1)[:2, :2])):
        if g.shape != zero[i].shape:
            g = g.reshape(2, 2, 40, 64)
        out = qk_norm_rope(*leaves, cos, sin, **kw)
        got = torch.autograd.grad(out[i], leaves, g, allow_unused=True)
        full = [g.contiguous() if j == i else z for j, z in enumerate(zero)]
        ref = torch.autograd.grad(qk_norm_rope(*leaves, cos, sin, **kw), leaves, full)
        assert all(torch.equal(a, b) for a, b in zip(got, ref))


def test_gradient_matches_differences(dev):
    """Central differences of the f32 kernel along random directions. The step h leaves h^2 / 6 of the third derivative and
    the outputs' rounding over 2 h: 1e-2 of values of order one on both counts is 3e-4 of the slope's size."""
    qkv, wq, wk, cos, sin = _inputs(dev, 2, 9, 3, 1, 32, 16, F32)
    leaves = [t.requires_grad_() for t in (qkv, wq, wk)]
    f = lambda a, x, y: qk_norm_rope(a, x, y, cos, sin, n_head=3, n_kv_head=1, interleaved=True)
    out = f(*leaves)
    grads = [torch.randn_like(t) for t in out]
    got = torch.autograd.grad(out, leaves, grads)
    with torch.no_grad():
        for i, g in enumerate(got):
            for seed in range(4):
                v = torch.randn(g.shape, generator=torch.Generator().manual_seed(seed)).to(dev)
                h = 1e-2 / float(v.norm())
                moved = [[t + sign * h * v if j == i else t for j, t in enumerate(leaves)] for sign in (1, -1)]
                up, down = (sum((o.double() * w.double()).sum() for o, w in zip(f(*m), grads)) for m in moved)
                slope, size = (g.double() * v.double()).sum(), float(g.double().norm() * v.double().norm())
                assert abs(float((up - down) / (2 * h) - slope)) <= 1e-3 * size


def test_empty_and_no_grad(dev):
    for b, s in ((0, 5), (3, 0)):
        qkv, wq, wk, cos, sin = _inputs(dev, b, s, 2, 1, 64, 64, BF16, rows=8)
        leaves = [t.requires_grad_() for t in (qkv, wq, wk)]
        out = qk_norm_rope(*leaves, cos, sin, n_head=2, n_kv_head=1)
        assert [tuple(t.shape) for t in out] == [(b, 2, s, 64), (b, 1, s, 64), (b, 1, s, 64)]
        got = torch.autograd.grad(out, leaves, [torch.zeros_like(t) for t in out])
        assert got[0].shape == qkv.shape and not got[1].any() and not got[2].any()
    qkv, wq, wk, cos, sin = _inputs(dev, 1, 4, 2, 1, 64, 64, BF16)
    with torch.no_grad():
        assert not any(t.requires_grad for t in qk_norm_rope(qkv.requires_grad_(), wq, wk, cos, sin, n_head=2, n_kv_head=1))


def test_large_and_infinite_values(dev):
    """One head's infinity, NaN or overflow stays in it."""
    qkv, wq, wk, cos, sin = _inputs(dev, 1, 8, 2, 2, 64, 64, F32)
    clean = qk_norm_rope(qkv, wq, wk, cos, sin, n_head=2)
    x = qkv.clone()
    x[0, 1, 5], x[0, 2, 64 + 7], x[0, 3, 128 + 1] = float("inf"), float("nan"), 1e30  # q head 0, q head 1, k head 0
    q, k, v = qk_norm_rope(x, wq, wk, cos, sin, n_head=2)
    hit = torch.zeros(1, 2, 8, 1, dtype=torch.bool, device=dev)
    hit[0, 0, 1], hit[0, 1, 2] = True, True
    assert torch.equal(torch.where(hit, 0.0, q), torch.where(hit, 0.0, clean[0])) and torch.equal(v, clean[2])
    assert torch.isnan(q[0, 1, 2]).all() and torch.equal(k[0, 1], clean[1][0, 1])
    zero = torch.zeros_like(qkv)
    assert not any(t.any() for t in qk_norm_rope(zero, wq, wk, cos, sin, n_head=2))


def test_streams_and_graph(dev):
    qkv, wq, wk, cos, sin = _inputs(dev, 2, 64, 4, 4, 64, 64, BF16)
    leaves = [t.requires_grad_() for t in (qkv, wq, wk)]
    grads = [torch.randn(2, 4, 64, 64, device=dev).to(BF16) for _ in range(3)]

    def step():
        out = qk_norm_rope(*leaves, cos, sin, n_head=4)
        return [*(t.detach() for t in out), *torch.autograd.grad(out, leaves, grads)]

    eager = [t.clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = [t.clone() for t in step()]
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(eager, other))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in range(3):
        with torch.no_grad():
            qkv.copy_(torch.randn(qkv.shape, generator=torch.Generator().manual_seed(seed)).to(dev))
        graph.replay()
        got = [t.clone() for t in out]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, step()))
    graph.reset()


@pytest.mark.parametrize("rows", [16, 32])
def test_capture_refuses_leaves_that_an_eager_graph_holds(dev, rows):
    """While an eager graph of the leaves lives, no pass that records a backward begins in a capture; once it is dropped,
    one that takes the leaves twice does, and its backward() replays as it runs. Of 16 rows the tables are too short for
    some of the second call's positions: NaN in their gradients and the weights'."""
    qkv, wq, wk, cos, sin = _inputs(dev, 2, 16, 4, 4, 64, 64, F32, rows=rows)
    leaves = [t.requires_grad_() for t in (qkv, wq, wk)]
    for t in leaves:
        t.grad = torch.zeros_like(t)

    def step():
        for t in leaves:
            t.grad.zero_()
        outs = [o for p in places for o in qk_norm_rope(*leaves, cos, sin, n_head=4, positions=p)]
        torch.autograd.backward(outs, grads)

    grads = [torch.randn(2, 4, 16, 64, device=dev) for _ in range(6)]
    places = [torch.arange(16, dtype=torch.int32, device=dev), torch.arange(16, dtype=torch.int32, device=dev) + 7]
    step()
    want = [t.grad.clone() for t in leaves]
    assert bool(torch.isnan(want[1]).any()) == (rows == 16) and not bool(torch.isnan(want[0]).all())
    alive = qk_norm_rope(*leaves, cos, sin, n_head=4)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="outside this capture"):
        with torch.cuda.graph(graph):
            qk_norm_rope(*leaves, cos, sin, n_head=4)
    with torch.no_grad():
        assert torch.equal(qk_norm_rope(*leaves, cos, sin, n_head=4)[0], alive[0])
    del alive
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for _ in range(3):
        for t in leaves:
            t.grad.fill_(3)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(t.grad.nan_to_num(7), w.nan_to_num(7)) for t, w in zip(leaves, want))
    graph.reset()


def test_feeds_attention_like_split_heads(dev):
    """With unit weights' norm undone the heads are split_heads'; and the outputs go straight into flash attention."""
    qkv, wq, wk, cos, sin = _inputs(dev, 2, 128, 4, 4, 64, 64, BF16)
    q, k, v = qk_norm_rope(qkv, wq, wk, cos, sin, n_head=4)
    assert torch.equal(v, split_heads(qkv, 3, 4)[2])
    leaf = qkv.clone().requires_grad_()
    o = flash_attention(*qk_norm_rope(leaf, wq, wk, cos, sin, n_head=4))
    g = torch.randn_like(o)
    got = torch.autograd.grad(o, leaf, g)[0]
    ref = qkv.float().requires_grad_()
    rq, rk, rv = qk_norm_rope_reference(ref, wq, wk, cos, sin, n_head=4)
    s = (rq @ rk.transpose(-1, -2).contiguous()) / 8
    s = s.masked_fill(torch.ones(128, 128, dtype=torch.bool, device=dev).triu(1), float("-inf"))
    ro = torch.softmax(s, -1) @ rv
    want = torch.autograd.grad(ro, ref, g.float())[0]
    o, ro = o.detach(), ro.detach()
    assert float((o.float() - ro).norm() / ro.norm()) <= 1e-2 and float((got.float() - want).norm() / want.norm()) <= 2e-2


def test_forward_mode_is_refused(dev):
    """There is no rule for tangents: a dual input raises, in whatever place and grad mode, as flash_attention does."""
    import torch.autograd.forward_ad as fwd

    inputs = list(_inputs(dev, 2, 5, 2, 1, 64, 32, F32))
    plain = qk_norm_rope(*inputs, n_head=2, n_kv_head=1)
    with fwd.dual_level():
        for i in range(5):
            for mode in (torch.no_grad, torch.enable_grad):
                dual = [fwd.make_dual(t, torch.ones_like(t)) if j == i else t for j, t in enumerate(inputs)]
                with mode(), pytest.raises(RuntimeError, match="jvp"):
                    qk_norm_rope(*dual, n_head=2, n_kv_head=1)
        heads = torch.randn(1, 2, 128, 64, device=dev)
        with pytest.raises(RuntimeError, match="jvp"):
            flash_attention(fwd.make_dual(heads, torch.ones_like(heads)), heads, heads)
        assert all(torch.equal(a, b) for a, b in zip(qk_norm_rope(*inputs, n_head=2, n_kv_head=1), plain))


# Sizes of training and prefill: up to eight heads to a wave (from 196608 heads on, 13 + 5 + 5 of them 7, 6 and 5 at a time), and more
# groups of tokens than the backward has blocks, so that each goes over several of them, the last round not full. A weight's gradient: a
# lane adds up to 7 heads of each of 5 groups of tokens, then come at most 4, 4, 17 and 6 additions: 66 of the 128 allowed.
@pytest.mark.parametrize("b,s,h,hkv,d,rot,dtype,inter", [
    (3, 2851, 13, 5, 64, 64, BF16, False),   # 16 tokens to a wave
    (3, 2851, 13, 5, 128, 64, BF16, True),
    (1, 8551, 13, 5, 40, 24, F32, False),
    (3, 2851, 13, 5, 130, 130, BF16, False),  # by elements, a token to a wave: five rounds
    (1, 2049, 13, 5, 130, 52, F32, True),     # the same with two heads to a wave
    (1, 4099, 3, 1, 512, 512, F32, False),    # vectors, a token to a wave, one head
    (2, 8200, 8, 2, 512, 256, BF16, False)])  # two tokens to a wave
def test_training_sizes(dev, b, s, h, hkv, d, rot, dtype, inter):
    test_forward_and_gradients(dev, b, s, h, hkv, d, rot, dtype, inter)


# Lanes to a head, and pairs in halves or side by side, that the cases above leave out.
@pytest.mark.parametrize("d,rot,dtype,inter", [
    (32, 16, BF16, False), (256, 128, BF16, True), (80, 40, BF16, True), (130, 4, BF16, True), (24, 16, F32, False), (16, 8, F32, True),
    (64, 64, F32, True), (256, 128, F32, False), (200, 200, F32, True), (512, 256, F32, True)])
def test_layouts(dev, d, rot, dtype, inter):
    test_forward_and_gradients(dev, 2, 75, 3, 2, d, rot, dtype, inter)
