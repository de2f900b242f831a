"""GPU tests of the drafted tree's attention (csrc/tree.hip) against the same sums in 64 bits
(tree_attention_reference on float64 copies).

Tolerances. Inputs are N(0, 1), scale 1 / sqrt(D). f32, u = 2^-24: a score is a sum of D products, off by at
most D u sum|q k| / sqrt(D), in practice by sqrt(D) u; taken as 32 u (D = 64 to 256, |q k| / sqrt(D) summed about 0.64 sqrt(D)), plus 3 u
of |score| <= 8 in base-2 units for the scale's and exponent's rounding: 60 u on each weight. The output is a convex sum
of values up to 5: 2 * 60 u * 5, and the f32 sums of the weights and of the products (each term rounded at the size of the
partial sum: n u in the worst case, sqrt(n) u in practice, n <= 16384): 128 u * 1. Together under 800 u = 4.8e-5 at most;
their norms (independent errors) under 1e-6 of the result's. bf16: the weights are rounded to 2^-8 of themselves (independent
errors: 2^-8 * sqrt(sum p^2 v^2) <= 2^-8 max|v| / 1), and the output by half a step of itself; together 2^-8 (|out| + 5
sqrt(sum p^2)) with sum p^2 <= 1: relative to the norm 2^-8 * sqrt(2)."""

import math

import pytest
import torch

from ferrite.kernels.decode_attention import decode_attention
from ferrite.kernels.drafts import accept_drafts, compact_cache
from ferrite.kernels.tree_attention import ancestors, tree_attention, tree_attention_reference
from tests.test_drafts_gpu import trees

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


def _inputs(dev, b, h, hkv, t, length, d, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    mk = lambda *s: torch.randn(*s, generator=g).to(dtype).to(dev)
    return mk(b, h, t, d), mk(b, hkv, t, d), mk(b, hkv, t, d), mk(b, hkv, length, d), mk(b, hkv, length, d)


def _check(dev, q, kn, vn, kc, vc, pos, parents, scale=None):
    """The call against the sums in 64 bits; the caches against the rows that belong in them; a second run bitwise."""
    p, par = torch.tensor(pos, dtype=torch.int32, device=dev), parents.to(dev)
    dbl = [x.double() for x in (q, kn, vn, kc, vc)]
    ref = tree_attention_reference(*dbl, p, par, scale=scale)
    k1, v1, k2, v2 = kc.clone(), vc.clone(), kc.clone(), vc.clone()
    out = tree_attention(q, kn, vn, k1, v1, p, par, scale=scale)
    assert out.shape == q.shape and out.dtype == q.dtype and out.transpose(1, 2).is_contiguous()
    assert torch.equal(k1.double(), dbl[3]) and torch.equal(v1.double(), dbl[4])
    assert torch.equal(torch.isnan(out), torch.isnan(ref))
    got, ref = out.double().nan_to_num(7), ref.nan_to_num(7)
    absent = ~ancestors(par).diagonal(dim1=1, dim2=2)
    assert not (got * absent[:, None, :, None])[(p >= 0) & (p + q.shape[2] <= kc.shape[2])].any()
    size = float(ref.norm())
    if q.dtype == F32:
        assert float((got - ref).abs().max()) <= 4.8e-5
        assert float((got - ref).norm()) <= 1e-6 * size
    else:
        assert bool(((got - ref).abs() <= 2.0**-8 * (ref.abs() + 5.5)).all())
        assert float((got - ref).norm()) <= 2.0**-8 * 1.42 * size
    again = tree_attention(q, kn, vn, k2, v2, p, par, scale=scale)
    assert torch.equal(out.nan_to_num(7), again.nan_to_num(7))
    return out


CASES = [
    # b, h, hkv, t, max_len, d, dtype, pos
    (1, 1, 1, 1, 1, 64, BF16, [0]),
    (2, 2, 2, 1, 300, 64, BF16, [0, 299]),
    (3, 4, 4, 8, 512, 128, BF16, [504, 0, 31]),
    (3, 4, 2, 5, 512, 256, BF16, [507, 32, 33]),
    (2, 3, 1, 7, 700, 64, BF16, [693, 128]),          # 21 rows: two tiles
    (2, 8, 2, 16, 1000, 128, BF16, [984, 511]),       # 64 rows: they share keys through LDS
    (2, 8, 1, 13, 1000, 128, BF16, [512, 513]),       # 104 rows, of the 256 that share keys
    (1, 16, 1, 64, 600, 64, BF16, [536]),             # 1024 rows: four row groups
    (2, 6, 1, 64, 900, 256, BF16, [836, 640]),
    (2, 32, 32, 4, 4100, 128, BF16, [4096, 1]),
    (9, 64, 64, 3, 2050, 64, BF16, [2047, 0, 1, 127, 128, 129, 1023, 1024, 2000]),
    (1, 2, 1, 33, 16384, 64, BF16, [16351]),
    (1, 1, 1, 1, 1, 64, F32, [0]),
    (3, 4, 4, 8, 250, 128, F32, [242, 0, 17]),
    (3, 6, 2, 13, 3001, 64, F32, [2988, 750, 1500]),
    (2, 8, 2, 17, 800, 128, F32, [783, 64]),
    (2, 2, 2, 40, 700, 256, F32, [660, 640]),
    (1, 20, 1, 64, 500, 64, F32, [436]),
    (16, 24, 24, 2, 1030, 64, F32, [1028 - 64 * i for i in range(16)]),
]


@pytest.mark.parametrize("b,h,hkv,t,length,d,dtype,pos", CASES)
def test_matches_64_bits(dev, b, h, hkv, t, length, d, dtype, pos):
    x = _inputs(dev, b, h, hkv, t, length, d, dtype, seed=length + t)
    _check(dev, *x, pos, trees(b, t, 1))
    _check(dev, *x, pos, trees(b, t, 2, absent=0.3), scale=0.3 / d**0.5)


@pytest.mark.parametrize("b,h,hkv,t,length,d,dtype", [
    (70, 2, 2, 3, 1200, 64, F32),      # cut, more than 64 sequences
    (200, 8, 4, 2, 2100, 64, F32),     # cut, more heads than workgroups
    (130, 4, 2, 5, 600, 128, BF16),    # whole
    (70, 3, 1, 30, 800, 64, BF16),     # 90 rows over shared keys: cut
    (80, 6, 2, 60, 300, 128, BF16),    # whole
    (66, 2, 1, 20, 500, 256, BF16)])
def test_many_sequences(dev, b, h, hkv, t, length, d, dtype):
    x = _inputs(dev, b, h, hkv, t, length, d, dtype, seed=b)
    pos = torch.randint(0, length - t + 1, (b,), generator=torch.Generator().manual_seed(b))
    pos[1], pos[b // 2], pos[b - 1], pos[65] = 0, -1, length - t, length
    _check(dev, *x, pos.tolist(), trees(b, t, 1, absent=0.1))


@pytest.mark.parametrize("h,hkv,t,length,d,dtype", [
    (2, 2, 7, 400, 128, BF16), (4, 1, 40, 300, 64, BF16), (5, 1, 52, 1500, 128, BF16), (1, 1, 64, 400, 256, BF16),
    (3, 1, 9, 500, 128, F32)])
def test_scales_of_any_sign(dev, h, hkv, t, length, d, dtype):
    x = _inputs(dev, 2, h, hkv, t, length, d, dtype, seed=t)
    for scale in (-0.7 / d**0.5, 0.0, -0.0):
        _check(dev, *x, [length - t, 40], trees(2, t, 1), scale=scale)


def test_chains_stars_and_forests(dev):
    """A chain, children of one node, roots only, the deepest branch, everything absent; 64 nodes and fewer."""
    for t in (64, 20):
        idx = torch.arange(t)
        lines = [idx - 1, torch.where(idx > 0, 0, -1), torch.full((t,), -1), torch.full((t,), -2), torch.full((t,), t),
                 torch.where(idx > 0, (idx - 1) // 2, -1), torch.where(idx > 1, idx - 2, -1), idx, -1 - idx]
        parents = torch.stack([x.expand(t) for x in lines]).int()
        for dtype in (BF16, F32):
            x = _inputs(dev, len(lines), 4, 2, t, 333, 64, dtype, seed=t)
            _check(dev, *x, [0, 333 - t, 100, 200, 50, 64, 96, 128, 31], parents)


def test_positions_outside_the_cache(dev):
    x = _inputs(dev, 6, 2, 2, 9, 600, 64, BF16)
    _check(dev, *x, [-1, 592, 591, 2**31 - 1, -(2**31), 600], trees(6, 9, 3))


def test_unseen_values_do_not_matter(dev):
    """NaN and infinities in the cache's rows past pos, and in the keys and values of absent nodes."""
    for dtype in (BF16, F32):
        q, kn, vn, kc, vc = _inputs(dev, 3, 4, 2, 12, 600, 64, dtype)
        pos, parents = [40, 588, 301], trees(3, 12, 4, absent=0.4)
        clean = _check(dev, q, kn, vn, kc, vc, pos, parents)
        there = ancestors(parents).diagonal(dim1=1, dim2=2).to(dev)
        for bad in (float("nan"), float("inf"), -float("inf"), torch.finfo(dtype).min):
            k, v, a, c = kc.clone(), vc.clone(), kn.clone(), vn.clone()
            for i, p in enumerate(pos):
                k[i, :, p:], v[i, :, p:] = bad, bad
            a[~there[:, None, :, None].expand_as(a)] = bad
            c[~there[:, None, :, None].expand_as(c)] = bad
            p = torch.tensor(pos, dtype=torch.int32, device=dev)
            assert torch.equal(tree_attention(q, a, c, k, v, p, parents.to(dev)), clean)


@pytest.mark.parametrize("b,h,hkv,t,length,d,dtype,pos", [
    (2, 2, 2, 9, 80, 64, BF16, [70, 0]), (2, 4, 2, 20, 3000, 128, BF16, [2900, 64]), (1, 6, 2, 18, 900, 256, BF16, [800]),
    (2, 8, 2, 40, 200, 128, BF16, [160, 31]), (1, 3, 1, 64, 2000, 64, BF16, [1900]), (1, 2, 1, 40, 700, 256, BF16, [650]),
    (2, 4, 2, 20, 700, 128, F32, [600, 3]), (1, 2, 2, 7, 60, 256, F32, [40])])
def test_what_a_branch_does_not_see_does_not_touch_it(dev, b, h, hkv, t, length, d, dtype, pos):
    """NaN and infinities in keys and values of a node that is there: rows that do not see it keep their bits; those
    that do are what the sums over the nodes they see are."""
    q, kn, vn, kc, vc = _inputs(dev, b, h, hkv, t, length, d, dtype, seed=t)
    parents = torch.where(torch.arange(t) > 1, torch.arange(t) - 2, -1).int().expand(b, t).contiguous()  # two branches
    clean = _check(dev, q, kn, vn, kc, vc, pos, parents)
    k, v = kn.clone(), vn.clone()
    v[:, 0, t // 2, 5], v[:, 0, t // 2 + 2, 5], v[:, -1, t - 1, 9] = float("inf"), -float("inf"), float("nan")
    v[:, 0, t // 2, 8] = -float("inf")
    k[:, -1, t // 2 + 1, 3] = float("nan")
    p, par = torch.tensor(pos, dtype=torch.int32, device=dev), parents.to(dev)
    dbl = [x.double() for x in (q, k, v, kc, vc)]
    ref = tree_attention_reference(*dbl, p, par)
    out = tree_attention(q, k, v, kc, vc, p, par)
    assert torch.equal(kc.double().nan_to_num(7), dbl[3].nan_to_num(7)) and torch.equal(vc.double().nan_to_num(7), dbl[4].nan_to_num(7))
    assert torch.equal(torch.isnan(out), torch.isnan(ref))
    assert torch.equal(out == float("inf"), ref == float("inf")) and torch.equal(out == -float("inf"), ref == -float("inf"))
    near = (out.double() - ref).abs() <= (4.8e-5 if dtype == F32 else 2.0**-8 * (ref.abs() + 5.5))
    assert bool((near | ~torch.isfinite(ref)).all()) and not bool(torch.isfinite(ref).all())
    other = (torch.arange(t) - t // 2) % 2 == 1  # the branch whose only bad node is a key of the last head and a value of it
    assert torch.equal(out[:, : h // hkv][:, :, other], clean[:, : h // hkv][:, :, other]) or hkv == 1


def test_large_scores(dev):
    """Scores of some hundreds: one key takes all the weight; rows whose keys are at -inf see only the others."""
    for dtype in (BF16, F32):
        q, kn, vn, kc, vc = _inputs(dev, 2, 4, 2, 6, 700, 64, dtype)
        _check(dev, q.sign() * 8, kn.sign() * 4, vn, kc.sign() * 4, vc, [694, 333], trees(2, 6, 5))
        k = kc.clone()
        k[0, 0, 100:500, 0] = -float("inf")
        qp = q.clone()
        qp[..., 0] = qp[..., 0].abs() + 0.1
        _check(dev, qp, kn, vn, k, vc, [600, 20], trees(2, 6, 5))


def test_strided_inputs(dev):
    """q, k_new and v_new where a projection leaves them (token-major, in one row), and views that need a copy."""
    for dtype in (BF16, F32):
        b, h, hkv, t, d = 2, 4, 2, 10, 64
        g = torch.Generator().manual_seed(3)
        qkv = torch.randn(b, t, (h + 2 * hkv), d, generator=g).to(dtype).to(dev)
        q, kn, vn = (x.transpose(1, 2) for x in qkv.split([h, hkv, hkv], 2))
        _, _, _, kc, vc = _inputs(dev, b, h, hkv, t, 500, d, dtype)
        want = _check(dev, q, kn, vn, kc, vc, [480, 7], trees(b, t, 1))
        assert torch.equal(want, _check(dev, q.contiguous(), kn.contiguous(), vn.contiguous(), kc, vc, [480, 7], trees(b, t, 1)))
        odd = torch.randn(b, t, (h + 2 * hkv) * d + 1, generator=g).to(dtype).to(dev)[..., 1:].unflatten(2, (-1, d))
        _check(dev, *(x.transpose(1, 2) for x in odd.split([h, hkv, hkv], 2)), kc, vc, [480, 7], trees(b, t, 1))
        _check(dev, q, kn[:, :1].expand(b, hkv, t, d), vn[:1].expand(b, hkv, t, d), kc, vc, [480, 7], trees(b, t, 1))


def test_one_node_is_decode_attention(dev):
    q, kn, vn, kc, vc = _inputs(dev, 3, 4, 4, 1, 900, 128, F32)
    pos = torch.tensor([0, 450, 899], dtype=torch.int32, device=dev)
    k1, v1 = kc.clone(), vc.clone()
    a = tree_attention(q, kn, vn, kc, vc, pos, torch.full((3, 1), -1, dtype=torch.int32, device=dev))
    e = decode_attention(q[:, :, 0], kn[:, :, 0], vn[:, :, 0], k1, v1, pos)
    assert torch.equal(kc, k1) and torch.equal(vc, v1) and float((a[:, :, 0] - e).abs().max()) <= 4.8e-5


def test_empty_batch(dev):
    q, kn, vn, kc, vc = _inputs(dev, 0, 4, 2, 3, 50, 64, BF16)
    z = torch.zeros(0, dtype=torch.int32, device=dev)
    assert tree_attention(q, kn, vn, kc, vc, z, z.reshape(0, 3)).shape == (0, 4, 3, 64)


def test_long_cache_offsets(dev):
    """A head whose cache passes 2^31 bytes: the last rows are read and written where they are."""
    length, d = (1 << 21) + 300, 256
    kc = torch.zeros(1, 1, length, d, device=dev, dtype=F32)
    vc = torch.zeros(1, 1, length, d, device=dev, dtype=F32)
    q, kn, vn = (torch.randn(1, 1, 3, d, device=dev) for _ in range(3))
    pos = length - 3
    kc[0, 0, pos - 5], vc[0, 0, pos - 5] = 40 * q[0, 0, 1] / q[0, 0, 1].norm(), 2.0
    kc[0, 0, 17], vc[0, 0, 17] = 40 * q[0, 0, 0] / q[0, 0, 0].norm(), -3.0
    out = tree_attention(q, kn * 0, vn, kc, vc, torch.tensor([pos], dtype=torch.int32, device=dev),
                         torch.tensor([[-1, -1, -1]], dtype=torch.int32, device=dev), scale=1.0)
    assert float((out[0, 0, 1] - 2.0).abs().max()) <= 1e-3 and float((out[0, 0, 0] + 3.0).abs().max()) <= 1e-3
    assert torch.equal(vc[0, 0, pos:], vn[0, 0]) and not kc[0, 0, pos:].any() and not vc[0, 0, pos - 4:pos].any()


@pytest.mark.parametrize("length", [200, 1500])
def test_streams_and_graphs(dev, length):
    """Other streams, two captured graphs replayed in turn on their own streams, positions and trees that change."""
    b, t = 3, 12
    q, kn, vn, kc, vc = _inputs(dev, b, 4, 2, t, length, 64, BF16)
    pos = torch.tensor([5, length - t, 77], dtype=torch.int32, device=dev)
    parents = trees(b, t, 1).to(dev)
    call = lambda: tree_attention(q, kn, vn, kc, vc, pos, parents)
    want = call().clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = call()
        side.synchronize()
        assert torch.equal(other, want)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call()
        graphs.append((graph, out, torch.cuda.Stream()))
    for seed in range(3):
        q.copy_(torch.randn(q.shape, generator=torch.Generator().manual_seed(seed)))
        pos.copy_(torch.tensor([seed, length - t - seed, 50 + seed], dtype=torch.int32))
        parents.copy_(trees(b, t, seed, absent=0.2))
        torch.cuda.synchronize()
        for graph, _, stream in graphs:
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        want = call()
        for _, out, _ in graphs:
            assert torch.equal(out, want)
    for graph, _, _ in graphs:
        graph.reset()


def test_accepted_rows_make_the_cache_of_plain_decoding(dev):
    """Tree attention, acceptance and compaction in turn: the cache then holds the accepted path's rows as decoding one
    token after another would have left them."""
    b, h, t, d, length, v = 2, 2, 10, 64, 128, 50
    q, kn, vn, kc, vc = _inputs(dev, b, h, h, t, length, d, F32, seed=4)
    pos = torch.tensor([20, 100], dtype=torch.int32, device=dev)
    parents = trees(b, t, 8)
    logits = torch.randn(b, t, v, generator=torch.Generator().manual_seed(2))
    tokens = logits.argmax(-1).gather(1, parents.clamp(min=0).long())  # every draft is right: the walk takes first children
    k0, v0 = kc.clone(), vc.clone()
    out = tree_attention(q, kn, vn, kc, vc, pos, parents.to(dev))
    path, count, _ = accept_drafts(logits.to(dev), tokens.to(dev), parents.to(dev))
    compact_cache(kc, vc, pos, path, count)
    assert int(count.min()) > 2
    for i in range(b):
        for n, node in enumerate(path[i, : count[i]].tolist()):
            one = lambda x: x[i:i + 1, :, node]
            at = pos[i:i + 1] + n
            e = decode_attention(one(q), one(kn), one(vn), k0[i:i + 1], v0[i:i + 1], at)
            assert float((e - out[i:i + 1, :, node]).abs().max()) <= 4.8e-5
        rows = int(pos[i] + count[i])
        assert torch.equal(kc[i, :, :rows], k0[i, :, :rows]) and torch.equal(vc[i, :, :rows], v0[i, :, :rows])


def _half_step(x):
    """Half the distance of bf16 values at |x|."""
    return torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0**-126))) - 8)


# bf16 kernels by rows: 16, 32 and 64 of a wave, and the ones that share keys through LDS; each head in one workgroup and cut.
BF16_ROWS = [(b, h, hkv, t, length, d)
             for d, rows in ((64, ((2, 2, 8), (3, 1, 7), (4, 1, 13), (4, 1, 40))), (128, ((1, 1, 1), (2, 2, 8), (4, 1, 8), (5, 1, 13), (8, 1, 40))),
                             (256, ((2, 2, 8), (4, 1, 8), (4, 1, 17))))
             for h, hkv, t in rows for b, length in ((2, 200), (2, 3000))]


@pytest.mark.parametrize("b,h,hkv,t,length,d", BF16_ROWS)
def test_weights_of_bf16_values_sum_to_one(dev, b, h, hkv, t, length, d):
    """One value for all keys and nodes: every output is that value, whatever the weights. Those are summed in f32 (n terms, n 2^-24
    <= 2^-12 with n <= 3000) and lie within 2^-16 of themselves in the product: together under 2^-9, half a step of any value.
    First all keys but one have a weight of 0.5 (1 + 0.97 * 2^-8), which one rounding to bf16 takes down by nearly 2^-8."""
    q, kn, vn, kc, vc = _inputs(dev, b, h, hkv, t, length, d, BF16, seed=t)
    value = vc[:, :, :1].clone()
    pos, parents = torch.tensor([length - t, length // 2], dtype=torch.int32, device=dev), trees(b, t, 1).to(dev)
    want = value.repeat_interleave(h // hkv, 1).expand(b, h, t, d)
    one, minus = torch.zeros_like(q), torch.zeros_like(kc)
    one[..., 0], minus[..., 0] = 1, -1
    minus[:, :, 3] = 0
    for qs, ks, news, scale in ((one, minus, minus[:, :, 4:4 + t], -math.log(0.5 * (1 + 0.97 * 2.0**-8))), (q, kc, kn, None)):
        out = tree_attention(qs, news, value.expand_as(vn), ks.clone(), value.expand_as(vc).contiguous(), pos, parents, scale=scale)
        assert torch.equal(out, want)


@pytest.mark.parametrize("b,h,hkv,t,length,d", BF16_ROWS)
def test_bf16_outputs_are_rounded_once(dev, b, h, hkv, t, length, d):
    """The distance from the sums in 64 bits is the output's half step, beside it 2^-16 of the weights' values (up to 5.5) and the f32
    sums' 4.8e-5. With few keys, whose outputs are of order one, that is under a tenth of most half steps."""
    for pos in ([length - t, length // 2], [9, 0]):
        q, kn, vn, kc, vc = _inputs(dev, b, h, hkv, t, length, d, BF16, seed=t + 1)
        p, parents = torch.tensor(pos, dtype=torch.int32, device=dev), trees(b, t, 2)
        ref = tree_attention_reference(*(x.double() for x in (q, kn, vn, kc, vc)), p, parents.to(dev))
        if t == 1 and h == hkv:
            one = lambda x: x[:, :, 0]
            e = decode_attention(one(q), one(kn), one(vn), kc.clone(), vc.clone(), p)
            assert bool(((e.double() - one(ref)).abs() <= _half_step(one(ref)) * 1.001 + 5.5 * 2.0**-16 + 4.8e-5).all())
        out = tree_attention(q, kn, vn, kc, vc, p, parents.to(dev))
        assert bool(((out.double() - ref).abs() <= _half_step(ref) * 1.001 + 5.5 * 2.0**-16 + 4.8e-5).all())


@pytest.mark.parametrize("b,h,hkv,t,length,d", BF16_ROWS)
def test_infinite_values_of_the_cache(dev, b, h, hkv, t, length, d):
    """Infinities and NaN in cached values, which every row sees: infinite in that element, NaN where two signs or a NaN meet."""
    q, kn, vn, kc, vc = _inputs(dev, b, h, hkv, t, length, d, BF16, seed=t + 2)
    inf = float("inf")
    for row, element, bad in ((5, 3, inf), (40, 7, -inf), (60, 9, float("nan")), (33, 11, inf), (2, 11, -inf), (7, 20, inf), (61, 20, inf)):
        vc[:, :, row, element] = bad
    p, parents = torch.tensor([length - t, length // 2], dtype=torch.int32, device=dev), trees(b, t, 3).to(dev)
    ref = tree_attention_reference(*(x.double() for x in (q, kn, vn, kc, vc)), p, parents)
    out = tree_attention(q, kn, vn, kc, vc, p, parents)
    assert bool((ref[..., 3] == inf).all()) and bool((ref[..., 7] == -inf).all()) and bool(torch.isnan(ref[..., [9, 11]]).all())
    assert torch.equal(torch.isnan(out), torch.isnan(ref)) and torch.equal(out.isinf(), ref.isinf())
    assert torch.equal(out == inf, ref == inf)
    near = (out.double() - ref).abs() <= _half_step(ref) * 1.001 + 5.5 * 2.0**-16 + 4.8e-5
    assert bool((near | ~torch.isfinite(ref)).all())


@pytest.mark.parametrize("b,h,hkv,t,length,d,dtype", [
    (130, 512, 1, 1, 6300, 64, F32),   # 512 rows a sequence: 1040 row groups
    (96, 32, 32, 2, 600, 64, F32)])    # 3072 heads
def test_many_whole_heads_of_unequal_lengths(dev, b, h, hkv, t, length, d, dtype):
    """More heads than fill the chip, each in one workgroup: short, empty, misplaced and full sequences side by side."""
    x = _inputs(dev, b, h, hkv, t, length, d, dtype, seed=b)
    pos = torch.randint(0, length - t + 1, (b,), generator=torch.Generator().manual_seed(b)) // 8
    pos[1], pos[b // 2 - 1], pos[b - 1], pos[65], pos[7] = 0, -1, length - t, length, length - t
    _check(dev, *x, pos.tolist(), trees(b, t, 1, absent=0.1))


def test_caches_beside_each_other(dev):
    """Two halves of one allocation are two caches; one for both, or nodes that are rows of one, are refused and nothing is written."""
    b, h, t, length, d = 2, 2, 5, 200, 64
    for dtype in (BF16, F32):
        q, kn, vn, kc, vc = _inputs(dev, b, h, h, t, length, d, dtype)
        both = torch.stack([kc, vc])
        pos, parents = torch.tensor([20, 100], dtype=torch.int32, device=dev), trees(b, t, 1).to(dev)
        want = tree_attention(q, kn, vn, kc, vc, pos, parents)
        assert torch.equal(tree_attention(q, kn, vn, both[0], both[1], pos, parents), want)
        assert torch.equal(both, torch.stack([kc, vc]))
        rows = both[0][:, :, 20:20 + t]
        for args in ((q, kn, vn, both[0], both[0]), (q, rows, vn, both[0], both[1]), (q, kn, rows, both[0], both[1]),
                     (rows, kn, vn, both[0], both[1]), (q, kn, both[1][:, :, :t], both[0], both[1])):
            with pytest.raises(RuntimeError, match="overlap"):
                tree_attention(*args, pos, parents)
        assert torch.equal(both, torch.stack([kc, vc]))


@pytest.mark.parametrize("h,hkv,t,length,d,dtype", [
    (2, 2, 7, 200, 64, BF16), (2, 2, 7, 3000, 128, BF16), (4, 2, 20, 300, 128, BF16), (4, 2, 40, 3000, 64, BF16), (4, 2, 13, 200, 256, BF16),
    (4, 2, 9, 200, 64, F32), (4, 2, 9, 3000, 128, F32), (4, 2, 33, 900, 64, F32)])
def test_rows_whose_scores_are_all_minus_infinity(dev, h, hkv, t, length, d, dtype):
    """The quotient of two zeros, as a softmax of such scores and decode_attention have it: NaN in the rows of that key head, and where
    one key is left its value. Absent nodes stay zero."""
    q, kn, vn, kc, vc = _inputs(dev, 2, h, hkv, t, length, d, dtype, seed=t)
    q[..., 0] = q[..., 0].abs() + 0.1
    kc[:, 0, :, 0], kn[:, 0, :, 0] = -float("inf"), -float("inf")
    kc[1, 0, 33, 0] = 1
    pos, parents = torch.tensor([length - t, length // 2], dtype=torch.int32, device=dev), trees(2, t, 1)
    parents[:, 2] = -2
    there = ancestors(parents).diagonal(dim1=1, dim2=2).to(dev)[:, None, :, None]
    ref = tree_attention_reference(*(x.double() for x in (q, kn, vn, kc, vc)), pos, parents.to(dev))
    out = tree_attention(q, kn, vn, kc.clone(), vc.clone(), pos, parents.to(dev))
    g = h // hkv
    assert torch.equal(torch.isnan(out), torch.isnan(ref)) and torch.equal(torch.isnan(out[0, :g]), there[0].expand_as(out[0, :g]))
    assert torch.equal(out[1, :g], torch.where(there[1], vc[1, 0, 33], torch.zeros_like(vc[1, 0, 33])).expand_as(out[1, :g]))
    assert not bool(torch.isnan(out[:, g:]).any()) and not bool(torch.where(there, 0, out).any())
    e = decode_attention(q[:, :, 0], *(x[:, :, 0].repeat_interleave(g, 1) for x in (kn, vn)),
                         *(x.repeat_interleave(g, 1) for x in (kc, vc)), pos)
    assert torch.equal(torch.isnan(e), torch.isnan(out[:, :, 0]))


# Two and four row tiles to a wave: heads whole (up to 16 steps), cut among few, and cut among many, whose pieces one line of the join
# adds up; and the narrowest rows over caches of many heads.
TILES = [(2, h, hkv, t, length, d, dtype)
         for d, dtype in ((64, BF16), (128, BF16), (256, BF16), (64, F32), (128, F32), (256, F32))
         for h, hkv, t in ((1, 1, 17), (6, 2, 8), (4, 1, 8)) for length in (230, 3000)]
TILES += [(2, h, hkv, t, length, 64, dtype) for dtype in (BF16, F32) for h, hkv, t in ((3, 1, 11), (8, 2, 13), (1, 1, 64))
          for length in (240, 1500)]
TILES += [(8, 32, 32, 4, 4200, 128, BF16), (8, 32, 32, 9, 4300, 64, BF16), (8, 96, 32, 8, 4200, 128, BF16), (8, 64, 32, 9, 4200, 256, BF16),
          (8, 128, 32, 13, 4200, 64, BF16), (8, 64, 32, 10, 2100, 128, F32),
          (16, 16, 4, 24, 1500, 128, BF16)]  # 96 rows over shared keys


@pytest.mark.parametrize("b,h,hkv,t,length,d,dtype", TILES)
def test_row_tiles(dev, b, h, hkv, t, length, d, dtype):
    x = _inputs(dev, b, h, hkv, t, length, d, dtype, seed=h * t + d)
    pos = [length - t - i * (length // 9) for i in range(b)]
    pos[1] = 31
    _check(dev, *x, pos, trees(b, t, 1))
    if b == 2:
        _check(dev, *x, pos[::-1], trees(b, t, 2, absent=0.3), scale=-0.3 / d**0.5)


@pytest.mark.parametrize("h,hkv,t,length,d,dtype", [
    (4, 2, 8, 230, 128, BF16), (6, 2, 8, 3000, 128, BF16), (8, 2, 8, 3000, 128, BF16), (4, 2, 9, 200, 256, BF16), (8, 2, 8, 3000, 256, BF16),
    (8, 2, 12, 1500, 64, BF16), (6, 2, 8, 3000, 64, F32), (6, 2, 8, 200, 256, F32)])
def test_branches_stay_apart_in_row_tiles(dev, h, hkv, t, length, d, dtype):
    test_what_a_branch_does_not_see_does_not_touch_it(dev, 2, h, hkv, t, length, d, dtype, [length - t, 40])
