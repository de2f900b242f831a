"""GPU tests of the drafted step's walk and of the cache's compaction (csrc/drafts.hip). Whole numbers and moved
rows: everything is compared for equality with the walk and the moves in Python."""

import pytest
import torch

from ferrite.kernels.drafts import accept_drafts, accept_drafts_reference, compact_cache, compact_cache_reference

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


def trees(b, t, seed, absent=0.0):
    """Parents int32 [B, T]: node 0 a root, every other node under one of the four before it; some absent."""
    g = torch.Generator().manual_seed(seed)
    idx = torch.arange(t)
    back = 1 + (torch.rand(b, t, generator=g) * idx.clamp(max=4)).long()
    parents = torch.where(idx > 0, (idx - back).clamp(min=0), -1)
    gone = torch.rand(b, t, generator=g) < absent
    odd = torch.tensor([-2, 64, 63, -(2**31), 2**31 - 1])[torch.randint(0, 5, (b, t), generator=g)]
    odd = torch.where((odd >= -1) & (odd < idx), -2, odd)
    return torch.where(gone, odd, parents).int()


def _drafts(dev, b, t, v, dtype, seed, absent=0.1, ties=False):
    g = torch.Generator().manual_seed(seed)
    logits = torch.randn(b, t, v, generator=g).to(dtype)
    if ties:
        logits = (logits * 2).round()
    parents = trees(b, t, seed, absent)
    wanted = logits.float().argmax(-1)  # on the CPU the lowest index of equal values
    hit = torch.rand(b, t, generator=g) < 0.8
    tokens = torch.where(hit, wanted.gather(1, parents.clamp(0, t - 1).long()), torch.randint(0, v, (b, t), generator=g))
    return logits, tokens, parents


def _check(dev, logits, tokens, parents):
    want = accept_drafts_reference(logits.float(), tokens, parents)
    got = accept_drafts(logits.to(dev), tokens.to(dev), parents.to(dev))
    for x, y in zip(got, want):
        assert x.dtype == y.dtype and x.shape == y.shape and torch.equal(x.cpu(), y)
    return got


@pytest.mark.parametrize("b,t,v", [
    (1, 1, 1), (3, 1, 257), (2, 8, 256), (5, 64, 7), (4, 17, 2048), (4, 17, 2049), (2, 64, 4097), (3, 5, 50257), (1, 2, 131071),
    (70, 60, 3001), (1, 64, 300),
])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_accept(dev, b, t, v, dtype):
    for ties in (False, True):
        logits, tokens, parents = _drafts(dev, b, t, v, dtype, seed=b * t + v, ties=ties)
        _check(dev, logits, tokens, parents)
        _check(dev, logits, tokens.int(), trees(b, t, 1))


@pytest.mark.parametrize("v", [300, 5000])
def test_accept_odd_values(dev, v):
    """Infinities, NaN of either sign, zeros of either sign, a whole row alike; the best value in each place of a vector."""
    b, t = 4, 16
    logits, _, _ = _drafts(dev, b, t, v, F32, 5)
    logits[0, 0] = float("-inf")
    logits[0, 1, 7], logits[0, 1, 9] = float("inf"), float("inf")
    logits[0, 2, 11], logits[0, 2, 3] = float("nan"), float("inf")
    logits[0, 3, 12], logits[0, 3, 10] = -float("nan"), float("nan")
    logits[0, 4] = -1
    logits[0, 4, 20], logits[0, 4, 21] = -0.0, 0.0
    logits[0, 5] = 3.0
    for j in range(6, t):
        logits[0, j, v - 1 - (j - 6)] = 50 + j
        logits[1, j, j] = 50 + j
    parents = torch.arange(-1, t - 1).expand(b, t).int().contiguous()  # chains
    wanted = logits.argmax(-1)
    assert wanted[0, :6].tolist() == [0, 7, 11, 10, 20, 0]
    tokens = torch.cat([torch.zeros(b, 1, dtype=torch.long), wanted[:, :-1]], 1)
    path, count, following = _check(dev, logits, tokens, parents)
    assert count.tolist() == [t] * b and torch.equal(following.cpu(), wanted[:, -1])


def test_accept_reads_nothing_of_absent_nodes_and_views(dev):
    """A strided view of logits, tokens and parents; rows of absent nodes hold NaN, which would win."""
    logits, tokens, parents = _drafts(dev, 3, 12, 3000, F32, 9, absent=0.4)
    _check(dev, logits, tokens, parents)
    wide = torch.full((3, 12, 3003), float("nan"))
    wide[..., 3:] = logits
    wide[(parents < -1) | (parents >= torch.arange(12))] = float("nan")
    got = accept_drafts(wide.to(dev)[..., 3:], tokens.t().contiguous().to(dev).t(), parents.t().contiguous().to(dev).t())
    for x, y in zip(got, accept_drafts_reference(logits, tokens, parents)):
        assert torch.equal(x.cpu(), y)
    none = accept_drafts(torch.zeros(0, 4, 9, device=dev), torch.zeros(0, 4, dtype=torch.long, device=dev),
                         torch.zeros(0, 4, dtype=torch.int32, device=dev))
    assert [tuple(t.shape) for t in none] == [(0, 4), (0,), (0,)]


def _paths(b, t, seed):
    g = torch.Generator().manual_seed(seed)
    path, count = torch.full((b, t), -1), torch.randint(0, t + 1, (b,), generator=g)
    for i in range(b):
        path[i, : count[i]] = torch.randperm(t, generator=g)[: count[i]].sort().values
    return path.int(), count.int()


@pytest.mark.parametrize("shape,t,dtype", [
    ((1, 1, 8, 64), 1, BF16), ((2, 3, 40, 64), 8, BF16), ((3, 2, 4, 200, 128), 64, BF16), ((2, 5, 1, 77, 256), 23, F32),
    ((2, 3, 30, 5), 9, BF16), ((2, 2, 3, 30, 3), 17, F32), ((4, 3, 2, 50, 12), 12, F32), ((1, 9, 4, 1, 64), 1, F32),
    ((12, 8, 12, 96, 64), 24, BF16),
])
def test_compact(dev, shape, t, dtype):
    b, length = shape[-4], shape[-2]
    for seed in range(3):
        g = torch.Generator().manual_seed(seed)
        k, v = (torch.randn(shape, generator=g).to(dtype) for _ in range(2))
        path, count = _paths(b, t, seed)
        pos = torch.randint(0, max(1, length - t + 1), (b,), generator=g).int()
        kd, vd = k.to(dev), v.to(dev)
        compact_cache(kd, vd, pos.to(dev), path.to(dev), count.to(dev))
        compact_cache_reference(k, v, pos, path, count)
        assert torch.equal(kd.cpu(), k) and torch.equal(vd.cpu(), v)


def test_compact_bad_paths_and_edges(dev):
    """A path ends where it stops going up or leaves the cache; positions and counts outside move nothing."""
    lines = [[0, 2, 1, 3], [0, 3, 3, 3], [-1, 1, 2, 3], [1, 2, 4, 5], [0, 2, 3, 2**31 - 1], [1, 2, 3, 4], [1, 2, 3, 4],
             [1, 2, 3, 4], [1, 2, 3, 4], [3, 2**31 - 1, 5, 6]]
    pos = [3, 0, 2, 11, 12, -1, 16, 2**31 - 1, 2, 10]
    count = [4, 4, 4, 4, 4, 4, 4, 4, -3, 100]
    path, pos, count = (torch.tensor(x, dtype=torch.int32) for x in (lines, pos, count))
    for d in (8, 5):
        k = torch.randn(2, len(lines), 2, 16, d)
        v = torch.randn_like(k)
        kd, vd = k.to(dev), v.to(dev)
        compact_cache(kd, vd, pos.to(dev), path.to(dev), count.to(dev))
        compact_cache_reference(k, v, pos, path, count)
        assert torch.equal(kd.cpu(), k) and torch.equal(vd.cpu(), v)
    compact_cache(torch.zeros(0, 2, 16, 8, device=dev), torch.zeros(0, 2, 16, 8, device=dev),
                  *(torch.zeros(s, dtype=torch.int32, device=dev) for s in ((0,), (0, 4), (0,))))


def test_compact_unaligned_cache(dev):
    """Caches that start off 16 bytes move by elements."""
    base = torch.randn(2, 1 + 2 * 3 * 20 * 8, device=dev).to(BF16)
    kd, vd = (r[1:].view(2, 3, 20, 8) for r in base)
    k, v = kd.cpu(), vd.cpu()
    path, count = _paths(2, 10, 3)
    pos = torch.tensor([4, 10], dtype=torch.int32)
    compact_cache(kd, vd, pos.to(dev), path.to(dev), count.to(dev))
    compact_cache_reference(k, v, pos, path, count)
    assert torch.equal(kd.cpu(), k) and torch.equal(vd.cpu(), v)


@pytest.mark.parametrize("v", [256, 20000])
def test_streams_and_graph(dev, v):
    """The walk and the moves captured together; replays follow what the buffers hold."""
    b, t = 3, 16
    logits, tokens, parents = (x.to(dev) for x in _drafts(dev, b, t, v, F32, 2))
    k0 = torch.randn(2, b, 2, 64, 64, device=dev).to(BF16)
    v0 = torch.randn_like(k0)
    k, vv = k0.clone(), v0.clone()
    pos = torch.tensor([3, 40, 17], dtype=torch.int32, device=dev)

    def step():
        path, count, following = accept_drafts(logits, tokens, parents)
        compact_cache(k, vv, pos, path, count)
        return path, count, following

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in range(3):
        fresh = _drafts(dev, b, t, v, F32, 50 + seed)
        for dst, src in zip((logits, tokens, parents), fresh):
            dst.copy_(src)
        k.copy_(k0), vv.copy_(v0)
        graph.replay()
        torch.cuda.synchronize()
        want = accept_drafts_reference(*fresh)
        assert all(torch.equal(x.cpu(), y) for x, y in zip(out, want))
        kr, vr = k0.cpu(), v0.cpu()
        compact_cache_reference(kr, vr, pos.cpu(), *want[:2])
        assert torch.equal(k.cpu(), kr) and torch.equal(vv.cpu(), vr)
    graph.reset()


@pytest.mark.parametrize("b,t,v", [(1030, 64, 7), (1030, 64, 1100), (70001, 1, 5)])
def test_accept_more_nodes_than_one_launch_takes(dev, b, t, v):
    """Over 65535 nodes in all, walked by one workgroup a sequence and cut into pieces."""
    logits, tokens, parents = _drafts(dev, b, t, v, BF16 if v > 1000 else F32, seed=b)
    _check(dev, logits, tokens, parents)


def test_caches_beside_each_other(dev):
    """Caches that end where the other begins are two; one for both, or shifted by a row, is refused and left as it is."""
    both = torch.randn(2, 2, 3, 16, 8, device=dev)
    want = [c.cpu() for c in both]
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)
    args = ints([3, 9]), ints([[0, 2, 5], [1, 2, 6]]), ints([3, 2])
    compact_cache_reference(*want, *(a.cpu() for a in args))
    compact_cache(both[0], both[1], *args)
    assert all(torch.equal(c.cpu(), w) for c, w in zip(both, want))
    flat = both.flatten()
    for k, v in ((both[0], both[0]), (both[1], flat[8 * 16 * 6 - 8:-8].view(2, 3, 16, 8))):
        with pytest.raises(RuntimeError, match="overlap"):
            compact_cache(k, v, *args)
    assert all(torch.equal(c.cpu(), w) for c, w in zip(both, want))
