"""GPU tests of gradient clipping (csrc/clip.hip) against 64 bits.

The squares are added in 64 bits, so the norm is off by its rounding to f32 alone (u = 2^-24, 1.01 allowed). An element is multiplied
in f32 by a factor that is rounded to f32: two u, and half a step of its type."""

import math

import pytest
import torch

from ferrite.kernels.clip import clip_grad_norm_, clip_grad_norm_reference

pytestmark = pytest.mark.gpu

U = 2.0**-24
HALF = {torch.bfloat16: 2.0**-8, torch.float32: 2.0**-24}
BF16, F32 = torch.bfloat16, torch.float32
SIZES = [0, 1, 7, 8, 255, 8191, 8192, 8193, 16384, 100003]


def _grads(dev, sizes, dtypes, scale=1.0, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [(scale * torch.randn(n, generator=g)).to(dev, dtypes[i % len(dtypes)]) for i, n in enumerate(sizes)]


def _check(grads, most):
    before = [g.clone() for g in grads]
    norm = clip_grad_norm_(grads, most)
    exact = math.sqrt(math.fsum(float(g.double().square().sum()) for g in before))
    assert norm.shape == () and norm.dtype == F32 and abs(float(norm) - exact) <= 1.01 * U * exact
    factor = most / (exact + 1e-6)
    for g, b in zip(grads, before):
        if factor >= 1:
            assert torch.equal(g, b)
        else:
            ref = b.double() * factor
            assert bool(((g.double() - ref).abs() <= (2 * U + HALF[g.dtype]) * 1.01 * ref.abs() + 2.0**-133).all())


@pytest.mark.parametrize("dtypes", [(F32,), (BF16,), (F32, BF16), (BF16, BF16, F32)])
@pytest.mark.parametrize("most", [0.0, 1e-3, 1.0, 1e9, math.inf])
def test_norm_and_scaling(dev, dtypes, most):
    _check(_grads(dev, SIZES, dtypes), most)
    _check(_grads(dev, [1], dtypes), most)
    _check(_grads(dev, [3000000], dtypes), most)


@pytest.mark.parametrize("n", [127, 128, 129, 300, 1000])
def test_many_tensors(dev, n):
    g = torch.Generator().manual_seed(n)
    sizes = torch.randint(0, 20000, (n,), generator=g).tolist()
    _check(_grads(dev, sizes, (BF16, F32)), 1.0)
    _check(_grads(dev, [0] * n, (F32,)), 1.0)
    _check(_grads(dev, [0] * (n - 1) + [9], (F32,)), 0.5)
    _check(_grads(dev, [9] + [0] * (n - 1), (F32,)), 0.5)


@pytest.mark.parametrize("most", [1.0, math.inf])
def test_gradients_past_the_caches(dev, most):
    """Above 128 MB in all the reads leave the caches out; many tensors, of sizes that end inside a tile, and one that is huge."""
    flat = torch.randn(48_000_000, generator=torch.Generator(dev).manual_seed(3), device=dev)
    _check([flat[1:40_000_000], flat[40_000_001:], *_grads(dev, SIZES * 20, (BF16, F32))], most)
    half = flat.to(BF16)
    _check([half.clone(), half[3:47_999_999]], most)


@pytest.mark.parametrize("scale", [1e-30, 1e25, 1e30])
def test_squares_past_the_range_of_floats(dev, scale):
    _check(_grads(dev, [5000, 100], (F32, BF16), scale), scale)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_a_norm_that_is_not_finite_leaves_the_gradients(dev, bad):
    grads = _grads(dev, SIZES, (F32, BF16))
    grads[6][17] = bad
    before = [g.clone() for g in grads]
    norm = clip_grad_norm_(grads, 0.1)
    assert not math.isfinite(float(norm)) and all(torch.equal(g.nan_to_num(3.0), b.nan_to_num(3.0)) for g, b in zip(grads, before))
    huge = [torch.full((64,), 3e38, device=dev)]  # finite elements, a norm past the floats
    assert float(clip_grad_norm_(huge, 1.0)) == math.inf and bool((huge[0] == 3e38).all())


def test_layouts(dev):
    flat = torch.randn(50000, device=dev)
    grads = [flat[1:10001], flat[10002:20002].view(100, 100).t(), flat[20003:50000].view(3, 9999), torch.randn((), device=dev),
             torch.randn(4, 5, 6, device=dev).to(memory_format=torch.contiguous_format).permute(2, 0, 1)]
    rest = flat[[0, 10001, 20002]].clone()
    grads.append(torch.randn(0, 10, device=dev)[:, ::2])  # nothing to scale, whatever its strides
    _check(grads, 0.5)
    assert torch.equal(flat[[0, 10001, 20002]], rest)  # what lies between them
    with pytest.raises(ValueError, match="dense"):
        clip_grad_norm_([torch.randn(10, 10, device=dev)[:, ::2]], 1.0)
    with pytest.raises(ValueError, match="dense"):
        clip_grad_norm_([torch.randn(1, device=dev).expand(10)], 1.0)
    with pytest.raises(RuntimeError, match="share memory"):
        clip_grad_norm_([flat[:100], flat[300:], flat[99:200]], 1.0)
    with pytest.raises(RuntimeError, match="share memory"):
        clip_grad_norm_([flat, flat], 1.0)


def test_against_the_reference_and_in_a_graph(dev):
    grads = _grads(dev, SIZES, (F32, BF16), seed=4)
    fresh = [g.clone() for g in grads]
    want = [g.clone() for g in grads]
    assert float(clip_grad_norm_reference(want, 2.0)) == float(clip_grad_norm_(grads, 2.0))
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = [g.clone() for g in fresh]
        clip_grad_norm_(other, 2.0)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(grads, other))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = clip_grad_norm_(other, 2.0)
    for k in range(3):
        for o, f in zip(other, fresh):
            o.copy_(f * (k + 1))
        graph.replay()
        eager = [f * (k + 1) for f in fresh]
        ref = clip_grad_norm_(eager, 2.0)
        torch.cuda.synchronize()
        assert torch.equal(norm, ref) and all(torch.equal(a, b) for a, b in zip(other, eager))


def test_a_saved_tensor_that_was_scaled_is_noticed(dev):
    x = torch.randn(100, device=dev, requires_grad=True)
    g = torch.randn(100, device=dev)
    y = x * g
    clip_grad_norm_([g], 0.1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_tensors_that_require_a_gradient(dev):
    g = torch.full((10,), 2.0, device=dev, requires_grad=True)
    with pytest.raises(RuntimeError, match="no_grad"):
        clip_grad_norm_([g], 1.0)
    assert bool((g == 2).all())
    with torch.no_grad():
        _check([g], 1.0)


@pytest.mark.parametrize("scale,most", [(1e30, 1e-9), (1e30, 1e-12), (1e34, 1e-14), (1e36, 1e-30), (1e-20, 1e-25)])
def test_factors_past_the_range_of_floats(dev, scale, most):
    """Elements and products that are ordinary floats, and a factor between them that f32 has few bits for, or none."""
    _check(_grads(dev, [5000, 100, 8192, 30000], (F32, BF16), scale, seed=6), most)
