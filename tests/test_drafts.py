"""CPU tests of the drafted step's and the rotated heads' operators: what they refuse, before any launch."""

import pytest
import torch

from ferrite import _hip
from ferrite.kernels.drafts import accept_drafts, accept_drafts_reference, compact_cache, compact_cache_reference
from ferrite.kernels.qk_norm_rope import qk_norm_rope, qk_norm_rope_reference, rope_tables
from ferrite.kernels.tree_attention import ancestors, tree_attention, tree_attention_reference

F32, BF16 = torch.float32, torch.bfloat16


def _heads(**change):
    a = dict(qkv=torch.zeros(2, 3, 8 * 64), q_weight=torch.ones(64), k_weight=torch.ones(64), cos=torch.ones(8, 32),
             sin=torch.zeros(8, 32), n_head=4, n_kv_head=2, positions=None)
    a.update(change)
    return a


@pytest.mark.parametrize("change,words", [
    (dict(n_head=3), "n_head"),
    (dict(n_head=0), "at least one"),
    (dict(n_kv_head=0), "at least one"),
    (dict(qkv=torch.zeros(3, 512)), "qkv as"),
    (dict(qkv=torch.zeros(2, 3, 0)), "qkv as"),
    (dict(qkv=torch.zeros(2, 3, 8 * 63)), "even"),
    (dict(qkv=torch.zeros(2, 3, 8 * 514)), "at most 512"),
    (dict(q_weight=torch.ones(32)), "weights"),
    (dict(k_weight=torch.ones(64, dtype=BF16)), "share a dtype"),
    (dict(sin=torch.zeros(8, 16)), "pairs"),
    (dict(cos=torch.ones(8, 33), sin=torch.ones(8, 33)), "pairs"),
    (dict(cos=torch.ones(8, 0), sin=torch.ones(8, 0)), "pairs"),
    (dict(cos=torch.ones(0, 8), sin=torch.ones(0, 8)), "pairs"),
    (dict(cos=torch.ones(8, 32, dtype=BF16)), "float32"),
    (dict(cos=torch.ones(8, 32, requires_grad=True)), "no gradient"),
    (dict(cos=torch.ones(2, 32), sin=torch.ones(2, 32)), "longer"),
    (dict(positions=torch.zeros(2, 4, dtype=torch.int32)), "positions"),
    (dict(positions=torch.zeros(3)), "int32"),
    (dict(positions=torch.zeros(3, dtype=torch.int64)), "int32"),
    (dict(qkv=torch.zeros(2, 3, 512, dtype=torch.float64)), "float32 or bfloat16"),
    (dict(q_weight=torch.ones(64).half(), k_weight=torch.ones(64).half()), "float32 or bfloat16"),
])
def test_heads_refusals(change, words):
    with pytest.raises(ValueError, match=words):
        qk_norm_rope(**_heads(**change))


def test_heads_refuse_the_cpu():
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        qk_norm_rope(**_heads())


def test_heads_abi_refusals():
    lib = _hip.lib()
    ok = dict(b=2, s=3, h=4, hkv=2, d=64, rot=64, table=8, dtype=_hip.BF16, w=_hip.F32)

    def call(**change):
        a = {**ok, **change}
        args = (a["b"], a["s"], a["h"], a["hkv"], a["d"], a["rot"], a["table"], a["dtype"], a["w"], 0, 1e-6)
        return (lib.ferrite_internal_heads_rope(None, 1, 1, *[None] * 8, *args, None),
                lib.ferrite_internal_heads_rope_bwd(None, 1, 1, *[None] * 11, *args, None, 0, None))

    for change, words in ((dict(), "null"), (dict(dtype=5), "dtype"), (dict(w=-1), "dtype"), (dict(h=0), "heads"),
                          (dict(hkv=20000), "heads"), (dict(b=-1), "tokens"), (dict(b=1 << 20, s=1 << 20), "tokens"),
                          (dict(d=63), "even"), (dict(d=514), "512"), (dict(rot=66), "even and within"), (dict(rot=3), "even"),
                          (dict(table=0), "tables")):
        assert call(**change) == (1, 1), change
        assert words in _hip.last_error()
    # nothing to do: no launch; the sums of no rows are still written by the backward, which needs its outputs
    assert call(b=0) == (0, 1)
    assert lib.ferrite_internal_heads_rope_bwd_workspace(1, 1, 1, 1, 3) == -1
    assert lib.ferrite_internal_heads_rope_bwd_workspace(8, 1024, 12, 12, 64) > 0
    # one token more than a launch's blocks hold
    a = 1 << 12
    assert lib.ferrite_internal_heads_rope(a, 2, 2, *[a] * 8, 1 << 14, 1 << 15, 1, 1, 2, 2, 1 << 15, _hip.BF16, _hip.F32, 0,
                                           1e-6, None) == 1
    assert "too many tokens" in _hip.last_error()


def test_rope_tables():
    cos, sin = rope_tables(5, 6, base=100.0)
    assert cos.shape == sin.shape == (5, 3) and cos.dtype == F32
    p = torch.arange(5, dtype=torch.float64)[:, None]
    rate = torch.tensor([1.0, 100.0 ** (-1 / 3), 100.0 ** (-2 / 3)], dtype=torch.float64)
    assert torch.allclose(cos.double(), (p * rate).cos(), atol=2.0**-24, rtol=0)
    assert torch.allclose(sin.double(), (p * rate).sin(), atol=2.0**-24, rtol=0)
    for n, d in ((0, 4), (4, 3), (4, 0)):
        with pytest.raises(ValueError):
            rope_tables(n, d)


def test_heads_reference_keeps_lengths_and_turns_by_distance():
    """A rotation keeps a head's length, and the product of two heads depends on the distance of their positions."""
    g = torch.Generator().manual_seed(0)
    x = torch.randn(1, 1, 3 * 8, generator=g, dtype=torch.float64)
    one = torch.ones(8, dtype=torch.float64)
    cos, sin = (t.double() for t in rope_tables(40, 8))
    for inter in (False, True):
        at = lambda p: qk_norm_rope_reference(x, one, one, cos, sin, n_head=1, positions=torch.tensor([p]),
                                              interleaved=inter, eps=0.0)
        assert abs(float(at(17)[0].square().sum()) - 8) <= 1e-6  # the tables are rounded to f32
        a, b = (float((at(p + 5)[0] * at(p)[1]).sum()) for p in (0, 30))
        assert abs(a - b) <= 1e-5


def _accept(**change):
    a = dict(logits=torch.zeros(2, 3, 8), tokens=torch.zeros(2, 3, dtype=torch.long),
             parents=torch.zeros(2, 3, dtype=torch.int32))
    a.update(change)
    return a


@pytest.mark.parametrize("change,words", [
    (dict(logits=torch.zeros(6, 8)), "logits as"),
    (dict(logits=torch.zeros(2, 65, 8)), "1 to 64"),
    (dict(logits=torch.zeros(2, 0, 8)), "1 to 64"),
    (dict(logits=torch.zeros(2, 3, 0)), "logits as"),
    (dict(tokens=torch.zeros(2, 4, dtype=torch.long)), "tokens as"),
    (dict(tokens=torch.zeros(2, 3)), "tokens must be int64 or int32"),
    (dict(parents=torch.zeros(3, 2, dtype=torch.int32)), "parents as"),
    (dict(parents=torch.zeros(2, 3, dtype=torch.long)), "parents must be int32"),
    (dict(logits=torch.zeros(2, 3, 8).half()), "float32 or bfloat16"),
])
def test_accept_refusals(change, words):
    with pytest.raises(ValueError, match=words):
        accept_drafts(**_accept(**change))
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        accept_drafts(**_accept())


def _compact(**change):
    a = dict(k_cache=torch.zeros(2, 4, 16, 8), v_cache=torch.zeros(2, 4, 16, 8), pos=torch.zeros(2, dtype=torch.int32),
             path=torch.zeros(2, 3, dtype=torch.int32), count=torch.zeros(2, dtype=torch.int32))
    a.update(change)
    return a


@pytest.mark.parametrize("change,words", [
    (dict(k_cache=torch.zeros(4, 16, 8)), "caches"),
    (dict(v_cache=torch.zeros(2, 4, 16, 9)), "one shape"),
    (dict(v_cache=torch.zeros(2, 4, 16, 8, dtype=BF16)), "share a dtype"),
    (dict(v_cache=torch.zeros(2, 4, 8, 16).transpose(2, 3)), "contiguous"),
    (dict(pos=torch.zeros(3, dtype=torch.int32)), "pos as"),
    (dict(pos=torch.zeros(2)), "pos must be int32"),
    (dict(path=torch.zeros(2, dtype=torch.int32)), "path as"),
    (dict(path=torch.zeros(2, 65, dtype=torch.int32)), "1 to 64"),
    (dict(path=torch.zeros(2, 3, dtype=torch.long)), "path must be int32"),
    (dict(count=torch.zeros(1, dtype=torch.int32)), "count as"),
    (dict(k_cache=torch.zeros(2, 4, 16, 8).half(), v_cache=torch.zeros(2, 4, 16, 8).half()), "float32 or bfloat16"),
])
def test_compact_refusals(change, words):
    with pytest.raises(ValueError, match=words):
        compact_cache(**_compact(**change))
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        compact_cache(**_compact())


def test_drafts_abi_refusals():
    lib = _hip.lib()
    a = 1 << 12
    accept = lambda b, t, v, dtype=_hip.F32, ws=None, n=0, p=a: lib.ferrite_internal_accept_drafts(
        p, a, a, a, a, a, b, t, v, dtype, ws, n, None)
    assert accept(0, 4, 8) == 0
    for args, words in (((2, 0, 8), "nodes"), ((2, 65, 8), "nodes"), ((2, 4, 0), "vocabulary"), ((2, 4, 1 << 31), "vocabulary"),
                        ((-1, 4, 8), "nodes"), ((65535, 2, 8), "65535"), ((2, 4, 8, 7), "dtype")):
        assert accept(*args) == 1 and words in _hip.last_error(), args
    assert accept(2, 4, 8, p=None) == 1 and "null" in _hip.last_error()
    need = lib.ferrite_internal_accept_drafts_workspace(2, 4, 50000)
    assert need > 0 and accept(2, 4, 50000, ws=a, n=need - 1) == 1 and "workspace" in _hip.last_error()
    assert accept(2, 4, 50000) == 1 and "workspace" in _hip.last_error()
    assert lib.ferrite_internal_accept_drafts_workspace(2, 65, 8) == -1
    compact = lambda layers, b, h, n, d, t, dtype=_hip.BF16, p=a: lib.ferrite_internal_compact_cache(
        p, a, a, a, a, layers, b, h, n, d, t, dtype, None)
    for zero in ((0, 2, 2), (2, 0, 2), (2, 2, 0)):
        assert compact(*zero, 16, 8, 4) == 0
    for args, words in (((1, 1, 1, 0, 8, 4), "max_len"), ((1, 1, 1, 16, 0, 4), "head dims"), ((1, 1, 1, 16, 8, 0), "nodes"),
                        ((1, 1, 1, 16, 8, 65), "nodes"), ((1, 1 << 16, 1, 16, 8, 4), "sequences"), ((-1, 1, 1, 16, 8, 4), "layers"),
                        ((65535, 1, 65535, 16, 65535, 4), "too many"), ((1, 1, 1, 16, 8, 4, 9), "dtype")):
        assert compact(*args) == 1 and words in _hip.last_error(), args
    assert compact(1, 1, 1, 16, 8, 4, p=None) == 1 and "null" in _hip.last_error()


def test_references_of_the_walk_and_the_moves():
    """By hand: node 0 wants token 5, its children 1 (token 4) and 2 (token 5); 2 wants 7, its children 3 and 4 both hold it;
    3 wants 1 and has no child. The second sequence's node 0 is absent, the third's tokens are all wrong."""
    logits = torch.zeros(3, 5, 9)
    for node, want in enumerate((5, 0, 7, 1, 2)):
        logits[:, node, want] = 1
    tokens = torch.tensor([[3, 4, 5, 7, 7]] * 2 + [[3, 4, 4, 7, 7]])
    parents = torch.tensor([[-1, 0, 0, 2, 2], [-2, 0, 0, 2, 2], [-1, 0, 0, 2, 2]], dtype=torch.int32)
    path, count, following = accept_drafts_reference(logits, tokens, parents)
    assert path.tolist() == [[0, 2, 3, -1, -1], [-1] * 5, [0, -1, -1, -1, -1]]
    assert count.tolist() == [3, 0, 1] and following.tolist() == [1, -1, 5]
    k = torch.arange(2 * 10.0).reshape(2, 1, 10, 1).clone()
    v = -k
    compact_cache_reference(k, v, torch.tensor([4, 8]), torch.tensor([[0, 2, 3], [0, 1, 2]]), torch.tensor([3, 3]))
    assert k[0, 0, :, 0].tolist() == [0, 1, 2, 3, 4, 6, 7, 7, 8, 9] and torch.equal(v, -k)
    assert k[1, 0, :, 0].tolist() == list(range(10, 20))


def _tree(**change):
    a = dict(q=torch.zeros(2, 4, 3, 64), k_new=torch.zeros(2, 2, 3, 64), v_new=torch.zeros(2, 2, 3, 64),
             k_cache=torch.zeros(2, 2, 16, 64), v_cache=torch.zeros(2, 2, 16, 64), pos=torch.zeros(2, dtype=torch.int32),
             parents=torch.zeros(2, 3, dtype=torch.int32))
    a.update(change)
    return a


@pytest.mark.parametrize("change,words", [
    (dict(q=torch.zeros(2, 3, 64)), "q as"),
    (dict(q=torch.zeros(2, 3, 3, 64)), "multiple"),
    (dict(q=torch.zeros(2, 0, 3, 64)), "multiple"),
    (dict(k_new=torch.zeros(2, 2, 4, 64)), "k_new"),
    (dict(v_new=torch.zeros(2, 2, 3, 32)), "v_new"),
    (dict(k_new=torch.zeros(2, 0, 3, 64), v_new=torch.zeros(2, 0, 3, 64)), "multiple"),
    (dict(q=torch.zeros(2, 4, 65, 64), k_new=torch.zeros(2, 2, 65, 64), v_new=torch.zeros(2, 2, 65, 64)), "1 to 64"),
    (dict(q=torch.zeros(2, 4, 0, 64), k_new=torch.zeros(2, 2, 0, 64), v_new=torch.zeros(2, 2, 0, 64)), "1 to 64"),
    (dict(k_cache=torch.zeros(2, 4, 16, 64)), "caches"),
    (dict(v_cache=torch.zeros(2, 2, 17, 64)), "caches"),
    (dict(v_new=torch.zeros(2, 2, 3, 64, dtype=BF16)), "share a dtype"),
    (dict(v_cache=torch.zeros(2, 2, 64, 16).transpose(2, 3)), "contiguous"),
    (dict(pos=torch.zeros(3, dtype=torch.int32)), "pos"),
    (dict(parents=torch.zeros(2, 4, dtype=torch.int32)), "parents"),
    (dict(pos=torch.zeros(2, dtype=torch.long)), "int32"),
    (dict(parents=torch.zeros(2, 3)), "int32"),
])
def test_tree_refusals(change, words):
    with pytest.raises(ValueError, match=words):
        tree_attention(**_tree(**change))
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        tree_attention(**_tree())


def test_tree_abi_refusals():
    lib = _hip.lib()
    import ctypes

    a = 1 << 12
    strides = (ctypes.c_int64 * 9)(*[64] * 9)

    def call(b=2, h=4, hkv=2, t=3, n=1 << 12, d=64, dtype=_hip.BF16, q=a, ws=None, size=0, st=strides):
        return lib.ferrite_internal_tree_attention(q, a, a, a, a, a, a, a, st, b, h, hkv, t, n, d, dtype, 0.1, ws, size, None)

    assert call(b=0) == 0
    for change, words in ((dict(dtype=3), "dtype"), (dict(b=-1), "65535"), (dict(h=3), "multiple"), (dict(hkv=0), "multiple"),
                          (dict(t=0), "nodes"), (dict(t=65), "nodes"), (dict(n=0), "max_len"), (dict(n=1 << 25), "max_len"),
                          (dict(d=80), "head dim"), (dict(q=None), "null"), (dict(q=a + 8), "aligned"), (dict(), "workspace"),
                          (dict(st=(ctypes.c_int64 * 9)(*[68] * 9)), "aligned"),
                          (dict(b=65535, h=65535, hkv=65535, t=1, n=64), "too many heads")):
        assert call(**change) == 1, change
        assert words in _hip.last_error(), (change, _hip.last_error())
    need = lib.ferrite_internal_tree_attention_workspace(2, 4, 2, 3, 1 << 12, 64, _hip.BF16)
    assert need > 0 and call(ws=a, size=need - 1) == 1 and call(ws=a + 8, size=need) == 1
    assert lib.ferrite_internal_tree_attention_workspace(2, 4, 2, 3, 64, 64, _hip.BF16) == 0
    assert lib.ferrite_internal_tree_attention_workspace(2, 4, 3, 3, 64, 64, _hip.BF16) == -1


def test_tree_reference_is_attention_along_each_branch():
    """Each node's output is plain causal attention over the committed rows and the tokens of its own line."""
    g = torch.Generator().manual_seed(0)
    mk = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)
    q, kn, vn, kc, vc = mk(1, 2, 5, 64), mk(1, 1, 5, 64), mk(1, 1, 5, 64), mk(1, 1, 12, 64), mk(1, 1, 12, 64)
    parents = torch.tensor([[-1, 0, 0, 2, 4]], dtype=torch.int32)  # the last is absent
    k0, v0 = kc.clone(), vc.clone()
    out = tree_attention_reference(q, kn, vn, kc, vc, torch.tensor([6]), parents)
    for t, line in ((0, [0]), (1, [0, 1]), (2, [0, 2]), (3, [0, 2, 3])):
        keys, values = torch.cat([k0[0, 0, :6], kn[0, 0, line]]), torch.cat([v0[0, 0, :6], vn[0, 0, line]])
        for h in range(2):
            e = torch.softmax(keys @ q[0, h, t] / 8, -1) @ values
            assert torch.allclose(out[0, h, t], e, atol=1e-12)
    assert not out[0, :, 4].any()
    assert torch.equal(kc[0, 0, 6:10], kn[0, 0, :4]) and torch.equal(kc[0, 0, 10:], k0[0, 0, 10:])
    assert ancestors(parents)[0].int().tolist() == [[1, 0, 0, 0, 0], [1, 1, 0, 0, 0], [1, 0, 1, 0, 0], [1, 0, 1, 1, 0], [0] * 5]


@pytest.mark.parametrize("t,pos", [(1, [0, 16]), (4, [2, 13]), (4, [2, 15]), (3, [0, 14, 13, -1, 16])])
def test_tree_reference_checks_every_sequence_against_the_whole_tree(t, pos):
    """A sequence whose rows pos .. pos + T - 1 do not lie in the cache is NaN and writes nothing, whatever nodes the one before it
    has."""
    g = torch.Generator().manual_seed(1)
    mk = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)
    b, length = len(pos), 16
    q, kn, vn, kc, vc = mk(b, 2, t, 64), mk(b, 1, t, 64), mk(b, 1, t, 64), mk(b, 1, length, 64), mk(b, 1, length, 64)
    parents = (torch.arange(t) - 1).int().expand(b, t).clone()
    parents[0, 1:] = -2  # the first sequence has one node
    k0, v0 = kc.clone(), vc.clone()
    out = tree_attention_reference(q, kn, vn, kc, vc, torch.tensor(pos), parents)
    for i, p in enumerate(pos):
        inside = 0 <= p <= length - t
        assert bool(torch.isnan(out[i]).any()) == (not inside)
        assert torch.equal(kc[i], k0[i]) != inside and torch.equal(vc[i], v0[i]) != inside


def test_overlapping_caches_are_refused():
    """By address, before any launch: caches that share a byte, and inputs that reach into one."""
    import ctypes

    lib = _hip.lib()
    k = 1 << 30
    compact = lambda v: lib.ferrite_internal_compact_cache(k, v, 4096, 4096, 4096, 3, 2, 4, 100, 64, 8, _hip.BF16, None)
    size = 3 * 2 * 4 * 100 * 64 * 2
    for v in (k, k + size - 16, k - size + 16, k + 2):
        assert compact(v) == 1 and "overlap" in _hip.last_error(), v
    b, h, hkv, t, n, d = 2, 4, 2, 3, 128, 64
    size, far = b * hkv * n * d * 2, 1 << 34
    dense = [v for heads in (h, hkv, hkv) for v in (heads * t * d, t * d, d)]

    def tree(q=far, kn=far + (1 << 20), vn=far + (2 << 20), vc=far << 1, st=dense):
        return lib.ferrite_internal_tree_attention(q, kn, vn, k, vc, 4096, 4096, 1 << 40, (ctypes.c_int64 * 9)(*st), b, h, hkv, t, n, d,
                                                   _hip.BF16, 0.1, None, 0, None)

    rows, q_rows = b * hkv * t * d * 2, b * h * t * d * 2
    for change in (dict(vc=k), dict(vc=k + size - 16), dict(vc=k - size + 16), dict(q=k), dict(q=k + size - 16), dict(q=k - q_rows + 16),
                   dict(kn=k + 512), dict(kn=k - rows + 16), dict(vn=k), dict(vn=(far << 1) + size - 16), dict(kn=(far << 1)),
                   dict(kn=k - 4096 + rows, st=[*dense[:3], 2048, t * d, d, *dense[6:]])):  # a view's last sequence
        assert tree(**change) == 1 and "overlap" in _hip.last_error(), change
