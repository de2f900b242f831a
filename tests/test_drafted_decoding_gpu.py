"""A drafted decoding step whole (csrc/heads_rope.hip, csrc/tree.hip, csrc/drafts.hip): two layers of projection, qk_norm_rope,
tree_attention and an output product, then accept_drafts and compact_cache, against greedy decoding of one token after
another over whole sequences in 64 bits on the host.

Both choose tokens, so nothing is compared within a tolerance: the weights' seed is one whose 64-bit logits keep
the chosen token 1e-3 above the next, which is asserted (f32 logits of size 1 from sums of 256 products are off by
under 256 * 2^-24 * 4 = 6e-5; the test's argmax cannot differ)."""

import pytest
import torch

from ferrite.kernels.drafts import accept_drafts, compact_cache
from ferrite.kernels.qk_norm_rope import qk_norm_rope, qk_norm_rope_reference, rope_tables
from ferrite.kernels.tree_attention import tree_attention

pytestmark = pytest.mark.gpu

VOCAB, H, HKV, D, LAYERS, LENGTH = 61, 4, 2, 64, 2, 96
C = H * D


def _weights(seed):
    g = torch.Generator().manual_seed(seed)
    mk = lambda *s, scale=1.0: torch.randn(*s, generator=g, dtype=torch.float64) * scale
    layers = [(mk(C, (H + 2 * HKV) * D, scale=C**-0.5), mk(D, scale=0.2) + 1, mk(D, scale=0.2) + 1, mk(C, C, scale=C**-0.5))
              for _ in range(LAYERS)]
    return mk(VOCAB, C), layers, mk(C, VOCAB, scale=C**-0.5)


def _plain(weights, tokens, n):
    """tokens and the n that greedy decoding puts behind them, and the smallest lead of a chosen one."""
    emb, layers, head = weights
    cos, sin = rope_tables(LENGTH, D)
    tokens, lead = list(tokens), float("inf")
    for _ in range(n):
        x, s = emb[tokens], len(tokens)
        hidden = torch.ones(s, s).triu(1).bool()
        for wqkv, wq, wk, wo in layers:
            q, k, v = qk_norm_rope_reference((x @ wqkv)[None], wq, wk, cos, sin, n_head=H, n_kv_head=HKV)
            k, v = (t.repeat_interleave(H // HKV, 1) for t in (k, v))
            w = torch.softmax((q @ k.transpose(2, 3) / D**0.5).masked_fill(hidden, float("-inf")), -1)
            x = x + (w @ v)[0].transpose(0, 1).reshape(s, C) @ wo
        top = (x[-1] @ head).topk(2)
        lead = min(lead, float(top.values[0] - top.values[1]))
        tokens.append(int(top.indices[0]))
    return tokens, lead


def _draft(line, t, right, g):
    """A tree of t nodes on the token line[0]: `right` more of the line as its main chain, wrong tokens beside and behind."""
    tokens, parents, depths, main = [line[0]], [-1], [0], 0
    for i in range(1, t):
        wrong = i % 3 == 0 or depths[main] >= right
        up = int(torch.randint(i, (1,), generator=g)) if wrong else main
        token = line[depths[main] + 1]
        if wrong:  # never what the line has after this node
            after = line[depths[up] + 1]
            token = (after + 1 + int(torch.randint(VOCAB - 1, (1,), generator=g))) % VOCAB
        tokens.append(token)
        parents.append(up)
        depths.append(depths[up] + 1)
        if not wrong:
            main = i
    return tokens, parents, depths


@pytest.mark.parametrize("t", [1, 5, 24])
def test_drafted_steps_decode_like_single_tokens(dev, t):
    weights = _weights(3)
    g = torch.Generator().manual_seed(t)
    starts = [[7], [3, 50, 21, 8, 30, 2, 44], [11, 19, 60]]
    b, n = len(starts), 48
    want, leads = zip(*(_plain(weights, s, n) for s in starts))
    assert min(leads) > 1e-3
    to = lambda x: x.float().to(dev)
    emb, head, layers = to(weights[0]), to(weights[2]), [[to(w) for w in layer] for layer in weights[1]]
    cos, sin = rope_tables(LENGTH, D, device=dev)
    kc, vc = (torch.full((LAYERS, b, HKV, LENGTH, D), float("nan"), device=dev) for _ in range(2))
    mk = lambda dtype: torch.zeros(b, t, dtype=dtype, device=dev)
    pos, tokens, parents, depths = torch.zeros(b, dtype=torch.int32, device=dev), mk(torch.int64), mk(torch.int32), mk(torch.int32)

    def step():
        """Attends, accepts, keeps and moves on."""
        x = emb[tokens]
        for layer, (wqkv, wq, wk, wo) in enumerate(layers):
            q, k, v = qk_norm_rope(x @ wqkv, wq, wk, cos, sin, n_head=H, n_kv_head=HKV, positions=pos[:, None] + depths)
            a = tree_attention(q, k, v, kc[layer], vc[layer], pos, parents)
            x = x + a.transpose(1, 2).reshape(b, t, C) @ wo
        path, count, following = accept_drafts(x @ head, tokens, parents)
        compact_cache(kc, vc, pos, path, count)
        pos.add_(count)
        return path, count, following

    with torch.no_grad():
        # The first tokens, a chain at a time; absent nodes fill the short ones up.
        done = [0] * b
        while any(d + 1 < len(s) for d, s in zip(done, starts)):
            parents.fill_(-2)
            for i, s in enumerate(starts):
                chunk = s[done[i]: done[i] + t][: len(s) - 1 - done[i]]
                tokens[i, : len(chunk)] = torch.tensor(chunk, dtype=torch.int64)
                parents[i, : len(chunk)] = torch.arange(len(chunk)) - 1
                depths[i, : len(chunk)] = torch.arange(len(chunk))
                done[i] += len(chunk)
            step()
            pos.copy_(torch.tensor(done))
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        before = pos.clone()
        with torch.cuda.graph(graph):
            outs = step()
        assert torch.equal(pos, before)
        got, steps = [list(s) for s in starts], 0
        while min(len(x) - len(s) for x, s in zip(got, starts)) < 20:
            for i in range(b):
                line = want[i][len(got[i]) - 1:]
                right = int(torch.randint(t, (1,), generator=g))
                if len(line) <= t + 2:  # this one has got far enough: it waits
                    parents[i] = -2
                    continue
                for x, y in zip((tokens, parents, depths), _draft(line, t, right, g)):
                    x[i] = torch.tensor(y)
            if steps % 2:
                path, count, following = step()
            else:
                graph.replay()
                path, count, following = outs
            for i in range(b):
                nodes = path[i, : count[i]].tolist()
                got[i] += tokens[i, nodes[1:]].tolist() + ([int(following[i])] if nodes else [])
                assert got[i] == want[i][: len(got[i])]
            steps += 1
        assert pos.tolist() == [len(x) - 1 for x in got]
        if t > 4:
            assert sum(len(x) - len(s) for x, s in zip(got, starts)) > b * steps  # drafts were taken
        graph.reset()


@pytest.mark.parametrize("h,hkv,t,d,length", [
    (4, 2, 8, 64, 300), (4, 4, 6, 128, 2500), (8, 2, 8, 128, 900), (8, 2, 24, 128, 1200), (4, 1, 40, 256, 700), (16, 2, 60, 64, 500)])
def test_bf16_steps_are_their_operators(dev, h, hkv, t, d, length):
    """Steps in bf16, with few rows a key head and with many that share keys, in turn plain and replayed: every operator's outputs are
    what its definition gives in 64 bits for the inputs that it had in that step. The heads are off by half a bf16 step and 20 * 2^-24
    of a pair's size (under 2 * 16), the attention by half a step, 2^-16 of the values (up to 5.5) and 4.8e-5; tokens, paths and
    cached rows are equal."""
    from ferrite.kernels.drafts import accept_drafts_reference, compact_cache_reference
    from ferrite.kernels.tree_attention import tree_attention_reference

    from tests.test_drafts_gpu import trees

    g = torch.Generator().manual_seed(t)
    b, c, bf = 3, h * d, torch.bfloat16
    mk = lambda *s, scale=1.0: (torch.randn(*s, generator=g) * scale).to(dev, bf)
    layers = [(mk(c, (h + 2 * hkv) * d, scale=c**-0.5), mk(d, scale=0.1) + 1, mk(d, scale=0.1) + 1, mk(c, c, scale=c**-0.5))
              for _ in range(2)]
    head, x0 = mk(c, 71, scale=c**-0.5), mk(b, t, c)
    cos, sin = rope_tables(length, d, device=dev)
    kc, vc = mk(2, b, hkv, length, d), mk(2, b, hkv, length, d)
    ints = lambda *s: torch.zeros(*s, dtype=torch.int32, device=dev)
    pos, tokens, parents, depths = ints(b), ints(b, t), ints(b, t), ints(b, t)

    def step():
        x, seen = x0, []
        for layer, (wqkv, wq, wk, wo) in enumerate(layers):
            qkv = x @ wqkv
            q, k, v = qk_norm_rope(qkv, wq, wk, cos, sin, n_head=h, n_kv_head=hkv, positions=pos[:, None] + depths)
            a = tree_attention(q, k, v, kc[layer], vc[layer], pos, parents)
            x = x + a.transpose(1, 2).reshape(b, t, c) @ wo
            seen.append((qkv, q, k, v, a))
        logits = x @ head
        kept = accept_drafts(logits, tokens, parents)
        compact_cache(kc, vc, pos, kept[0], kept[1])
        return seen, logits, kept

    def draw(seed):
        up = trees(b, t, seed, absent=0.1)
        up[:, 0] = -1
        deep = torch.zeros(b, t, dtype=torch.int32)
        for i in range(1, t):
            deep[:, i] = torch.where((up[:, i] >= 0) & (up[:, i] < i), deep.gather(1, up[:, i:i + 1].clamp(0, t - 1).long())[:, 0] + 1, 0)
        parents.copy_(up)
        depths.copy_(deep)
        pos.copy_(torch.tensor([length - t - seed, 40 + seed, length // 2]))
        x0.copy_(mk(b, t, c))

    half = lambda r: torch.exp2(torch.floor(torch.log2(r.abs().clamp(min=2.0**-126))) - 8) * 1.001
    with torch.no_grad():
        draw(0)
        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step()
        taken = 0
        for seed in range(1, 5):
            draw(seed)
            held = kc.clone(), vc.clone()
            wanted = step()[1].float().argmax(-1)  # the drafts do not feed the step: most of them hold what it wants
            hit = (torch.rand(b, t, generator=g) < 0.7).to(dev)
            tokens.copy_(torch.where(hit, wanted.gather(1, parents.clamp(0, t - 1).long()), 70 - wanted))
            for c0, c1 in zip((kc, vc), held):
                c0.copy_(c1)
            if seed % 2:
                graph.replay()
                seen, logits, kept = outs
            else:
                seen, logits, kept = step()
            k64, v64 = (x.double() for x in held)
            for layer, ((qkv, q, k, v, a), (_, wq, wk, _)) in enumerate(zip(seen, layers)):
                ref = qk_norm_rope_reference(*(x.double() for x in (qkv, wq, wk, cos, sin)), n_head=h, n_kv_head=hkv,
                                             positions=pos[:, None] + depths)
                for x, r in zip((q, k, v), ref):
                    assert bool(((x.double() - r).abs() <= half(r) + 20 * 2.0**-24 * 32).all())
                r = tree_attention_reference(*(x.double() for x in (q, k, v)), k64[layer], v64[layer], pos, parents)
                assert bool(((a.double() - r).abs() <= half(r) + 5.5 * 2.0**-16 + 4.8e-5).all())
            want = accept_drafts_reference(logits.float().cpu(), tokens.cpu(), parents.cpu())
            assert all(torch.equal(x.cpu(), y) for x, y in zip(kept, want))
            compact_cache_reference(k64, v64, pos, kept[0], kept[1])
            assert torch.equal(kc.double(), k64) and torch.equal(vc.double(), v64)
            taken += int(kept[1].sum()) - b
        assert taken > 4
        graph.reset()
