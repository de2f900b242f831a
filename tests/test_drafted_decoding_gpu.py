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
