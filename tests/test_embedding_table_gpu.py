"""GPU tests of the embedding over any vocabulary (csrc/embedding.hip), against the formulas in 64 bits.

The forward is one f32 product, rounded once: compared bit by bit. A table row's gradient adds n rows of dout in f32: at most 64 in a
piece, then 16 sums of every 16th piece and those: with u = 2^-24, off by at most (min(n, 64) + n / 256 + 20) u of the sum of their
sizes, one more u for the scale, and half a step of the table's type."""

import pytest
import torch

from ferrite import _hip
from ferrite.kernels.embedding import embedding, embedding_reference

pytestmark = pytest.mark.gpu

U = 2.0**-24
HALF = {torch.bfloat16: 2.0**-8, torch.float32: 2.0**-24}
BF16, F32 = torch.bfloat16, torch.float32


def _tokens(kind, rows, vocab, g):
    if kind == "even":
        return torch.randint(0, vocab, (rows,), generator=g)
    if kind == "text":  # the k-th token about once in k
        return (float(vocab) ** torch.rand(rows, generator=g, dtype=torch.float64)).long().clamp(1, vocab) - 1
    if kind == "one":
        return torch.full((rows,), vocab // 2)
    if kind == "runs":  # tokens whose rows end with a piece and one row before or behind it
        return torch.repeat_interleave(torch.arange(8 * rows), torch.tensor([16, 15, 17, 1, 48, 64, 128, 31]).repeat(rows))[:rows] % vocab
    return torch.arange(rows - 1, -1, -1) % vocab  # "down"


def _check_grad(d, tokens, dy, table, scale, pad=None):
    t, n = tokens.reshape(-1), table.shape[0]
    keep = (t >= 0) & (t < n) & (t != (-1 if pad is None else pad))
    line, rows = t[keep], dy.reshape(-1, dy.shape[-1])[keep].double()
    ref = torch.zeros(table.shape, dtype=torch.float64, device=table.device).index_add_(0, line, rows) * scale
    size = torch.zeros(table.shape, dtype=torch.float64, device=table.device).index_add_(0, line, rows.abs()) * abs(scale)
    count = torch.bincount(line, minlength=n).double()[:, None]
    tol = U * (count.clamp(max=64) + count / 256 + 21) * size + 1.01 * HALF[d.dtype] * ref.abs()
    assert d.shape == table.shape and d.dtype == table.dtype
    assert bool(((d.double() - ref).abs() <= tol).all())  # rows of no token: exactly zero


CASES = [
    # rows, vocab, dim, tokens
    (1, 1, 1, "even"), (1, 50257, 64, "even"), (2, 3, 7, "one"), (63, 256, 8, "even"), (64, 256, 512, "text"),
    (65, 10, 9, "even"), (1000, 2, 515, "even"), (1000, 100, 16, "runs"), (4097, 1000, 24, "down"), (4096, 32768, 768, "text"),
    (8192, 50257, 130, "text"), (5000, 7, 3, "one"), (5000, 262143, 40, "text"), (16384, 262143, 12, "text"), (16384, 3000, 520, "runs"),
    (3000, 262144, 33, "text"), (16385, 1, 5, "one"), (16385, 1025, 72, "text"), (20000, 300000, 10, "even"), (40000, 50000, 96, "text"),
    (70001, 255, 8, "runs"), (70001, 1 << 21, 8, "even"), (131072, 5, 64, "one"), (33000, 1023, 1, "down"),
]


@pytest.mark.parametrize("rows,vocab,dim,kind", CASES)
@pytest.mark.parametrize("table_dtype,out_dtype", [(BF16, BF16), (F32, F32), (F32, BF16), (BF16, F32)])
def test_forward_and_gradient(dev, rows, vocab, dim, kind, table_dtype, out_dtype):
    g = torch.Generator().manual_seed(rows + vocab)
    tokens = _tokens(kind, rows, vocab, g).to(dev)
    table = torch.randn(vocab, dim, generator=g).to(dev, table_dtype).requires_grad_()
    dy = torch.randn(rows, dim, generator=g).to(dev, out_dtype)
    out = embedding(tokens, table, scale=1.7, dtype=out_dtype)
    ref = embedding_reference(tokens, table.detach(), scale=1.7, dtype=out_dtype)
    assert out.dtype == out_dtype and torch.equal(out.detach(), ref)
    with torch.no_grad():
        assert torch.equal(embedding(tokens.int(), table, scale=1.7, dtype=out_dtype), ref)
    d, = torch.autograd.grad(out, table, dy, retain_graph=True)
    _check_grad(d, tokens, dy, table.detach(), 1.7)
    assert torch.equal(d, torch.autograd.grad(out, table, dy)[0])


@pytest.mark.parametrize("rows", [100, 5000, 20000])
def test_padding_and_tokens_outside_the_table(dev, rows):
    g = torch.Generator().manual_seed(rows)
    tokens = torch.randint(0, 50, (2, rows // 2), generator=g).to(dev)
    tokens[1, rows // 3:] = 7
    tokens[0, ::5] = 50
    tokens[0, 1::5] = -1
    tokens[1, 0] = 1 << 40
    tokens[1, 1] = -(1 << 40)
    table = torch.randn(50, 24, generator=g).to(dev).requires_grad_()
    dy = torch.randn(2, rows // 2, 24, generator=g).to(dev)
    for pad in (None, 7, 0):
        out = embedding(tokens, table, scale=0.5, padding_idx=pad)
        ref = embedding_reference(tokens, table.detach(), scale=0.5)
        assert torch.equal(out.isnan(), ref.isnan()) and torch.equal(out.nan_to_num(), ref.nan_to_num())
        d, = torch.autograd.grad(out, table, dy)
        _check_grad(d, tokens, dy, table.detach(), 0.5, pad)
        assert pad is None or not d[pad].any()


def test_no_row_has_a_gradient(dev):
    table = torch.randn(9, 16, device=dev, requires_grad=True)
    for tokens in (torch.zeros(0, 4, dtype=torch.long, device=dev), torch.full((300,), 9, device=dev), torch.full((20000,), -5, device=dev)):
        out = embedding(tokens, table)
        assert out.shape == (*tokens.shape, 16)
        assert not torch.autograd.grad(out, table, torch.ones_like(out))[0].any()


def test_bad_rows_reach_their_token_alone(dev):
    tokens = torch.arange(40, device=dev).repeat(50)
    table = torch.randn(40, 20, device=dev, requires_grad=True)
    out = embedding(tokens, table)
    dy = torch.randn(2000, 20, device=dev)
    good, = torch.autograd.grad(out, table, dy, retain_graph=True)
    dy[83, 3], dy[124, 4] = float("nan"), float("inf")
    bad, = torch.autograd.grad(out, table, dy)
    mask = torch.zeros_like(good, dtype=torch.bool)
    mask[3, 3] = mask[4, 4] = True
    assert torch.equal(good[~mask], bad[~mask]) and bool(bad[3, 3].isnan()) and bool(bad[4, 4].isinf())


def test_one_token(dev):
    table = torch.randn(300, 20, device=dev, requires_grad=True)
    token = torch.tensor(123, device=dev)
    out = embedding(token, table, scale=3.0)
    assert out.shape == (20,) and torch.equal(out.detach(), table.detach()[123] * 3)
    d, = torch.autograd.grad(out.sum(), table)
    assert bool((d[123] == 3).all()) and int(d.count_nonzero()) == 20


def test_layouts(dev):
    big = torch.randn(100, 66, device=dev)
    tokens = torch.randint(0, 50, (6, 10), device=dev)
    for table in (big[:50, 1:65], big.t()[:50], big.reshape(-1)[1:3201].view(50, 64)):
        leaf = table.detach().requires_grad_()
        for ids in (tokens, tokens.t(), tokens[:, ::3]):
            out = embedding(ids, leaf)
            assert torch.equal(out.detach(), table[ids])
            dy = torch.randn(table.shape[1], *ids.shape, device=dev).movedim(0, -1)
            _check_grad(torch.autograd.grad(out, leaf, dy, retain_graph=True)[0], ids, dy, table, 1.0)
    row = torch.randn(64, device=dev)
    d, = torch.autograd.grad(out, leaf, row[:table.shape[1]].expand_as(out))  # one gradient for every row
    _check_grad(d, ids, row[:table.shape[1]].expand_as(out).contiguous(), table, 1.0)


@pytest.mark.parametrize("rows", [50, 17000])
@pytest.mark.parametrize("offset", [0, 1, 3])
def test_nothing_beside_the_table_is_written(dev, rows, offset):
    """Through the entry point, into the middle of a buffer that starts between 16-byte boundaries."""
    vocab, dim = 61, 19
    g = torch.Generator().manual_seed(3)
    tokens = torch.randint(-1, vocab + 1, (rows,), generator=g).to(dev)
    dy = torch.randn(rows, dim, generator=g).to(dev, BF16)
    room = torch.full((vocab * dim + 64,), 5.0, device=dev, dtype=BF16)
    d = room[24 + offset:24 + offset + vocab * dim]
    lib = _hip.lib()
    ws = torch.empty(lib.ferrite_internal_embedding_bwd_workspace(rows, dim, vocab), dtype=torch.uint8, device=dev)
    rc = lib.ferrite_internal_embedding_bwd(tokens.data_ptr(), dy.data_ptr(), d.data_ptr(), rows, dim, vocab, -1, 1.0, 0, _hip.BF16,
                                            _hip.BF16, ws.data_ptr(), ws.numel(), _hip.stream_of(d))
    assert rc == _hip.OK
    _check_grad(d.view(vocab, dim), tokens, dy, d.view(vocab, dim), 1.0)
    assert bool((room[:24 + offset] == 5).all()) and bool((room[24 + offset + vocab * dim:] == 5).all())


@pytest.mark.parametrize("rows", [2000, 30000])
def test_another_stream_and_a_captured_step(dev, rows):
    g = torch.Generator().manual_seed(rows)
    tokens = torch.randint(0, 500, (rows,), generator=g).to(dev)
    table = torch.randn(500, 72, generator=g).to(dev, BF16).requires_grad_()
    dy = torch.randn(rows, 72, generator=g).to(dev, BF16)

    def step(table):
        out = embedding(tokens, table, scale=2.0)
        return out, *torch.autograd.grad(out, table, dy)

    ref = step(table)
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        leaf = table.detach().clone().requires_grad_()
        out = step(leaf)
    side.synchronize()
    assert torch.equal(out[0], ref[0]) and torch.equal(out[1], ref[1])
    del out
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(leaf)
    for k in range(3):
        tokens.copy_(tokens.roll(k) // (k + 1))
        graph.replay()
        want = step(table)
        torch.cuda.synchronize()
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


@pytest.mark.parametrize("rows", [900, 20000])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_the_model_embeds_large_vocabularies_with_it(dev, rows, dtype):
    """GPT's residual stream over a vocabulary past 1024: as torch's indexing gives it, negative tokens counted from the end, and the
    table's gradient within the tolerance above."""
    from ferrite.model.gpt import GPTConfig, _embed_tokens

    cfg = GPTConfig(vocab_size=3000, seq_len=rows // 2, d_model=72, n_head=1)
    g = torch.Generator().manual_seed(rows)
    tok = torch.randn(3000, 72, generator=g).to(dev, dtype).requires_grad_()
    pe = torch.randn(rows // 2, 72, generator=g).to(dev, dtype).requires_grad_()
    tokens = torch.randint(-3000, 3000, (2, rows // 2), generator=g).to(dev)
    dh = torch.randn(2, rows // 2, 72, generator=g).to(dev, BF16)
    h = _embed_tokens(tok, pe, tokens, cfg)
    def names(fn):
        return [] if fn is None else [fn.name(), *(n for f, _ in fn.next_functions for n in names(f))]

    assert any("EmbeddingFn" in n for n in names(h.grad_fn))
    assert torch.equal(h, (tok[tokens] + pe).to(BF16))
    d, dp = torch.autograd.grad(h, (tok, pe), dh)
    _check_grad(d, tokens % 3000, dh.to(dtype), tok.detach(), 1.0)
    want = torch.autograd.grad((tok[tokens] + pe).to(BF16), pe, dh)[0]
    assert torch.equal(dp, want)


def test_a_graphed_training_step_over_a_large_vocabulary(dev):
    """The model's captured step beside the eager one, from the same parameters at every step, text-like tokens. Losses agree to 1e-6, moments
    and parameters to 1e-6 where a step moves parameters by 3e-3."""
    from ferrite.model.gpt import GPTConfig, init_params
    from ferrite.model.train import TrainConfig, adamw_init, build_train_step, leaves

    cfg = GPTConfig(vocab_size=3000, seq_len=128, d_model=256, n_head=2, n_layer=1, d_ff=512, linear="pallas")
    tcfg = TrainConfig(steps=10, warmup=2, lr=3e-3)
    pa, pb = init_params(4, cfg, device=dev), init_params(4, cfg, device=dev)
    sa, sb = adamw_init(pa), adamw_init(pb)
    eager, graphed = build_train_step(cfg, tcfg), build_train_step(cfg, tcfg, graph=True)
    g = torch.Generator().manual_seed(6)
    for _ in range(6):
        with torch.no_grad():
            for a, b in zip(leaves(pa) + leaves(sa["m"]) + leaves(sa["v"]), leaves(pb) + leaves(sb["m"]) + leaves(sb["v"])):
                a.copy_(b)
        sa["step"] = sb["step"]
        x, y = (_tokens("text", 512, 3000, g).view(4, 128).to(dev) for _ in range(2))
        pa, sa, la, _ = eager(pa, sa, x, y)
        pb, sb, lb, _ = graphed(pb, sb, x, y)
        assert abs(float(la) - float(lb)) <= 1e-6 * abs(float(la))
        for a, b in zip(leaves(pa) + leaves(sa["m"]) + leaves(sa["v"]), leaves(pb) + leaves(sb["m"]) + leaves(sb["v"])):
            assert float((a.detach() - b.detach()).abs().max()) <= 1e-6
    assert graphed.graph is not None


def test_capture_refuses_leaves_that_an_eager_graph_holds(dev):
    table, tokens = torch.randn(40, 8, device=dev, requires_grad=True), torch.zeros(5, dtype=torch.long, device=dev)
    held = embedding(tokens, table)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="holds one of its leaves"):
        with torch.cuda.graph(graph):
            embedding(tokens, table)
    del held


def test_forward_mode_is_refused(dev):
    import torch.autograd.forward_ad as fwd

    table, tokens = torch.randn(40, 8, device=dev), torch.zeros(5, dtype=torch.long, device=dev)
    with fwd.dual_level(), pytest.raises((RuntimeError, NotImplementedError)):
        embedding(tokens, fwd.make_dual(table, torch.ones_like(table)))


def test_a_table_that_is_not_dense_is_not_copied_to_look_it_up(dev):
    from ferrite.model.gpt import GPTConfig, _embed_tokens

    cfg = GPTConfig(vocab_size=40000, seq_len=16, d_model=512, n_head=1)
    tok, pe = torch.randn(40000, 520, device=dev)[:, :512], torch.randn(16, 512, device=dev)
    tokens = torch.randint(0, 40000, (2, 8), device=dev)
    with torch.no_grad():
        _embed_tokens(tok, pe, tokens, cfg)
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        h = _embed_tokens(tok, pe, tokens, cfg)
        assert torch.cuda.max_memory_allocated() - before < 1 << 20
    assert torch.equal(h, (tok[tokens] + pe[:8]).to(cfg.dtype))
