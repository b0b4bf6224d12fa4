"""Embedding, residual norms and the 8-bit cache on streams of their own, and captured into graphs."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def state(seed, *, t=300, c=512, vocab=181, slot=700, docs=3):
    g = torch.Generator().manual_seed(seed)
    s = {"ids": torch.randint(-1, vocab, (t,), generator=g).int(), "table": torch.randn(vocab, c, generator=g), "dy": torch.randn(t, c, generator=g),
         "z": torch.randn(t, c, generator=g), "w": 1 + 0.1 * torch.randn(c, generator=g), "q": torch.randn(docs, 8, 64, generator=g),
         "kv": torch.randn(2, docs, 4, 64, generator=g), "k_len": torch.randint(1, slot + 1, (docs,), generator=g).int(),
         "codes": torch.randint(-127, 128, (2, docs * slot, 4, 64), generator=g).to(torch.int8), "scales": torch.rand(2, 4, docs * slot, generator=g) * 0.02}
    return {k: v.cuda() for k, v in s.items()} | {"q_off": torch.arange(docs + 1).int().cuda(), "k_off": (torch.arange(docs + 1) * slot).int().cuda()}


def work(ctx, s):
    """Every operator once, each on what the one before it made where it can be."""
    from brosoundml_amd import tokens
    cache = tokens.Cache(*s["codes"], *s["scales"])
    x = tokens.embedding(ctx, s["table"], s["ids"], scale=2.0)
    rule = dict(post=s["w"], pre=(s["w"], s["w"]), gate=s["w"], kind="layer")
    r, y, stats = tokens.residual_norm(ctx, x, s["z"], keep=True, **rule)
    dx, dz, dgate, dpost, dpre = tokens.residual_norm_bwd(ctx, x, s["z"], s["dy"], y, stats, **rule)
    dtable = tokens.embedding_bwd(ctx, s["ids"], dx, s["table"].shape[0], scale=2.0)
    where = s["q_off"], s["k_off"], s["k_len"]
    tokens.cache_write(ctx, *s["kv"], cache, *where)
    k, v = tokens.cache_read(ctx, cache, *where, rows=3, width=64, dtype=torch.float32)
    o, lse = tokens.cache_attention(ctx, s["q"], cache, *where, causal=True)
    return [x, r, y, dx, dz, dgate, dpost[0], dpre[0], dpre[1], dtable, k, v, o, lse, *cache]


def same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


def test_a_stream_of_its_own():
    from brosoundml_amd import native
    s = state(1)
    want = [t.clone() for t in work(native.Context(0), s)]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    ctx = native.Context(0, stream=side)
    got = work(ctx, state(1))  # called on the current stream, run on the context's
    side.synchronize()
    assert same(got, want)
    # both at once, each with its context
    other = native.Context(0)
    s1, s2 = state(1), state(1)
    torch.cuda.synchronize()
    a, b = work(ctx, s1), work(other, s2)
    torch.cuda.synchronize()
    assert same(a, want) and same(b, want)


def test_two_graphs_of_one_context():
    """Two captured passes share the context's workspaces; replayed in turn on its stream, with its own calls between,
    each gives what its inputs make."""
    from brosoundml_amd import native
    side = torch.cuda.Stream()
    ctx = native.Context(0, stream=side)
    states = [state(2), state(3, t=1000, slot=2000)]
    graphs, outs = [], []
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for s in states:
            work(ctx, s)
    side.synchronize()
    for s in states:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            outs.append(work(ctx, s))
        graphs.append(g)
    for turn in range(4):
        for s, g, o in zip(states, graphs, outs):
            fresh = state(10 * turn + 5, t=s["ids"].shape[0], slot=s["codes"].shape[1] // 3)
            with torch.cuda.stream(side):
                for k, v in fresh.items():
                    s[k].copy_(v)
                g.replay()
                want = work(ctx, fresh)
            side.synchronize()
            assert same(o, want), turn


def test_a_graph_keeps_its_workspaces():
    """A later call whose workspace the device cannot hold makes the context give back its pooled blocks: not those that a
    graph uses. What the blocks' memory could become meanwhile is written over between the replays."""
    from brosoundml_amd import native, tokens
    side = torch.cuda.Stream()
    ctx = native.Context(0, stream=side)
    s = state(4)
    want = [t.clone() for t in work(native.Context(0), state(4))]
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        work(ctx, s)
    side.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        out = work(ctx, s)
    ids = torch.zeros(1 << 24, dtype=torch.int32, device="cuda")
    dy = torch.zeros(1, 1 << 20, dtype=torch.bfloat16, device="cuda").expand(1 << 24, 1 << 20)
    torch.cuda.synchronize()
    for _ in range(3):
        with torch.cuda.stream(side):
            with pytest.raises(native.KdecError, match="memory|hipMalloc"):
                tokens.embedding_bwd(ctx, ids, dy, 1)  # 2 TB of partial sums
        other = torch.full((1 << 24,), float("nan"), device="cuda")
        with torch.cuda.stream(side):
            g.replay()
        side.synchronize()
        assert same(out, want)
        del other
