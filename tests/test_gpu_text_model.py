"""The example's text model: embedding, norms, attention, adapters and the 8-bit cache together."""
import importlib.util
import os

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "voiced_text.py")
    spec = importlib.util.spec_from_file_location("voiced_text", path)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


@pytest.fixture(scope="module")
def ctx():
    from brosoundml_amd import native
    return native.Context(0)


def low_rank(model, seed):
    g = torch.Generator().manual_seed(seed)
    for block in model.blocks:
        for i in (1, 3):
            block.low[i].copy_(torch.randn(block.low[i].shape, generator=g) * 0.3)


@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_gradients_against_torch(example, ctx, dtype, kind):
    """All gradients (no dropout) against autograd in 64 bits on the same weights. In float the sums are good to
    2^-20 of their terms' norm; in bf16 each of the two blocks rounds some nine tensors on the way forward and as
    many back (2^-9 root mean square each): 36 of them make 1.2 %, and 3 % leaves room for the softmax and the norms
    passing them on enlarged."""
    width, head, voices, rank, vocab = 128, 32, 3, 8, 40
    model = example.TextModel(ctx, vocab, width, head, voices, rank, kind=kind, causal=True, dtype=dtype)
    low_rank(model, 3)
    cuts = [0, 5, 6, 90]
    g = torch.Generator().manual_seed(4)
    ids = torch.randint(-1, vocab, (90,), generator=g).int()
    off, voice = torch.tensor(cuts, dtype=torch.int32).cuda(), torch.repeat_interleave(torch.tensor([2, 0, 1]), torch.tensor(cuts).diff()).int().cuda()
    dh = torch.randn(90, width, generator=g).to(dtype).cuda()
    h, state = model.forward(ids.cuda(), voice, off, 0, 0)
    got = model.backward(dh, state)

    leaf = lambda t: None if t is None else t.double().cpu().requires_grad_()  # noqa: E731
    table, who = leaf(model.table), voice.long().cpu()
    pre, post = [tuple(map(leaf, p)) for p in model.pre], [tuple(map(leaf, p)) for p in model.post]
    gate, low = [leaf(t) for t in model.gate], [[leaf(t) for t in b.low] for b in model.blocks]

    def norm(u, wb):
        u = u - u.mean(1, keepdim=True) if kind == "layer" else u
        u = u / torch.sqrt((u * u).mean(1, keepdim=True) + 1e-5) * wb[0]
        return u if wb[1] is None else u + wb[1]

    def proj(z, w, a, b, units):
        t = torch.einsum("tc,trc->tr", z, a[who]).view(-1, units, rank)
        return z @ w.T + torch.einsum("tur,tuor->tuo", t, b[who].view(z.shape[0], units, -1, rank)).reshape(z.shape[0], -1)

    x = table[ids.clamp(min=0).long()] * (ids >= 0)[:, None] * model.scale
    y = norm(x, pre[0])
    for i, b in enumerate(model.blocks):
        q, k, v = proj(y, b.wqkv.double().cpu(), *low[i][:2], 3).view(90, 3, width // head, head).unbind(1)
        o = []
        for s, e in zip(cuts, cuts[1:]):
            z = torch.einsum("ihd,jhd->hij", q[s:e], k[s:e]) * head ** -0.5
            z = z.masked_fill(torch.ones(e - s, e - s).triu(1).bool(), float("-inf"))
            o.append(torch.einsum("hij,jhd->ihd", z.softmax(-1), v[s:e]))
        z = proj(torch.cat(o).reshape(90, width), b.wo.double().cpu(), *low[i][2:], 1) + b.bo.double().cpu()
        x = x + gate[i] * norm(z, post[i])
        y = norm(x, pre[i + 1])
    y.backward(dh.double().cpu())
    tol = 2e-5 if dtype == torch.float32 else 3e-2
    pairs = [(h, y.detach()), (got["table"], table.grad), *zip(got["first"], pre[0])]
    for i, b in enumerate(got["blocks"]):
        pairs += [(b["gate"], gate[i]), *zip(b["post"], post[i]), *zip(b["pre"], pre[i + 1]), *zip(b["adapters"], low[i])]
    for a, w in pairs:
        if w is None:
            assert a is None
            continue
        w = w.grad if w.grad is not None else w.detach()
        assert float((a.double().cpu() - w).norm()) <= tol * float(w.norm())


def test_steps_over_the_cache(example, ctx):
    """Each block's rows, one token at a time over its 8-bit cache, are attention over what the cache reads back, to
    float: the sums' 2^-20 of the terms' norm."""
    from brosoundml_amd import tokens
    width, head, voices, n, slot, T = 128, 64, 4, 3, 40, 33
    model = example.TextModel(ctx, 50, width, head, voices, 8, causal=True, dtype=torch.float32)
    low_rank(model, 5)
    voice = torch.tensor([1, 3, 0], dtype=torch.int32, device="cuda")
    caches, filled = model.caches(n, slot), torch.zeros(n, dtype=torch.int32, device="cuda")
    seen = [[] for _ in model.blocks]
    for i, b in enumerate(model.blocks):
        b._qkv = lambda h, v, b=b, keep=seen[i], **kw: (keep.append(h), type(b)._qkv(b, h, v, **kw))[1]
    ids = torch.randint(0, 50, (T, n)).int().cuda()
    out = [model.step(t, voice, caches, filled, slot) for t in ids]
    assert (filled == T).all() and all(torch.isfinite(t).all() for t in out)
    x = tokens.embedding(ctx, model.table, ids.t().reshape(-1).contiguous(), scale=model.scale)
    off, at, full = (torch.arange(n + 1, dtype=torch.int32, device="cuda") * k for k in (T, slot, 1))
    who = voice.repeat_interleave(T)
    for i, (b, cache) in enumerate(zip(model.blocks, caches)):
        del b._qkv
        h = torch.stack(seen[i], 1).reshape(n * T, width)
        k, v = tokens.cache_read(ctx, cache, off, at, filled, rows=n * T, width=head, dtype=torch.float32)
        q, k0, v0 = b._split(b._qkv(h, who))
        # a code is off by half a step at most, and a step is a 127th of the largest
        for a, c in ((k, k0), (v, v0)):
            assert ((a - c).abs() <= c.abs().amax(-1, keepdim=True) * (0.5 / 127 * (1 + 1e-5))).all()
        o, _ = tokens.attention(ctx, q, k, v, off, causal=True)
        z = tokens.adapter_proj(ctx, o.reshape(n * T, width), b.wo, *b.low[2:], b.scale, who, b.units[1], bias=b.bo)
        x, h = tokens.residual_norm(ctx, x, z, **model._rule(i))
        want = torch.stack(seen[i + 1] if i + 1 < len(seen) else out, 1).reshape(n * T, width)
        assert float((h - want).norm()) <= 2e-5 * float(want.norm())


def test_the_example_runs(example, ctx, capsys, monkeypatch):
    monkeypatch.setattr("sys.argv", ["voiced_text.py", "--tokens", "600", "--voices", "4", "--steps", "2"])
    example.main()
    assert "8-bit caches" in capsys.readouterr().out
