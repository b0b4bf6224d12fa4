"""Attention's outputs (kdec_attn_fwd / kdec_attn_bwd): tensors whose rows repeat are refused, layouts that lie apart taken."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    from brosoundml_amd import native
    return native.Context(0)


def test_outputs_that_overlap(ctx):
    from brosoundml_amd import native, tokens
    q, k, v, do = (torch.randn(9, h, 64, device="cuda") for h in (4, 2, 2, 4))
    off = torch.tensor([0, 9], dtype=torch.int32).cuda()
    o, lse = tokens.attention(ctx, q, k, v, off)
    grads = dict(zip(("dq", "dk", "dv"), tokens.attention_bwd(ctx, q, k, v, o, lse, do, off)))
    repeated = {"rows": lambda t: t[:1].expand(t.shape), "heads": lambda t: t[:, :1].expand(t.shape),
                "steps": lambda t: t.new_empty(9 * 64 * 8).as_strided(t.shape, (64 * 4, 32, 1))}
    for make in repeated.values():
        with pytest.raises(native.KdecError, match="overlap"):
            tokens.attention(ctx, q, k, v, off, out=make(torch.empty_like(o)))
        for n, g in grads.items():
            with pytest.raises(native.KdecError, match="overlap"):
                tokens.attention_bwd(ctx, q, k, v, o, lse, do, off, **{n: make(torch.empty_like(g))})
    heads_first = lambda t: torch.empty(t.shape[1], t.shape[0], t.shape[2], device="cuda").transpose(0, 1)  # noqa: E731
    assert torch.equal(tokens.attention(ctx, q, k, v, off, out=heads_first(o))[0], o)
    got = tokens.attention_bwd(ctx, q, k, v, o, lse, do, off, **{n: heads_first(g) for n, g in grads.items()})
    for a, b in zip(got, grads.values()):
        assert torch.equal(a, b)
    # one row or one head has nothing to overlap, whatever its stride says
    o1, _ = tokens.attention(ctx, q[:1], k, v, off[:0].new_tensor([0, 1]), off)
    assert torch.equal(tokens.attention(ctx, q[:1], k, v, off.new_tensor([0, 1]), off, out=torch.empty_like(o1).as_strided(o1.shape, (0, 64, 1)))[0], o1)
