"""The token operators make no autograd graph, and say so where a tensor asks for one."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    from brosoundml_amd import native
    return native.Context(0)


def test_tensors_that_require_grad(ctx):
    from brosoundml_amd import tokens
    r = lambda *s: torch.randn(*s, device="cuda")  # noqa: E731
    off = torch.tensor([0, 9], dtype=torch.int32).cuda()
    q, k, v, sl = r(9, 2, 64), r(9, 2, 64), r(9, 2, 64), r(2).abs()
    o, lse = tokens.attention(ctx, q, k, v, off, slopes=sl)
    x, w, a, b, s, bias = r(9, 16), r(24, 16), r(2, 4, 16), r(2, 24, 4), r(2), r(24)
    idx, units = torch.zeros(9, dtype=torch.int32).cuda(), torch.tensor([0, 24], dtype=torch.int32).cuda()
    y, h = tokens.adapter_proj(ctx, x, w, a, b, s, idx, units, bias=bias, keep_h=True)
    calls = {
        "attention": (lambda t: tokens.attention(ctx, t["q"], t["k"], t["v"], off, slopes=t["sl"])[0], dict(q=q, k=k, v=v, sl=sl)),
        "attention_bwd": (lambda t: tokens.attention_bwd(ctx, t["q"], k, v, t["o"], t["lse"], t["do"], off, slopes=sl)[0], dict(q=q, o=o, lse=lse, do=q)),
        "adapter_proj": (lambda t: tokens.adapter_proj(ctx, t["x"], t["w"], t["a"], t["b"], t["s"], idx, units, bias=t["bias"]),
                         dict(x=x, w=w, a=a, b=b, s=s, bias=bias)),
        "adapter_proj_bwd": (lambda t: tokens.adapter_proj_bwd(ctx, x, w, t["a"], b, s, idx, units, t["h"], t["dy"])[0], dict(a=a, h=h, dy=y)),
        "dropout": (lambda t: tokens.dropout(ctx, t["x"], 0.5, 1, residual=t["r"]), dict(x=x, r=x)),
    }
    for name, (call, given) in calls.items():
        want = call(given)
        for n in given:
            t = dict(given)
            t[n] = given[n].detach().clone().requires_grad_()
            with pytest.raises(ValueError, match="requires grad"):
                call(t)
            with torch.no_grad():
                assert torch.equal(call(t), want), (name, n)
