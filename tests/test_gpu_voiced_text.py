"""The example's text block: the token operators together, trained and token by token."""
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


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_training_fits_the_voices(example, ctx, dtype):
    losses, _ = example.train(ctx, tokens_=777, width=128, head=64, voices=5, rank=8, steps=30, dtype=dtype)
    assert losses[-1] < 0.7 * losses[0] and all(v == v for v in losses)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_gradients_against_torch(example, ctx, dtype):
    """The block's gradients (no dropout) against autograd in 64 bits on the same weights. In float the kernels' sums
    are good to 2^-20 of their terms' norm; in bf16 qkv, o, the gradients between the operators and the results are
    rounded, seven roundings of 2^-9 root mean square in a row: 1 % of the norm is 1.5 times their sum's share."""
    width, head, voices, rank = 128, 32, 3, 8
    block = example.TextBlock(ctx, width, head, voices, rank, causal=True, p=0.0, dtype=dtype)
    g = torch.Generator().manual_seed(3)
    for i in (1, 3):
        block.low[i].copy_(torch.randn(block.low[i].shape, generator=g) * 0.3)
    cuts = [0, 5, 6, 90]
    off = torch.tensor(cuts, dtype=torch.int32).cuda()
    voice = torch.repeat_interleave(torch.tensor([2, 0, 1]), torch.tensor(cuts).diff()).int().cuda()
    x, dy = (torch.randn(90, width, generator=g).to(dtype).cuda() for _ in range(2))
    y, kept = block.forward(x, voice, off, 0, 0)
    dx, grads = block.backward(dy, kept)

    X = x.double().cpu().requires_grad_()
    low = [t.double().cpu().requires_grad_() for t in block.low]
    wqkv, wo, bo, who = block.wqkv.double().cpu(), block.wo.double().cpu(), block.bo.double().cpu(), voice.long().cpu()

    def proj(z, w, a, b, units):
        h = torch.einsum("tc,trc->tr", z, a[who]).view(-1, units, rank)
        return z @ w.T + torch.einsum("tur,tuor->tuo", h, b[who].view(z.shape[0], units, -1, rank)).reshape(z.shape[0], -1)

    q, k, v = proj(X, wqkv, low[0], low[1], 3).view(90, 3, width // head, head).unbind(1)
    o = []
    for a, b in zip(cuts, cuts[1:]):
        s = torch.einsum("ihd,jhd->hij", q[a:b], k[a:b]) * head ** -0.5
        s = s.masked_fill(torch.ones(b - a, b - a).triu(1).bool(), float("-inf"))
        o.append(torch.einsum("hij,jhd->ihd", s.softmax(-1), v[a:b]))
    Y = X + proj(torch.cat(o).reshape(90, width), wo, low[2], low[3], 1) + bo
    Y.backward(dy.double().cpu())
    tol = 2e-5 if dtype == torch.float32 else 1e-2
    for got, want in [(y, Y), (dx, X.grad), *zip(grads, (t.grad for t in low))]:
        assert float((got.double().cpu() - want).norm()) <= tol * float(want.norm())


def test_token_by_token_as_at_once(example, ctx):
    """A causal block's rows, one at a time over the cache, are those of one call on whole utterances, to float."""
    width, head, voices, n, slot = 128, 64, 4, 3, 40
    block = example.TextBlock(ctx, width, head, voices, 8, causal=True, p=0.0, dtype=torch.float32)
    for i in (1, 3):
        block.low[i].normal_(0.0, 0.3)
    x = torch.randn(n, 33, width, device="cuda")
    voice = torch.tensor([1, 3, 0], dtype=torch.int32, device="cuda")
    off = torch.arange(n + 1, dtype=torch.int32, device="cuda") * 33
    want, _ = block.forward(x.view(-1, width), voice.repeat_interleave(33), off, 0, 0)
    cache = torch.full((n * slot, 2, width // head, head), float("nan"), device="cuda")
    filled = torch.zeros(n, dtype=torch.int32, device="cuda")
    got = torch.stack([block.step(x[:, t], voice, cache, filled, slot) for t in range(33)], 1)
    assert float((got - want.view(n, 33, width)).norm()) <= 2e-5 * float(want.norm())
