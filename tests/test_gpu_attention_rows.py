"""A row's output does not depend on its neighbours: a running softmax rescales a row when that row's own maximum moves."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    from brosoundml_amd import native
    return native.Context(0)


def inputs(heads, rows, n, d, ty):
    """Causal rows at the end of n keys whose scores rise by less than a rescaling's step from tile to tile. The last key,
    which the last row alone sees, is far above them."""
    g = torch.Generator().manual_seed(rows)
    k, v = (torch.randn(n, heads, d, generator=g) for _ in range(2))
    k[:, :, 0] = torch.linspace(0, 3, n)[:, None]
    q = 0.1 * torch.randn(rows, heads, d, generator=g)
    q[:, :, 0] = d ** 0.5
    far = k.clone()
    far[-1, :, 0] = 60.0
    return [t.to(ty).cuda() for t in (q, k, far, v)]


OFF = dict(dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("ty", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("rows", [2, 5, 16, 40, 200])
@pytest.mark.parametrize("cap", [0.0, 30.0])
def test_over_keys(ctx, ty, rows, cap):
    from brosoundml_amd import tokens
    q, k, far, v = inputs(2, rows, 400, 64, ty)
    where = torch.tensor([0, rows], **OFF), torch.tensor([0, 400], **OFF)
    a, b = (tokens.attention(ctx, q, x, v, *where, causal=True, cap=cap) for x in (k, far))
    assert torch.equal(a[0][:-1], b[0][:-1]) and torch.equal(a[1][:, :-1], b[1][:, :-1]) and not torch.equal(a[0][-1], b[0][-1])


@pytest.mark.parametrize("ty", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("rows", [2, 5, 16, 40, 200])
@pytest.mark.parametrize("cap", [0.0, 30.0])
def test_over_the_cache(ctx, ty, rows, cap):
    from brosoundml_amd import tokens
    q, k, far, v = inputs(2, rows, 400, 64, ty)
    where = torch.tensor([0, rows], **OFF), torch.tensor([0, 400], **OFF)
    out = []
    for x in (k, far):
        cache = tokens.new_cache(ctx, 400, 2, 64)
        tokens.cache_write(ctx, x, v, cache, where[1], where[1])
        out.append(tokens.cache_attention(ctx, q, cache, *where, causal=True, cap=cap))
    a, b = out
    assert torch.equal(a[0][:-1], b[0][:-1]) and torch.equal(a[1][:, :-1], b[1][:, :-1]) and not torch.equal(a[0][-1], b[0][-1])
