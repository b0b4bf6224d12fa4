"""Dropout (kdec_dropout) of inputs whose rows overlap: what the call gives on a copy of them, bit for bit."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    from brosoundml_amd import native
    return native.Context(0)


@pytest.mark.parametrize("ty", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("cols", [512, 77])
def test_rows_that_overlap(ctx, ty, cols):
    from brosoundml_amd import tokens
    g = torch.Generator().manual_seed(cols)
    base = torch.randn(300 + cols, generator=g).to(ty).cuda()
    one, windows = base[:cols].expand(300, cols), base.as_strided((300, cols), (1, 1))
    for x, r in ((one, None), (one, windows), (windows, one), (windows.contiguous(), windows)):
        want = tokens.dropout(ctx, x.contiguous(), 0.3, 5, 2, residual=None if r is None else r.contiguous())
        assert torch.equal(tokens.dropout(ctx, x, 0.3, 5, 2, residual=r), want)
    # rows of an output may not overlap
    from brosoundml_amd import native
    with pytest.raises(native.KdecError, match="row stride of Y"):
        tokens.dropout(ctx, windows, 0.3, 5, 2, out=base.clone().as_strided((300, cols), (1, 1)))
