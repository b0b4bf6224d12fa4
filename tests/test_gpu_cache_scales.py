"""Caches whose scales a caller made: a row that sees a token whose key or value scale is not finite becomes NaN, whatever the
products with its codes, and no other row changes a bit."""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_cache import ints  # noqa: E402


@pytest.fixture(scope="module")
def ctx():
    from brosoundml_amd import native
    return native.Context(0)


@pytest.mark.parametrize("ty", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("side", ["k_scale", "v_scale"])
@pytest.mark.parametrize("hq,hkv,cap,slopes", [(4, 4, 0.0, False), (16, 2, 0.0, False), (8, 2, 5.0, False), (4, 2, 0.0, True), (34, 1, 30.0, True)])
def test_rows_that_see_the_token_are_nan(ctx, ty, value, side, hq, hkv, cap, slopes):
    from brosoundml_amd import tokens
    g = torch.Generator().manual_seed(hq)
    n, d, lq = 300, 64, [1, 100]
    q = torch.randn(sum(lq), hq, d, generator=g)
    q[1::3] = q[1::3].abs()  # rows whose product with the token's codes is negative, and others
    codes = torch.randint(-127, 128, (2, 2 * n, hkv, d), generator=g).to(torch.int8).cuda()
    codes[0, [50, n + 250]] = -codes[0, [50, n + 250]].abs()
    codes[1, [50, n + 250], :, ::2] = 0
    scales = (torch.rand(2, hkv, 2 * n, generator=g) * 0.02).cuda()
    clean = tokens.Cache(codes[0], codes[1], scales[0], scales[1])
    bad = clean._replace(**{side: getattr(clean, side).clone()})
    getattr(bad, side)[0, [50, n + 250]] = value  # seen by the first document's row, and by the second's from its 50th on
    where = ints(np.cumsum([0, *lq])), ints([0, n, 2 * n])
    kw = dict(causal=True, cap=cap, slopes=torch.linspace(0.5, 0.001, hq).cuda() if slopes else None)
    q = q.to(ty).cuda()
    o, lse = tokens.cache_attention(ctx, q, bad, *where, **kw)
    want, lse_want = tokens.cache_attention(ctx, q, clean, *where, **kw)
    sees = torch.zeros(sum(lq), hq, dtype=torch.bool)
    rows = torch.arange(lq[1]) + n - lq[1] >= 250
    sees[0, :hq // hkv], sees[1:, :hq // hkv] = True, rows[:, None]
    sees = sees.cuda()
    assert torch.isnan(o[sees]).all() and torch.isnan(lse.t()[sees]).all()
    assert torch.equal(o[~sees], want[~sees]) and torch.equal(lse.t()[~sees], lse_want.t()[~sees])
    assert torch.isfinite(want).all()
