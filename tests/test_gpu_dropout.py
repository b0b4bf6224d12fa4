"""Dropout (kdec_dropout) against the generator restated in numpy: the mask bit for bit, the values to their
one rounding."""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    from brosoundml_amd import native
    return native.Context(0)


def philox(counter, key):
    """Philox4x32-10 on python integers."""
    c, k = list(counter), list(key)
    for _ in range(10):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [(b >> 32) ^ c[1] ^ k[0], b & 0xFFFFFFFF, (a >> 32) ^ c[3] ^ k[1], a & 0xFFFFFFFF]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return c


def halves(rows, cols, seed, offset):
    out = np.zeros((rows, cols), np.int64)
    for r in range(rows):
        for c in range(0, cols, 8):
            w = philox([c >> 3, r, offset & 0xFFFFFFFF, offset >> 32], [seed & 0xFFFFFFFF, seed >> 32])
            h = [x >> s & 0xFFFF for x in w for s in (0, 16)]
            out[r, c:c + 8] = h[:min(8, cols - c)]
    return out


def test_generator_known_answers():
    """The generator's published known-answer vectors (the zero and the all-ones counter and key)."""
    assert philox([0] * 4, [0] * 2) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    assert philox([0xFFFFFFFF] * 4, [0xFFFFFFFF] * 2) == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]


@pytest.mark.parametrize("ty", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("rows,cols,p,res,odd", [(1, 1, 0.5, False, False), (3, 8, 0.1, True, False), (17, 64, 0.5, True, False),
                                                 (5, 77, 0.3, True, False), (9, 40, 0.9999, False, True), (4, 24, 0.0, True, True)])
def test_against_definition(ctx, ty, rows, cols, p, res, odd):
    from brosoundml_amd import tokens
    rng = np.random.default_rng([rows, cols])
    seed, offset = 0x123456789ABCDEF, 5 << 33 | 7
    mk = lambda: torch.from_numpy(rng.standard_normal((rows, cols + 3)).astype(np.float32)).to(ty).cuda()[:, 1:1 + cols] if odd else \
        torch.from_numpy(rng.standard_normal((rows, cols)).astype(np.float32)).to(ty).cuda()  # noqa: E731
    x, r = mk(), mk() if res else None
    y = tokens.dropout(ctx, x, p, seed, offset, residual=r)
    thr = int(p * 65536 + 0.5)
    want = np.where(halves(rows, cols, seed, offset) >= thr, 65536 / (65536 - thr), 0.0) * x.double().cpu().numpy()
    if res:
        want = want + r.double().cpu().numpy()
    u = 2.0 ** -24 if ty == torch.float32 else 2.0 ** -8
    off = np.abs(y.double().cpu().numpy() - want)
    # one product, one sum (both in float) and the output's rounding
    scale = np.abs(want) + 65536 / (65536 - thr) * np.abs(x.double().cpu().numpy())
    assert (off <= u * np.abs(want) + 3 * 2.0 ** -24 * scale).all()
    if p == 0.0 and not res:
        assert torch.equal(y, x)


def test_backward_is_the_same_mask_and_in_place(ctx):
    from brosoundml_amd import tokens
    x = torch.ones(300, 512, device="cuda")
    y = tokens.dropout(ctx, x, 0.25, 11, 3)
    g = tokens.dropout(ctx, torch.full_like(x, 2.0), 0.25, 11, 3)
    assert torch.equal(g, 2 * y)
    z = x.clone()
    assert tokens.dropout(ctx, z, 0.25, 11, 3, out=z) is z and torch.equal(z, y)
    # the share kept is 3/4 within five standard deviations, and other seeds, offsets and rows differ
    n = x.numel()
    assert abs(float((y > 0).float().mean()) - 0.75) < 5 * math.sqrt(0.1875 / n)
    for s, o in ((12, 3), (11, 4), (11 + (1 << 40), 3), (11, 3 + (1 << 40))):
        assert float((tokens.dropout(ctx, x, 0.25, s, o) != y).float().mean()) > 0.3
    # the mask does not depend on the layout or the type
    wide = torch.ones(300, 600, device="cuda")[:, 5:517]
    assert torch.equal(tokens.dropout(ctx, wide, 0.25, 11, 3), y)
    assert torch.equal(tokens.dropout(ctx, x.bfloat16(), 0.25, 11, 3) > 0, y > 0)


def test_special_values_and_refusals(ctx):
    from brosoundml_amd import native, tokens
    x = torch.full((64, 64), math.nan, device="cuda")
    y = tokens.dropout(ctx, x, 0.5, 1)
    kept = tokens.dropout(ctx, torch.ones_like(x), 0.5, 1) > 0
    assert torch.equal(torch.isnan(y), kept) and not y[~kept].any()  # a dropped value is zero whatever it was
    for p in (1.0, -0.1, math.nan, 0.999999):
        with pytest.raises(native.KdecError, match="p must"):
            tokens.dropout(ctx, x, p, 1)
    with pytest.raises(ValueError):
        tokens.dropout(ctx, x, 0.5, 1, residual=x[:3])
    with pytest.raises(ValueError):
        tokens.dropout(ctx, x.half(), 0.5, 1)
    with pytest.raises(ValueError):
        tokens.dropout(ctx, x.t()[:, ::2], 0.5, 1)
    assert tokens.dropout(ctx, x[:0], 0.5, 1).shape == (0, 64)
