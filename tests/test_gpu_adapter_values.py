"""The adapter projection (kdec_adapter_fwd / _bwd) with infinite values: an infinity in one factor of a product comes
out as the definition in 64 bits has it, infinite with its sign or NaN, and what it does not enter stays as near the
definition as it is without."""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_adapter import TYPES, ctx, make  # noqa: E402, F401


@pytest.mark.parametrize("ty", TYPES, ids=["f32", "bf16"])
@pytest.mark.parametrize("T", [20, 50, 200, 700, 7100])
@pytest.mark.parametrize("which", ["a", "b", "x", "dy"])
@pytest.mark.parametrize("value", [math.inf, -math.inf])
def test_infinities_stay_infinities(ctx, ty, T, which, value):  # noqa: F811
    from brosoundml_amd import tokens
    cin, sizes, n, rank = 136, [100, 24, 76], 3, 8
    d = make(ty, T, cin, sizes, n, rank)
    idx = np.random.default_rng(T).integers(-1, n, T)
    idx[5] = 1
    at = dict(a=(1, 11, 17), b=(1, 110, 2), x=(5, 17), dy=(5, 110))[which]
    d[which][at] = value
    I = torch.from_numpy(idx.astype(np.int32)).cuda()
    edges = torch.tensor(d["edges"], dtype=torch.int32).cuda()
    args = (ctx, d["x"], d["w"], d["a"], d["b"], d["scale"], I, edges)
    y, h = tokens.adapter_proj(*args, keep_h=True)
    dx, da, db = tokens.adapter_proj_bwd(*args, h, d["dy"])
    # the definition by adapter, in 64 bits: nothing of another adapter's rows enters a product
    x, w, a, b, dy = (d[k].double() for k in ("x", "w", "a", "b", "dy"))
    want = dict(y=x @ w.T, dx=dy @ w, h=torch.zeros_like(h, dtype=torch.float64), da=torch.zeros_like(a), db=torch.zeros_like(b))
    for v in range(n):
        r = torch.from_numpy(np.flatnonzero(idx == v)).cuda()
        if len(r) == 0:
            continue
        s = float(d["scale"][v])
        want["h"][r] = s * (x[r] @ a[v].T)
        for u in range(3):
            c, e = slice(u * rank, (u + 1) * rank), slice(d["edges"][u], d["edges"][u + 1])
            want["y"][r, e] += want["h"][r, c] @ b[v, e].T
            g = s * (dy[r, e] @ b[v, e])
            want["dx"][r] += g @ a[v, c]
            want["da"][v, c] = g.T @ x[r]
            want["db"][v, e] = dy[r, e].T @ want["h"][r, c]
    seen = 0
    for k, got in dict(y=y, h=h, dx=dx, da=da, db=db).items():
        g, t = got.double(), want[k]
        wild = ~torch.isfinite(t)
        seen += int(wild.sum())
        assert torch.equal(~torch.isfinite(g), wild), k
        assert torch.equal(torch.nan_to_num(g[wild], 0.0, 1.0, -1.0), torch.nan_to_num(t[wild], 0.0, 1.0, -1.0)), k
        off, size = (g - t)[~wild].norm(), t[~wild].norm()
        # one rounding of the result (root mean square 2^-9.8 and less for bf16), or float sums
        assert float(off) <= (2.0 ** -8 if ty == torch.bfloat16 and k in ("y", "dx") else 2.0 ** -18) * float(size), k
    assert seen
