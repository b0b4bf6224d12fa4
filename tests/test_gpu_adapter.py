"""The projection with adapters chosen per row (kdec_adapter_fwd / _bwd) against the definition in 64 bits,
row by row.

Tolerances, per element: u the type's unit roundoff (2^-p at p bits: 2^-8 bf16, 2^-24 float) once for the
rounding of a bf16 or float result, e = 2^-24 (4 sqrt(longest sum) + 16) for the float sums, on the sums of
the products' magnitudes, and for bf16 outputs 2^-15 on the low-rank product, whose float factor enters it as
two bf16 terms (16 bits). The adapters' gradients take it as three (24 bits): e alone.
"""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
TYPES = [torch.float32, torch.bfloat16]


@pytest.fixture(scope="module")
def ctx():
    from brosoundml_amd import native
    return native.Context(0)


def mask(rows, cols, drop):
    """The dropout factors, from the operator that its own test pins."""
    from brosoundml_amd import native, tokens
    if drop is None:
        return torch.ones(rows, cols, dtype=torch.float64)
    c = native.Context(0)
    y = tokens.dropout(c, torch.ones(rows, cols, device="cuda"), *drop).cpu().double()
    thr = int(drop[0] * 65536 + 0.5)
    return (y > 0).double() * (65536 / (65536 - thr))


def oracle(x, w, bias, a, b, scale, idx, edges, dy, drop):
    x, w, a, b, dy = (t.double().cpu() for t in (x, w, a, b, dy))
    scale = scale.double().cpu()
    T, cin = x.shape
    n, out, rank = b.shape
    keep = mask(T, cin, drop)
    xd = x * keep
    r = dict(y=x @ w.T, dx=dy @ w, da=torch.zeros_like(a), db=torch.zeros_like(b))
    m = dict(y=x.abs() @ w.abs().T, dx=dy.abs() @ w.abs(), da=torch.zeros_like(a), db=torch.zeros_like(b))
    low = dict(y=torch.zeros_like(r["y"]), dx=torch.zeros_like(r["dx"]))
    if bias is not None:
        r["y"] += bias.double().cpu()
        m["y"] += bias.double().cpu().abs()
    for t in range(T):
        v = idx[t]
        if not 0 <= v < n:
            continue
        s = float(scale[v])
        for u in range(len(edges) - 1):
            e = slice(edges[u], edges[u + 1])
            c = slice(u * rank, (u + 1) * rank)
            A, B = a[v, c], b[v, e]
            h, ha = A @ xd[t], A.abs() @ xd[t].abs()
            d, da = s * B.T @ dy[t, e], abs(s) * B.abs().T @ dy[t, e].abs()
            r["y"][t, e] += s * B @ h
            m["y"][t, e] += abs(s) * B.abs() @ ha
            low["y"][t, e] = abs(s) * B.abs() @ h.abs()
            r["dx"][t] += keep[t] * (A.T @ d)
            m["dx"][t] += keep[t] * (A.abs().T @ da)
            low["dx"][t] += keep[t] * (A.abs().T @ d.abs())
            r["da"][v, c] += d[:, None] * xd[t]
            m["da"][v, c] += da[:, None] * xd[t].abs()
            r["db"][v, e] += s * dy[t, e][:, None] * h
            m["db"][v, e] += abs(s) * dy[t, e].abs()[:, None] * ha
    return r, m, low


def make(ty, T, cin, sizes, n, rank, bias=False, seed=0, odd=False):
    rng = np.random.default_rng([seed, T, cin, rank])
    out, units = sum(sizes), len(sizes)

    def t(*shape, std=1.0, wide=False):
        v = torch.from_numpy((std * rng.standard_normal(shape)).astype(np.float32)).to(ty).cuda()
        if wide and odd:  # rows that start anywhere
            s = torch.full((shape[0], shape[1] + 5), math.nan, dtype=ty, device="cuda")
            s[:, 3:3 + shape[1]] = v
            return s[:, 3:3 + shape[1]]
        return v
    return dict(x=t(T, cin, wide=True), w=t(out, cin, std=cin ** -0.5), a=t(n, units * rank, cin, std=cin ** -0.5), b=t(n, out, rank, std=0.5),
                scale=torch.from_numpy(rng.uniform(0.5, 2.0, n).astype(np.float32)).cuda(),
                edges=[0] + np.cumsum(sizes).tolist(), bias=t(out) if bias else None, dy=t(T, out, wide=True))


CASES = [
    dict(T=1, cin=64, sizes=[48], n=1, rank=8),
    dict(T=1, cin=7, sizes=[5], n=2, rank=1),
    dict(T=16, cin=256, sizes=[128, 32, 32], n=12, rank=16, order="mixed"),
    dict(T=130, cin=200, sizes=[136], n=3, rank=16, bias=True),
    dict(T=200, cin=96, sizes=[100, 29, 71], n=70, rank=4, order="mixed"),
    dict(T=97, cin=77, sizes=[45, 18], n=4, rank=5, bias=True, order="mixed", odd=True),
    dict(T=150, cin=128, sizes=[40, 0, 88], n=3, rank=33, drop=(0.25, 1 << 35 | 5, 9)),
    dict(T=70, cin=104, sizes=[64], n=2, rank=128, drop=(0.5, 3, 0), order="none"),
    dict(T=65, cin=77, sizes=[45], n=4, rank=16, drop=(0.1, 3, 1), odd=True),
    dict(T=300, cin=64, sizes=[64, 64], n=1, rank=16),
    dict(T=24, cin=128, sizes=[12, 20] * 30 + [600], n=5, rank=4, order="mixed"),  # many units, few rows
    dict(T=40, cin=130, sizes=[3000], n=2, rank=8),                                # the input grad's depth split over blocks
]


@pytest.mark.parametrize("ty", TYPES, ids=["f32", "bf16"])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(f"{k}{v}" for k, v in c.items()).replace(" ", "")[:80])
def test_against_definition(ctx, ty, case):
    from brosoundml_amd import tokens
    case = dict(case)
    drop, order = case.pop("drop", None), case.pop("order", "runs")
    d = make(ty, **case)
    T, n = case["T"], case["n"]
    rng = np.random.default_rng(T)
    idx = rng.integers(-1, n, T)
    if order == "runs":
        idx = np.sort(idx)[::-1].copy()
    elif order == "none":
        idx[:] = rng.choice([-1, n, -5, n + 3], T)
    if T > 2:
        idx[T // 2] = n + 7  # outside: none
    edges = torch.tensor(d["edges"], dtype=torch.int32).cuda()
    I = torch.tensor(idx, dtype=torch.int32).cuda()
    args = (d["x"], d["w"], d["a"], d["b"], d["scale"], I, edges)
    y, h = tokens.adapter_proj(ctx, *args, bias=d["bias"], drop=drop, keep_h=True)
    assert torch.equal(tokens.adapter_proj(ctx, *args, bias=d["bias"], drop=drop), y)
    dx, da, db = tokens.adapter_proj_bwd(ctx, *args, h, d["dy"], drop=drop)
    r, m, low = oracle(d["x"], d["w"], d["bias"], d["a"], d["b"], d["scale"], idx.tolist(), d["edges"], d["dy"], drop)
    e = 2.0 ** -24 * (4 * math.sqrt(max(T, case["cin"], sum(case["sizes"]))) + 16)
    for k, got in (("y", y), ("dx", dx), ("da", da), ("db", db)):
        tol = e * m[k] + 1e-30
        if k in low:
            tol = tol + U[ty] * r[k].abs() + (2.0 ** -15 * low[k] if ty == torch.bfloat16 else 0.0)
        off = (got.cpu().double() - r[k]).abs()
        assert torch.isfinite(off).all(), k
        assert float((off / tol).max()) <= 1.0, (k, float((off / tol).max()))
    # accumulating, and without the input grad
    base_a, base_b = torch.full_like(da, 3.0), torch.full_like(db, -2.0)
    none, a2, b2 = tokens.adapter_proj_bwd(ctx, *args, h, d["dy"], drop=drop, need_dx=False, da=base_a, db=base_b, beta=0.5)
    assert none is None and a2 is base_a and b2 is base_b
    assert torch.allclose(a2, da + 1.5, rtol=1e-6, atol=1e-6 * float(1 + da.abs().max()))
    assert torch.allclose(b2, db - 1.0, rtol=1e-6, atol=1e-6 * float(1 + db.abs().max()))
    # the same bits again
    dx3, da3, db3 = tokens.adapter_proj_bwd(ctx, *args, h, d["dy"], drop=drop)
    assert torch.equal(dx3, dx) and torch.equal(da3, da) and torch.equal(db3, db)


@pytest.mark.parametrize("ty", TYPES, ids=["f32", "bf16"])
@pytest.mark.parametrize("T", [20, 200])
def test_an_adapter_that_is_not_finite_reaches_its_rows_alone(ctx, ty, T):
    from brosoundml_amd import tokens
    d = make(ty, T, 64, [64, 32], 3, 8)
    I = (torch.arange(T) % 3).int().cuda()
    edges = torch.tensor(d["edges"], dtype=torch.int32).cuda()

    def run(a, b):
        y, h = tokens.adapter_proj(ctx, d["x"], d["w"], a, b, d["scale"], I, edges, keep_h=True)
        return (y, *tokens.adapter_proj_bwd(ctx, d["x"], d["w"], a, b, d["scale"], I, edges, h, d["dy"]))

    want = run(d["a"], d["b"])
    others = (I != 1).cpu()
    for which in "ab":
        t = {k: d[k].clone() for k in "ab"}
        t[which][1] = math.nan
        got = run(t["a"], t["b"])
        for g, w in zip(got[:2], want[:2]):
            assert torch.equal(g.cpu()[others], w.cpu()[others]) and torch.isnan(g.cpu()[~others]).any()
        for g, w in zip(got[2:], want[2:]):
            assert torch.equal(g[0], w[0]) and torch.equal(g[2], w[2])


def test_one_adapter_equals_the_style_projection(ctx):
    """With one adapter for all rows and the gate at one this is kdec_lora_proj_fwd, within both calls' float sums."""
    from brosoundml_amd import native, tokens
    d = make(torch.float32, 6, 128, [64, 96, 40], 1, 8, bias=True)
    edges = torch.tensor(d["edges"], dtype=torch.int32).cuda()
    y = tokens.adapter_proj(ctx, d["x"], d["w"], d["a"], d["b"], d["scale"], torch.zeros(6, dtype=torch.int32, device="cuda"), edges, bias=d["bias"])
    g = torch.ones(8, device="cuda")
    H, want = torch.empty(6, 24, device="cuda"), torch.empty(6, 200, device="cuda")
    P = native.ptr
    ctx.call("kdec_lora_proj_fwd", P(d["w"]), P(d["bias"]), P(d["a"]), P(d["b"]), P(g), 0, float(d["scale"][0]), P(edges), 3, 8, P(d["x"]), 128,
             P(H), P(want), 200, 6, 200, 128)
    mag = d["x"].abs() @ d["w"].abs().T + d["bias"].abs() + float(d["scale"][0]) * 8 * 8
    assert ((y - want).abs() <= 2 * 2.0 ** -24 * (4 * math.sqrt(128) + 16) * mag).all()


def test_gradients_against_differences(ctx):
    """The loss sum(y * dy) is linear in x and in each of a and b alone, so a difference over a step of one has no
    remainder: only the two forwards' float sums, 2^-24 of the loss's terms' magnitude times their root count."""
    from brosoundml_amd import tokens
    d = make(torch.float32, 50, 64, [32, 32], 3, 4)
    I = (torch.arange(50) % 4 - 1).int().cuda()
    edges = torch.tensor(d["edges"], dtype=torch.int32).cuda()
    drop = (0.2, 77, 0)
    _, h = tokens.adapter_proj(ctx, d["x"], d["w"], d["a"], d["b"], d["scale"], I, edges, drop=drop, keep_h=True)
    grads = dict(zip("xab", tokens.adapter_proj_bwd(ctx, d["x"], d["w"], d["a"], d["b"], d["scale"], I, edges, h, d["dy"], drop=drop)))
    rng = np.random.default_rng(3)
    for k in "xab":
        dr = torch.from_numpy(rng.standard_normal(tuple(d[k].shape)).astype(np.float32)).cuda()
        f = []
        for s in (1, -1):
            t = dict(d)
            t[k] = d[k] + s * dr
            y = tokens.adapter_proj(ctx, t["x"], t["w"], t["a"], t["b"], t["scale"], I, edges, drop=drop)
            f.append((y.double() * d["dy"].double()).sum())
        num, ana = float(f[0] - f[1]) / 2, float((grads[k].double() * dr.double()).sum())
        assert abs(num - ana) <= 1e-4 * float(grads[k].double().norm() * 2), (k, num, ana)


def test_refusals(ctx):
    from brosoundml_amd import native, tokens
    d = make(torch.float32, 4, 16, [8, 8], 2, 4)
    edges = torch.tensor([0, 8, 16], dtype=torch.int32).cuda()
    I = torch.zeros(4, dtype=torch.int32, device="cuda")
    args = [d["x"], d["w"], d["a"], d["b"], d["scale"], I, edges]

    def wrong(i, v):
        a = list(args)
        a[i] = v
        return a
    for i, v in ((0, d["x"].bfloat16()), (1, d["w"][:, :8]), (2, d["a"][:, :4]), (3, d["b"][:1]), (4, d["scale"].double()), (5, I[:3]), (5, I.long()),
                 (6, edges[:1]), (0, d["x"].t())):
        with pytest.raises(ValueError):
            tokens.adapter_proj(ctx, *wrong(i, v))
    with pytest.raises(native.KdecError, match="p must"):
        tokens.adapter_proj(ctx, *args, drop=(1.0, 0, 0))
    wide = make(torch.float32, 4, 16, [16], 2, 129)
    with pytest.raises(native.KdecError, match="rank"):
        tokens.adapter_proj(ctx, wide["x"], wide["w"], wide["a"], wide["b"], wide["scale"], I, edges[::2].contiguous())
    y, h = tokens.adapter_proj(ctx, *args, keep_h=True)
    with pytest.raises(ValueError):
        tokens.adapter_proj_bwd(ctx, *args, h, d["dy"][:, :8])
    with pytest.raises(ValueError):
        tokens.adapter_proj_bwd(ctx, *args, h, d["dy"], beta=1.0)
    # no rows: nothing forward, zeros for the adapters
    e = [d["x"][:0], d["w"], d["a"], d["b"], d["scale"], I[:0], edges]
    y, h = tokens.adapter_proj(ctx, *e, keep_h=True)
    dx, da, db = tokens.adapter_proj_bwd(ctx, *e, h, d["dy"][:0])
    assert y.shape == (0, 16) and dx.shape == (0, 16) and not da.any() and not db.any()
    # no adapters at all: the plain projection
    y = tokens.adapter_proj(ctx, d["x"], d["w"], d["a"][:0], d["b"][:0], d["scale"][:0], I, edges)
    assert torch.allclose(y, d["x"] @ d["w"].t(), atol=1e-5)


@pytest.mark.parametrize("drop", [None, (0.3, 9, 2)], ids=["", "drop"])
def test_many_rows_equal_few_rows(ctx, drop):
    """A call of enough rows for the large product tiles gives each row the bits that a call of fewer rows gives it
    (the same products in the same order), at sizes that end inside a tile in every direction."""
    from brosoundml_amd import tokens
    T, cin, sizes, n, rank = 14999, 200, [500, 24, 404], 5, 8
    d = make(torch.bfloat16, T, cin, sizes, n, rank, bias=True)
    wide = make(torch.bfloat16, T, 928, [200], n, rank)  # the input grad's large tiles: 928 features
    for d, out in ((d, 928), (wide, 200)):
        I = torch.from_numpy(np.random.default_rng(1).integers(-1, n, T).astype(np.int32)).cuda()
        edges = torch.tensor(d["edges"], dtype=torch.int32).cuda()
        y, h = tokens.adapter_proj(ctx, d["x"], d["w"], d["a"], d["b"], d["scale"], I, edges, bias=d["bias"], keep_h=True)
        dx, _, _ = tokens.adapter_proj_bwd(ctx, d["x"], d["w"], d["a"], d["b"], d["scale"], I, edges, h, d["dy"])
        part = slice(0, 700)
        args = (d["x"][part], d["w"], d["a"], d["b"], d["scale"], I[part].contiguous(), edges)
        y2, h2 = tokens.adapter_proj(ctx, *args, bias=d["bias"], keep_h=True)
        assert torch.equal(h[part], h2) and torch.equal(y[part], y2)
        dx2, _, _ = tokens.adapter_proj_bwd(ctx, *args, h2, d["dy"][part])
        if out < 256:  # (a shorter call may split a longer depth)
            assert torch.equal(dx[part], dx2)
        if drop:
            y, h = tokens.adapter_proj(ctx, d["x"], d["w"], d["a"], d["b"], d["scale"], I, edges, drop=drop, keep_h=True)
            dx, _, _ = tokens.adapter_proj_bwd(ctx, d["x"], d["w"], d["a"], d["b"], d["scale"], I, edges, h, d["dy"], drop=drop)
            y2, h2 = tokens.adapter_proj(ctx, *args, drop=drop, keep_h=True)  # the mask goes by row: the first rows' is theirs
            dx2, _, _ = tokens.adapter_proj_bwd(ctx, *args, h2, d["dy"][part], drop=drop)
            assert torch.equal(y[part], y2) and (out >= 256 or torch.equal(dx[part], dx2))


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("T", [700, 14999])
def test_adapter_not_finite_among_many_rows(ctx, T, bad):
    """Values of one adapter that are not finite reach its rows' outputs that they enter, and no bit of any other's."""
    from brosoundml_amd import tokens
    cin, sizes, n, rank = 928, [500, 24, 404], 5, 8
    d = make(torch.bfloat16, T, cin, sizes, n, rank, bias=True)
    I = torch.from_numpy(np.random.default_rng(2).integers(-1, n, T).astype(np.int32)).cuda()
    edges = torch.tensor(d["edges"], dtype=torch.int32).cuda()

    def run(a, b):
        args = (ctx, d["x"], d["w"], a, b, d["scale"], I, edges)
        y, h = tokens.adapter_proj(*args, bias=d["bias"], keep_h=True)
        return y, h, tokens.adapter_proj_bwd(*args, h, d["dy"])[0]

    y0, _, dx0 = run(d["a"], d["b"])
    a, b = d["a"].clone(), d["b"].clone()
    b[3, 510, 2] = bad
    a[3, 17, 300] = bad
    y, h, dx = run(a, b)
    mine = I == 3
    assert torch.equal(y[~mine], y0[~mine]) and torch.equal(dx[~mine], dx0[~mine])
    assert not torch.isfinite(y[mine][:, 510].float()).any()       # (its H is of order one, its x too)
    assert torch.equal(y[mine][:, :500], y0[mine][:, :500])
    assert not torch.isfinite(dx[mine][:, 300].float()).any()
