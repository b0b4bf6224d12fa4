"""The norms around a block with gate and residual (kdec_resnorm_fwd / kdec_resnorm_bwd) against their definition in
64 bits.

Tolerances are a running error analysis of the kernels' formulas: every quantity is carried with a bound of its
error, e = 2^-24 of the result for each float operation, a sum of C values with 32 additions in a row at most (16 in
a lane, 6 across lanes, 8 waves), a sum over T rows with T additions; an output adds its type's rounding u. The
bounds are of first order, so 1.01 of them.
"""
import itertools

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
E = 2.0 ** -24


@pytest.fixture(scope="module")
def ctx():
    from brosoundml_amd import native
    return native.Context(0)


class Q:
    """A value in 64 bits and a bound of the float kernel's error in it."""

    def __init__(self, v, err=None):
        self.v = v.double() if isinstance(v, torch.Tensor) else torch.tensor(float(v), dtype=torch.float64)
        self.err = torch.zeros_like(self.v) if err is None else err

    def made(self, v, err):
        return Q(v, err + E * v.abs())

    def __add__(self, o):
        return self.made(self.v + o.v, self.err + o.err)

    def __sub__(self, o):
        return self.made(self.v - o.v, self.err + o.err)

    def __mul__(self, o):
        return self.made(self.v * o.v, self.err * o.v.abs() + o.err * self.v.abs())

    def row_mean(self):
        n = self.v.shape[1]
        return self.made(self.v.mean(1, keepdim=True), (self.err.sum(1, keepdim=True) + 32 * E * self.v.abs().sum(1, keepdim=True)) / n)

    def columns(self):
        return self.made(self.v.sum(0), self.err.sum(0) + self.v.shape[0] * E * self.v.abs().sum(0))

    def rsqrt(self, eps):
        v = 1 / torch.sqrt(self.v + eps)
        return self.made(v, v * (self.err / (self.v + eps) / 2 + 3 * E))


def normed(u, layer, eps):
    if layer:
        u = u - u.row_mean()
    rs = (u * u).row_mean().rsqrt(eps)
    return u * rs, rs


def back(e, hat, rs, layer):
    d = e - hat * (e * hat).row_mean()
    return rs * (d - e.row_mean() if layer else d)


def oracle(x, z, gate, post, pre, layer, eps, scale, x_scale, dr, dy):
    q = lambda t: None if t is None else Q(t.cpu())  # noqa: E731
    x, z, gate, dr, dy = map(q, (x, z, gate, dr, dy))
    one, zero = Q(1.0), Q(0.0)
    (w1, b1), (w2, b2) = ((one, zero) if p is None else (q(p[0]) or one, q(p[1]) or zero) for p in (post, pre))
    a, b, g = Q(np.float32(scale)), Q(np.float32(x_scale)), gate or one
    out = {}
    if z is not None:
        u = z
        if post is not None:
            zh, s1 = normed(z, layer, eps)
            u = zh * w1 + b1
        r = a * g * u + b * x
        out["r"] = r
    else:
        r = x
    if pre is not None:
        rh, s2 = normed(r, layer, eps)
        out["y"] = rh * w2 + b2
    if dr is None and dy is None:
        return out
    top = dr or zero
    if pre is not None:
        top = top + back(dy * w2, rh, s2, layer)
        out["dw2"], out["db2"] = (dy * rh).columns(), dy.columns()
    out["dx"] = b * top if z is not None else top
    if z is not None:
        du = a * g * top
        dg = a * u * top
        out["dgate"] = dg.columns() if gate is not None and gate.v.dim() == 1 else dg
        out["dz"] = du
        if post is not None:
            out["dw1"], out["db1"] = (du * zh).columns(), du.columns()
            out["dz"] = back(du * w1, zh, s1, layer)
    return out


def near(name, got, want):
    u = U[got.dtype] if name not in ("dw1", "db1", "dw2", "db2") else E
    off, tol = (got.double().cpu() - want.v).abs(), 1.01 * (want.err + u * want.v.abs()) + 1e-300
    assert (off <= tol).all(), (name, float((off / tol).max()))


def tensor(rng, ty, shape, layout="packed", mid=0.0, std=1.0):
    a = torch.from_numpy((mid + std * rng.standard_normal(shape)).astype(np.float32)).to(ty)
    if layout == "odd" and len(shape) == 2:
        s = torch.zeros(shape[0], shape[1] + 3, dtype=ty)
        s[:, 1:1 + shape[1]] = a
        return s.cuda()[:, 1:1 + shape[1]]
    if layout == "wide" and len(shape) == 2:  # a part of wider rows
        s = torch.zeros(shape[0], 2, shape[1], dtype=ty)
        s[:, 1] = a
        return s.cuda()[:, 1]
    return a.cuda()


def compare(ctx, ty, t, c, *, layer=False, post="wb", pre="wb", gate="none", block=True, dr=True, scale=0.75, x_scale=1.25, eps=1e-5,
            layout="packed", seed=0, loud=1.0):
    from brosoundml_amd import tokens
    rng = np.random.default_rng([seed, t, c, layer])
    x, z = tensor(rng, ty, (t, c), layout, 0.3, loud), tensor(rng, ty, (t, c), layout) if block else None
    vec = lambda kind: None if kind == "none" else tuple(tensor(rng, ty, (c,), mid=m, std=0.3) if k in kind else None for k, m in (("w", 1.0), ("b", 0.0)))  # noqa: E731
    post, pre = vec(post), vec(pre)
    if not block:
        post, gate, x_scale = None, "none", 1.0
    g = {"none": None, "column": tensor(rng, ty, (c,)), "row": tensor(rng, ty, (t, c), layout)}[gate]
    rule = dict(gate=g, post=post, pre=pre, kind="layer" if layer else "rms", eps=eps, scale=scale, x_scale=x_scale)
    dr = tensor(rng, ty, (t, c), layout) if dr else None
    dy = tensor(rng, ty, (t, c), layout) if pre is not None else None
    want = oracle(x, z, g, post, pre, layer, np.float64(np.float32(eps)), scale, x_scale, dr, dy)
    r, y = tokens.residual_norm(ctx, x, z, **rule)
    r2, y2, stats = tokens.residual_norm(ctx, x, z, keep=True, **rule)
    assert torch.equal(r, r2) and (y is None or torch.equal(y, y2))
    got = {"y": y} if y is not None else {}
    if block:
        got["r"] = r
    else:
        assert r is x
    dx, dz, dgate, dpost, dpre = grads = tokens.residual_norm_bwd(ctx, x, z, dr, dy, stats, **rule)
    got["dx"] = dx
    if block:
        got["dz"] = dz
    if g is not None:
        got["dgate"] = dgate
    for name, w, d in (("1", post, dpost), ("2", pre, dpre)):
        assert (d is None) == (w is None)
        for k, p, v in zip("wb", w or (), d or ()):
            assert (v is None) == (p is None)
            if v is not None:
                assert v.dtype == torch.float32
                got[f"d{k}{name}"] = v
    for name, v in got.items():
        near(name, v, want[name])
    again = tokens.residual_norm_bwd(ctx, x, z, dr, dy, stats, **rule)
    flat = lambda o: [v for v in (*o[:3], *(o[3] or ()), *(o[4] or ())) if v is not None]  # noqa: E731
    assert all(torch.equal(a, b) for a, b in zip(flat(grads), flat(again)))  # the same bits every time


TYPES = pytest.mark.parametrize("ty", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])


@TYPES
@pytest.mark.parametrize("layer", [False, True], ids=["rms", "layer"])
@pytest.mark.parametrize("t,c", [(1, 1), (1, 8), (3, 77), (1, 512), (5, 513), (7, 1024), (16, 1021), (2, 1025), (9, 2048), (3, 2049), (4, 4096),
                                 (3, 4100), (2, 8192), (700, 64), (1100, 520)])
def test_sizes(ctx, ty, layer, t, c):
    compare(ctx, ty, t, c, layer=layer, gate="column")


@TYPES
@pytest.mark.parametrize("layer,post,pre,gate", [k for k in itertools.product([False, True], ["none", "w", "wb"], ["none", "w", "wb", ""], ["none", "column", "row"])])
def test_parts(ctx, ty, layer, post, pre, gate):
    compare(ctx, ty, 13, 264, layer=layer, post=post, pre=pre, gate=gate, dr=pre in ("none", "w"))


@TYPES
@pytest.mark.parametrize("layout", ["odd", "wide"])
@pytest.mark.parametrize("t,c", [(6, 96), (11, 700), (5, 1024), (4, 2600)])
def test_layouts(ctx, ty, layout, t, c):
    compare(ctx, ty, t, c, layer=True, gate="row", layout=layout)


@TYPES
@pytest.mark.parametrize("layer", [False, True], ids=["rms", "layer"])
def test_norm_alone(ctx, ty, layer):
    for dr in (False, True):
        compare(ctx, ty, 21, 768, layer=layer, block=False, dr=dr)


def test_values_far_from_one(ctx):
    for loud, eps in ((1e-6, 1e-12), (1e6, 1e-5), (1e12, 1e-5)):
        compare(ctx, torch.float32, 5, 640, layer=True, loud=loud, eps=eps)
    # rows of zeros: the variance is eps alone
    from brosoundml_amd import tokens
    x = torch.zeros(4, 100, device="cuda")
    r, y, st = tokens.residual_norm(ctx, x, x, post=torch.ones(100, device="cuda"), pre=torch.ones(100, device="cuda"), keep=True)
    dx, dz, _, _, _ = tokens.residual_norm_bwd(ctx, x, x, None, torch.ones_like(x), st, post=torch.ones(100, device="cuda"), pre=torch.ones(100, device="cuda"))
    assert not r.any() and not y.any() and torch.isfinite(dx).all() and torch.isfinite(dz).all()


def test_rows_keep_to_themselves(ctx):
    """A row that is not finite changes no other row's outputs or gradients; the columns' sums take it."""
    from brosoundml_amd import tokens
    g = torch.Generator().manual_seed(3)
    x, z, dy = (torch.randn(50, 300, generator=g).cuda() for _ in range(3))
    w = torch.ones(300, device="cuda")
    rule = dict(post=w, pre=(w, None), gate=torch.rand(50, 300, generator=g).cuda())

    def run(x, z):
        r, y, st = tokens.residual_norm(ctx, x, z, keep=True, **rule)
        return (r, y, *tokens.residual_norm_bwd(ctx, x, z, dy, dy, st, **rule)[:3])

    clean = run(x, z)
    x2, z2 = x.clone(), z.clone()
    x2[7, 5], z2[31, 299] = float("nan"), float("inf")
    rest = [i for i in range(50) if i not in (7, 31)]
    for a, b in zip(clean, run(x2, z2)):
        assert torch.equal(a[rest], b[rest]) and torch.isnan(b[31]).any()


def test_outputs_given_and_in_place(ctx):
    from brosoundml_amd import tokens
    g = torch.Generator().manual_seed(4)
    x, z = (torch.randn(40, 520, generator=g).bfloat16().cuda() for _ in range(2))
    w = torch.ones(520, device="cuda").bfloat16()
    r, y = tokens.residual_norm(ctx, x, z, post=w, pre=w)
    both = torch.full((40, 2, 521), 3.0, device="cuda").bfloat16()
    tokens.residual_norm(ctx, x, z, post=w, pre=w, out=(both[:, 0, :520], both[:, 1, :520]))
    assert torch.equal(both[:, 0, :520], r) and torch.equal(both[:, 1, :520], y) and (both[:, :, 520] == 3).all()
    x2, z2 = x.clone(), z.clone()
    got = tokens.residual_norm(ctx, x2, z2, post=w, pre=w, out=(x2, z2))
    assert got[0] is x2 and torch.equal(x2, r) and torch.equal(z2, y)


def test_one_gate_row_of_any_stride(ctx):
    """A (1, C) gate is a row's own, of the tensors' type, whatever stride its single row has."""
    from brosoundml_amd import tokens
    x, z = torch.randn(1, 64, device="cuda").bfloat16(), torch.randn(1, 64, device="cuda").bfloat16()
    gate = torch.randn(64, device="cuda").bfloat16()
    w = torch.ones(64, device="cuda").bfloat16()
    want = None
    for v in (gate[None].clone(), gate.expand(1, 64), gate.as_strided((1, 64), (0, 1))):
        r, y, st = tokens.residual_norm(ctx, x, z, gate=v, pre=w, keep=True)
        d = tokens.residual_norm_bwd(ctx, x, z, x, z, st, gate=v, pre=w)[2]
        assert d.dtype == torch.bfloat16 and d.shape == (1, 64)
        want = d if want is None else want
        assert torch.equal(d, want)


def test_rows_past_32_bits(ctx):
    from brosoundml_amd import tokens
    x = torch.empty(3, (1 << 30) + 16, dtype=torch.bfloat16, device="cuda")[:, :256]
    g = torch.Generator().manual_seed(6)
    x.copy_(torch.randn(3, 256, generator=g))
    z, w = torch.randn(3, 256, generator=g).bfloat16().cuda(), torch.ones(256, device="cuda").bfloat16()
    near_x = x.clone()
    for a, b in zip(tokens.residual_norm(ctx, x, z, post=w, pre=w), tokens.residual_norm(ctx, near_x, z, post=w, pre=w)):
        assert torch.equal(a, b)
    tokens.residual_norm(ctx, near_x, z, post=w, out=(x, None))
    assert torch.equal(x, tokens.residual_norm(ctx, near_x, z, post=w)[0])


def test_gradient_against_differences(ctx):
    """Float gradients against central differences of the float forward's sums in 64 bits.

    The loss <r, dr> + <y, dy> along a direction d with step h: the third derivative makes h^2 times order one per
    direction's length cubed, the outputs' roundings 2^-24 of about 2000 terms over h; h = 2^-6 holds both below
    2^-9 of the sum of magnitudes."""
    from brosoundml_amd import tokens
    g = torch.Generator().manual_seed(9)
    t, c = 6, 40
    new = lambda *s: torch.randn(*s, generator=g).cuda()  # noqa: E731
    x, z, dr, dy = (new(t, c) for _ in range(4))
    p = dict(gate=new(c), post=(1 + 0.2 * new(c), new(c)), pre=(1 + 0.2 * new(c), new(c)), kind="layer", scale=0.7, x_scale=1.3)
    st = tokens.residual_norm(ctx, x, z, keep=True, **p)[2]
    dx, dz, dgate, dpost, dpre = tokens.residual_norm_bwd(ctx, x, z, dr, dy, st, **p)

    def loss(x, z, p):
        r, y = tokens.residual_norm(ctx, x, z, **p)
        return float((r.double() * dr.double()).sum() + (y.double() * dy.double()).sum())

    h = 2.0 ** -6
    for what, grad in (("x", dx), ("z", dz), ("gate", dgate), ("w1", dpost[0]), ("b1", dpost[1]), ("w2", dpre[0]), ("b2", dpre[1])):
        d = new(*grad.shape)
        def at(s):  # noqa: E306
            q = dict(p)
            if what == "gate":
                q["gate"] = p["gate"] + s * d
            elif what in ("w1", "b1", "w2", "b2"):
                k = "post" if what[1] == "1" else "pre"
                q[k] = tuple(v + s * d if n == what[0] else v for n, v in zip("wb", p[k]))
            return loss(x + s * d if what == "x" else x, z + s * d if what == "z" else z, q)
        slope, want = (at(h) - at(-h)) / (2 * h), float((d.double() * grad.double()).sum())
        size = float((d.double() * grad.double()).abs().sum()) + float(dr.abs().sum() + dy.abs().sum())
        assert abs(slope - want) <= 2.0 ** -9 * size, (what, slope, want)


def test_refusals(ctx):
    from brosoundml_amd import native, tokens
    x, w = torch.ones(4, 32, device="cuda"), torch.ones(32, device="cuda")
    st = torch.ones(4, 4, device="cuda")
    fine = dict(post=w, pre=w)
    for call in (lambda: tokens.residual_norm(ctx, x, x[:3], **fine), lambda: tokens.residual_norm(ctx, x, x.bfloat16(), **fine),
                 lambda: tokens.residual_norm(ctx, x.half(), None, pre=w.half()), lambda: tokens.residual_norm(ctx, x, None, post=w),
                 lambda: tokens.residual_norm(ctx, x, None), lambda: tokens.residual_norm(ctx, x, None, pre=w, x_scale=2.0),
                 lambda: tokens.residual_norm(ctx, x, x, gate=torch.ones(1, device="cuda"), pre=w),
                 lambda: tokens.residual_norm(ctx, x, x, gate=w.expand(4, 32), pre=w), lambda: tokens.residual_norm(ctx, x, x, pre=w[:31]),
                 lambda: tokens.residual_norm(ctx, x, x, kind="batch", **fine), lambda: tokens.residual_norm(ctx, x.t(), x.t(), pre=w[:4]),
                 lambda: tokens.residual_norm(ctx, x, x, pre=(w, w, w)), lambda: tokens.residual_norm(ctx, x, x, out=(x[:2], None)),
                 lambda: tokens.residual_norm(ctx, x, x.clone().requires_grad_(), **fine),
                 lambda: tokens.residual_norm_bwd(ctx, x, x, x, None, st, **fine), lambda: tokens.residual_norm_bwd(ctx, x, x, x, x, st[:2], **fine)):
        with pytest.raises(ValueError, match="brosoundml"):
            call()
    for eps in (0.0, -1.0, float("nan"), float("inf")):
        with pytest.raises(native.KdecError, match="eps"):
            tokens.residual_norm(ctx, x, x, eps=eps, **fine)
    big = torch.ones(1, 8193, device="cuda")
    with pytest.raises(native.KdecError, match="columns"):
        tokens.residual_norm(ctx, big, big)
    with pytest.raises(native.KdecError, match="too small"):
        tokens.residual_norm(ctx, x, x, out=(torch.empty(32, device="cuda").expand(4, 32), None))
    with pytest.raises(native.KdecError, match="aligned"):
        tokens.residual_norm_bwd(ctx, x, x, x, x, torch.ones(17, device="cuda")[1:].view(4, 4), **fine)
    none = x[:0]
    r, y, s = tokens.residual_norm(ctx, none, none, keep=True, **fine)
    assert r.shape == y.shape == (0, 32)
    dx, dz, dg, (dw, _), _ = tokens.residual_norm_bwd(ctx, none, none, none, none, s, gate=w, **fine)
    assert dx.shape == (0, 32) and not dg.any() and not dw.any()


def test_more_rows_than_a_launch_holds(ctx):
    """2^26 rows in blocks of four would be 2^32 threads: refused, with nothing written."""
    from brosoundml_amd import native, tokens
    t = 1 << 26
    y = torch.full((t, 1), 7.0, device="cuda")
    x = torch.ones(1, 1, device="cuda").expand(t, 1)
    with pytest.raises(native.KdecError, match="too many rows"):
        tokens.residual_norm(ctx, x, pre=torch.ones(1, device="cuda"), out=(None, y))
    assert (y == 7).all()
    n = t - 4
    tokens.residual_norm(ctx, x[:n], pre=torch.ones(1, device="cuda"), out=(None, y[:n]), eps=3.0)
    # 1 / sqrt(1 + 3), the root and its reciprocal within a few steps of a float's half rounding
    assert ((y[:n] - 0.5).abs() <= 4 * 2.0 ** -24).all() and (y[n:] == 7).all()
