"""The 8-bit cache: its codes bit for bit, and attention over it (kdec_cache_write / kdec_cache_read /
kdec_attn_cache_fwd) against the definition in 64 bits, document by document.

Attention's tolerances, per element, from the roundings that the kernel makes; u is the type's unit roundoff, e the
float sums' share as for the attention over float keys, with one rounding more for each scale and three terms' sums
for float queries:
  e = 2^-24 (12 sqrt(D) max_j sum_d |q k| scale + 4 sqrt(keys) + 24)
  o : one rounding of every p times the value's scale and one of o: (2 u + e) sum_j p |v|;  lse: e (1 + |lse|)
"""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
TYPES = pytest.mark.parametrize("ty", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])


@pytest.fixture(scope="module")
def ctx():
    from brosoundml_amd import native
    return native.Context(0)


def ints(a):
    return None if a is None else torch.tensor(np.asarray(a), dtype=torch.int32).cuda()


def coded(x):
    """Scales and codes of (rows, heads, width) by the definition, ties decided on exact quotients of float values."""
    x = x.double().cpu()
    bad = ~torch.isfinite(x).all(-1)
    s = torch.clamp((torch.where(bad[..., None], torch.zeros_like(x), x).abs().amax(-1) / 127).float(), min=2.0 ** -126)
    q = torch.round(torch.nan_to_num(x, 0, 0, 0) / s.double()[..., None])
    q[bad] = 0
    s[bad] = math.nan
    return s, q


def empty(rows, heads, width, layout="new"):
    from brosoundml_amd import tokens
    W = (width + 15) // 16 * 16
    if layout == "heads":  # (heads, rows, width) storage
        codes = [torch.full((heads, rows, W), 99, dtype=torch.int8, device="cuda").permute(1, 0, 2) for _ in range(2)]
    elif layout == "both":  # keys and values of a token side by side
        codes = list(torch.full((rows, 2, heads, W), 99, dtype=torch.int8, device="cuda").unbind(1))
    else:
        codes = [torch.full((rows, heads, W), 99, dtype=torch.int8, device="cuda") for _ in range(2)]
    return tokens.Cache(*codes, *(torch.full((heads, rows), 5.0, device="cuda") for _ in range(2)))


def places(lq, k_off, k_len, rows_q, tk):
    """The cache row of every query row, -1 for none."""
    at = np.full(rows_q, -1)
    a = 0
    for d, n in enumerate(lq):
        slot = min(k_off[d + 1], tk) - k_off[d]
        lk = slot if k_len is None else min(max(k_len[d], 0), slot)
        for i in range(n):
            p = i + lk - n
            if p >= 0:
                at[a + i] = k_off[d] + p
        a += n
    return at


@TYPES
@pytest.mark.parametrize("layout", ["new", "heads", "both"])
@pytest.mark.parametrize("h,d,lq,slots,k_len", [
    (1, 1, [1], [1], None), (4, 128, [1] * 7, [5] * 7, [1, 5, 2, 0, 3, 4, 5]), (3, 40, [3, 0, 17, 1], [3, 4, 30, 9], [3, 2, 29, 9]),
    (12, 64, [33, 70], [33, 200], None), (2, 77, [5], [3], [3]), (1, 128, [1] * 150, [2] * 150, [1, 2] * 75), (5, 16, [9, 9], [9, 20], [30, -4])])
def test_write_and_read(ctx, ty, layout, h, d, lq, slots, k_len):
    from brosoundml_amd import tokens
    rng = np.random.default_rng([h, d, len(lq)])
    k_off = np.concatenate([[2], 2 + np.cumsum(slots)])
    tk, tq = int(k_off[-1]) + 3, sum(lq) + 2
    W = (d + 15) // 16 * 16
    mk = lambda: torch.from_numpy((rng.standard_normal((tq, h, d)) * np.exp(rng.uniform(-20, 20, (tq, h, 1)))).astype(np.float32)).to(ty)  # noqa: E731
    k, v = mk(), mk()
    wide = torch.stack([k, v, k], 1).cuda()  # parts of a fused projection's rows
    cache = empty(tk, h, d, layout)
    q_off = ints(np.concatenate([[0], np.cumsum(lq)]))
    args = (q_off, ints(k_off), ints(k_len))
    tokens.cache_write(ctx, wide[:, 0], wide[:, 1], cache, *args)
    at = places(lq, k_off, k_len, tq, tk)
    written = torch.zeros(tk, dtype=torch.bool)
    written[at[at >= 0]] = True
    for x, codes, scales in ((k, cache.k, cache.k_scale), (v, cache.v, cache.v_scale)):
        s, q = coded(x)
        codes, scales = codes.cpu(), scales.cpu()
        rows = at >= 0
        assert torch.equal(scales[:, at[rows]].t(), s[rows]) and torch.equal(codes[at[rows]][..., :d].double(), q[rows])
        assert not codes[at[rows]][..., d:].any()
        assert (codes[~written] == 99).all() and (scales[:, ~written] == 5).all()
    got = tokens.cache_read(ctx, cache, *args, rows=tq, width=d, dtype=ty)
    for x, g in zip((k, v), got):
        s, q = coded(x)
        want = q * s.double()[..., None]
        want[at < 0] = 0
        assert ((g.double().cpu() - want).abs() <= (U[ty] + 2.0 ** -24) * want.abs()).all()
    if W != d or layout == "new":
        out = [torch.full((tq, h, d + 3), 3.0, dtype=ty, device="cuda") for _ in range(2)]
        tokens.cache_read(ctx, cache, *args, rows=tq, width=d, dtype=ty, out=[o[..., 1:1 + d] for o in out])
        assert all(torch.equal(o[..., 1:1 + d], g) and (o[..., 0] == 3).all() and (o[..., 1 + d:] == 3).all() for o, g in zip(out, got))


def test_codes_at_ties_and_ends(ctx):
    """Values half between two codes go to the even one, those a last place beside to their side; the smallest and largest
    floats, and rows of zeros."""
    from brosoundml_amd import tokens
    rows = []
    for top in (127.0, 1.0, 3.1e38, 2.0 ** -126, 2.0 ** -149, 1e-30, 127.0 * 2.0 ** -126):
        s = max(np.float32(top / 127), np.float32(2.0 ** -126))
        x = [np.float32(top)]
        for m in range(31):
            mid = np.float32((m + 0.5) * float(s))
            x += [mid, np.nextafter(mid, np.float32(np.inf)), np.nextafter(mid, np.float32(-np.inf)), -mid]
        rows.append(np.clip(np.array(x + [0, 0, -top], np.float32), -np.float32(top), np.float32(top)))
    rows.append(np.zeros(128, np.float32))
    rng = np.random.default_rng(1)
    for _ in range(400):
        r = rng.standard_normal(128).astype(np.float32)
        s = np.float32(np.abs(r).max() / np.float64(127))
        r[:64] = np.where(np.abs(r[:64]) < np.abs(r).max(), ((np.floor(r[:64] / s) + 0.5) * s.astype(np.float64)).astype(np.float32), r[:64])
        rows.append(r)
    x = torch.from_numpy(np.stack(rows))[:, None]
    n = x.shape[0]
    cache = empty(n, 1, 128)
    tokens.cache_write(ctx, x.cuda(), x.cuda(), cache, ints([0, n]), ints([0, n]))
    s, q = coded(x)
    assert torch.equal(cache.k_scale.cpu()[0], s[:, 0]) and torch.equal(cache.k.cpu().double(), q) and torch.equal(cache.v.cpu().double(), q)
    assert q.abs().max() == 127


def test_values_that_are_not_finite(ctx):
    """They make their token's scale in that head NaN and nothing else; the rows that see the token NaN, no others."""
    from brosoundml_amd import tokens
    g = torch.Generator().manual_seed(2)
    n = 300
    k, v, q = (torch.randn(n, 2, 64, generator=g).cuda() for _ in range(3))
    off = ints([0, 100, n])
    cache, clean = empty(n, 2, 64), empty(n, 2, 64)
    tokens.cache_write(ctx, k, v, clean, off, off)
    k2, v2 = k.clone(), v.clone()
    k2[150, 0, 63], v2[200, 1, 0] = math.nan, -math.inf
    tokens.cache_write(ctx, k2, v2, cache, off, off)
    assert torch.isnan(cache.k_scale[0, 150]) and torch.isnan(cache.v_scale[1, 200])
    assert int(torch.isnan(cache.k_scale).sum() + torch.isnan(cache.v_scale).sum()) == 2
    back = tokens.cache_read(ctx, cache, off, off, rows=n, width=64, dtype=torch.float32)
    assert torch.isnan(back[0][150, 0]).all() and torch.isnan(back[1][200, 1]).all() and int(torch.isnan(back[0]).sum()) == 64
    o, lse = tokens.cache_attention(ctx, q, cache, off, off, causal=True)
    o2, lse2 = tokens.cache_attention(ctx, q, clean, off, off, causal=True)
    for h, at in ((0, 150), (1, 200)):
        assert torch.isnan(o[at:, h]).all() and torch.isnan(lse[h, at:]).all()
        assert torch.equal(o[:at, h], o2[:at, h]) and torch.equal(lse[h, :at], lse2[h, :at])


def oracle(q, cache, D, lq, k_off, k_len, causal, prefix, scale, cap, slopes):
    q = q.double().cpu()
    tq, hq, _ = q.shape
    hkv = cache.k.shape[1]
    tk = cache.k.shape[0]
    K, V = ((c.cpu().double()[..., :D] * s.cpu().double().t()[..., None]) for c, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)))
    o, w, lse, reach, most = torch.zeros_like(q), torch.zeros_like(q), torch.full((hq, tq), -math.inf, dtype=torch.float64), 0.0, 0
    a = 0
    for d, n in enumerate(lq):
        slot = min(k_off[d + 1], tk) - k_off[d]
        lk = slot if k_len is None else min(max(k_len[d], 0), slot)
        b, k0 = a + n, k_off[d]
        if n and lk:
            pos, key = torch.arange(n)[:, None] + lk - n, torch.arange(lk)[None]
            see = torch.ones(n, lk, dtype=torch.bool)
            if causal:
                see = key <= pos
                if prefix is not None:
                    see = see | (key < prefix[d])
            for h in range(hq):
                k, v = K[k0:k0 + lk, h * hkv // hq], V[k0:k0 + lk, h * hkv // hq]
                s = scale * q[a:b, h] @ k.T
                reach = max(reach, float(torch.where(see, scale * q[a:b, h].abs() @ k.abs().T, torch.zeros(()).double()).max()))
                if cap:
                    s = cap * torch.tanh(s / cap)
                if slopes is not None:
                    s = s - float(slopes[h]) * (pos - key).abs()
                s = s.masked_fill(~see, -math.inf)
                L = torch.logsumexp(s, -1)
                p = torch.where(see, torch.exp(s - torch.where(L == -math.inf, torch.zeros(()).double(), L)[:, None]), torch.zeros(()).double())
                o[a:b, h], w[a:b, h], lse[h, a:b] = p @ v, p @ v.abs(), L
                most = max(most, lk)
        a = b
    return o, w, lse, 2.0 ** -24 * (12 * math.sqrt(D) * reach + 4 * math.sqrt(most) + 24)


def compare(ctx, ty, lq, lk, hq, hkv, D, *, slots=None, causal=True, prefix=None, cap=0.0, slopes=False, pad=0, layout="both", odd=False, spoil=True,
            full=False):
    from brosoundml_amd import tokens
    rng = np.random.default_rng([sum(lq), sum(lk), hq, D])
    slots = [n + int(rng.integers(0, 40)) for n in lk] if slots is None and not full else slots or lk
    k_off = np.concatenate([[1], 1 + np.cumsum(slots)]).tolist()
    tk, tq = k_off[-1] + pad, sum(lq) + pad
    mk = lambda n, h: torch.from_numpy(rng.standard_normal((n, h, D)).astype(np.float32))  # noqa: E731
    cache = empty(tk, hkv, D, layout)
    for codes, scales in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        s, c = coded(mk(tk, hkv))
        codes[..., :D] = c.to(torch.int8).cuda()
        codes[..., D:] = 0
        scales.copy_(s.t())
    q = mk(tq, hq).to(ty).cuda()
    if odd:
        s = torch.zeros(tq, hq * D + 3, dtype=ty, device="cuda")
        s[:, 1:1 + hq * D] = q.view(tq, -1)
        q = s[:, 1:1 + hq * D].unflatten(1, (hq, D))
    if spoil:  # what no document holds must not matter
        keep = torch.zeros(tk, dtype=torch.bool)
        for a, n in zip(k_off, lk):
            keep[a:a + n] = True
        for codes, scales in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
            scales[:, ~keep.cuda()] = math.nan
            codes[~keep.cuda()] = -128
    sl = [2.0 ** (-8.0 * (h + 1) / hq) for h in range(hq)] if slopes else None
    args = (ints(np.concatenate([[0], np.cumsum(lq)])), ints(k_off), None if full else ints(lk))
    kw = dict(causal=causal, prefix=ints(prefix), cap=cap, slopes=None if sl is None else torch.tensor(sl).cuda())
    o, lse = tokens.cache_attention(ctx, q, cache, *args, **kw)
    want, w, L, e = oracle(q, cache, D, lq, k_off, None if full else lk, causal, prefix, D ** -0.5, cap, sl)
    off, tol = (o.double().cpu() - want).abs(), (2 * U[ty] + e) * w + 1e-30
    assert (off <= tol).all(), float((off / tol).max())
    got = lse.double().cpu()
    assert torch.equal(got == -math.inf, L == -math.inf)
    seen = L > -math.inf
    assert ((got - L).abs()[seen] <= e * (1 + L.abs()[seen])).all()
    out = torch.full((tq, hq, D + 5), 9.0, dtype=ty, device="cuda")  # into a part of something wider, the same bits
    o2, lse2 = tokens.cache_attention(ctx, q, cache, *args, **kw, out=out[..., 2:2 + D])
    assert torch.equal(out[..., 2:2 + D], o) and torch.equal(lse, lse2) and (out[..., :2] == 9).all() and (out[..., 2 + D:] == 9).all()


@TYPES
@pytest.mark.parametrize("hq,hkv,D", [(1, 1, 64), (16, 4, 128), (12, 12, 64), (8, 1, 128), (14, 2, 40), (5, 5, 1), (40, 1, 96), (33, 1, 17), (6, 2, 80), (70, 2, 128)])
def test_one_row_for_a_request(ctx, ty, hq, hkv, D):
    lk = [1, 31, 0, 32, 33, 260, 700]
    compare(ctx, ty, [1] * 7, lk, hq, hkv, D, pad=3)
    compare(ctx, ty, [1, 1], [5, 40], hq, hkv, D, full=True, spoil=False)


@TYPES
@pytest.mark.parametrize("lq,lk", [([4] * 5, [4, 9, 100, 333, 64]), ([1, 4, 0, 2, 3], [50, 4, 7, 200, 1]), ([90, 33], [290, 33]), ([200], [1111]),
                                   ([0, 0, 6], [5, 0, 6]), ([3], [0]), ([70, 1, 1, 8], [64, 300, 2, 8])])
@pytest.mark.parametrize("hq,hkv,D", [(16, 4, 128), (12, 12, 64), (7, 1, 24)])
def test_rows(ctx, ty, lq, lk, hq, hkv, D):
    compare(ctx, ty, lq, lk, hq, hkv, D, pad=2)


@TYPES
@pytest.mark.parametrize("cap,slopes,prefix,causal", [(30.0, False, None, True), (0.0, True, None, True), (5.0, True, [0, 17, 400, 3], True), (100.0, False, None, False),
                                                      (0.0, False, [9, 80, 2, 0], True), (0.0, True, None, False)])
def test_masks_and_scores(ctx, ty, cap, slopes, prefix, causal):
    for hq, hkv, D in ((8, 2, 128), (6, 6, 48)):
        compare(ctx, ty, [12, 40, 1, 5], [33, 90, 500, 5], hq, hkv, D, cap=cap, slopes=slopes, prefix=prefix, causal=causal, pad=4)


@TYPES
@pytest.mark.parametrize("layout,odd", [("new", False), ("heads", True), ("both", True)])
def test_layouts(ctx, ty, layout, odd):
    compare(ctx, ty, [1, 1, 20], [77, 600, 90], 8, 4, 128, layout=layout, odd=odd)
    compare(ctx, ty, [2, 3], [600, 90], 3, 3, 50, layout=layout, odd=odd)


@TYPES
def test_long_caches_in_parts(ctx, ty):
    compare(ctx, ty, [1], [6001], 12, 12, 64, slopes=True)
    compare(ctx, ty, [1, 2], [9000, 13], 16, 4, 128)
    compare(ctx, ty, [3], [20000], 2, 1, 128)


@TYPES
def test_many_documents(ctx, ty):
    rng = np.random.default_rng(4)
    compare(ctx, ty, [1] * 300, rng.integers(0, 40, 300).tolist(), 2, 2, 64)
    lq = rng.integers(0, 4, 200).tolist()
    compare(ctx, ty, lq, (np.array(lq) + rng.integers(0, 30, 200)).tolist(), 6, 2, 32, pad=5)


def test_as_attention_over_the_values_read_back(ctx):
    """A step through the cache is a step of ``attention`` over what ``cache_read`` gives, in float to its sums."""
    from brosoundml_amd import tokens
    g = torch.Generator().manual_seed(7)
    slot, docs, lk = 200, 5, [200, 1, 64, 130, 33]
    k, v = (torch.randn(sum(lk), 4, 64, generator=g).cuda() for _ in range(2))
    q = torch.randn(docs, 8, 64, generator=g).cuda()
    cache = tokens.new_cache(ctx, docs * slot, 4, 64)
    k_off, rows = ints(np.arange(docs + 1) * slot), ints(np.arange(docs + 1))
    full = ints(np.concatenate([[0], np.cumsum(lk)]))
    tokens.cache_write(ctx, k, v, cache, full, k_off, ints(lk))
    kr, vr = tokens.cache_read(ctx, cache, full, k_off, ints(lk), rows=sum(lk), width=64, dtype=torch.float32)
    a, la = tokens.cache_attention(ctx, q, cache, rows, k_off, ints(lk), causal=True)
    b, lb = tokens.attention(ctx, q, kr, vr, rows, full, causal=True)
    # both are off by e sum p |v| at most, e below 2^-24 (12 * 8 * 30 + 4 * 15 + 24) with sum |q k| / 8 below 30
    e = 2 * 2.0 ** -24 * 3000
    assert float((a - b).abs().max()) <= e * float(vr.abs().max()) and float((la - lb).abs().max()) <= e * (1 + float(lb.abs().max()))


def test_offsets_past_32_bits(ctx):
    from brosoundml_amd import tokens
    rows, h, d = 2300000, 8, 128
    g = torch.Generator().manual_seed(1)
    cache = tokens.Cache(*(torch.empty(rows, h, d, dtype=torch.int8, device="cuda") for _ in range(2)),
                         *(torch.empty(h, rows, device="cuda") for _ in range(2)))
    k, v, q = (torch.randn(300, h, d, generator=g).cuda() for _ in range(3))
    off = ints([0, 300])
    near = empty(300, h, d)
    tokens.cache_write(ctx, k, v, near, off, off)
    far = ints([rows - 300, rows])
    tokens.cache_write(ctx, k, v, cache, off, far)
    for a, b in zip(near, cache):
        assert torch.equal(a, b[-300:] if a.dtype == torch.int8 else b[:, -300:])
    args = dict(rows=300, width=d, dtype=torch.float32)
    assert all(torch.equal(a, b) for a, b in zip(tokens.cache_read(ctx, near, off, off, **args), tokens.cache_read(ctx, cache, off, far, **args)))
    # as many parts as the far cache's length makes of it: the sums' grouping differs, no more
    a, b = (tokens.cache_attention(ctx, q, c, off, o, causal=True)[0] for c, o in ((near, off), (cache, far)))
    assert float((a - b).abs().max()) <= 2 * 2.0 ** -24 * 6000 * float(v.abs().max())


def test_refusals(ctx):
    from brosoundml_amd import native, tokens
    k = torch.ones(4, 2, 40, device="cuda")
    cache = tokens.new_cache(ctx, 8, 2, 40)
    q_off, k_off, k_len = ints([0, 4]), ints([0, 8]), ints([6])
    w = lambda k=k, v=None, c=cache, a=(q_off, k_off, k_len): tokens.cache_write(ctx, k, k if v is None else v, c, *a)  # noqa: E731
    r = lambda c=cache, rows=4, width=40, a=(q_off, k_off, k_len), **kw: tokens.cache_read(ctx, c, *a, rows=rows, width=width, **kw)  # noqa: E731
    at = lambda q=k, c=cache, a=(q_off, k_off, k_len), **kw: tokens.cache_attention(ctx, q, c, *a, **kw)  # noqa: E731
    w(), r(), at()
    part = tokens.Cache(*(t[..., :40] for t in cache[:2]), *cache[2:])
    for call in (lambda: w(k.half()), lambda: w(k[..., :32]), lambda: w(k, k[:3]), lambda: w(c=part), lambda: w(k[:, :1], k[:, :1]),
                 lambda: w(a=(q_off, k_off[:1], k_len)), lambda: w(a=(q_off.long(), k_off, k_len)), lambda: w(a=(q_off, k_off, k_len.cpu())),
                 lambda: w(k.clone().requires_grad_()), lambda: w(c=cache._replace(k_scale=cache.k_scale.t())), lambda: w(c=cache._replace(k=cache.k.float())),
                 lambda: r(width=50), lambda: r(dtype=torch.float16), lambda: r(out=(k, k[:3])), lambda: at(k.half()), lambda: at(k.cpu()),
                 lambda: at(out=k[:3]), lambda: at(prefix=q_off), lambda: at(slopes=torch.ones(3, device="cuda")), lambda: at(k.clone().requires_grad_())):
        with pytest.raises(ValueError, match="brosoundml"):
            call()
    far = torch.empty(8 << 24, dtype=torch.int8, device="cuda")
    odd = torch.zeros(8 * 2 * 48 + 64, dtype=torch.int8, device="cuda")
    for call, why in ((lambda: w(c=cache._replace(k=odd.as_strided((8, 2, 48), (96, 48, 1), 8))), "16 bytes"),
                      (lambda: w(c=cache._replace(v=odd.as_strided((8, 2, 48), (104, 48, 1)))), "16 bytes"),
                      (lambda: w(c=cache._replace(v=odd.as_strided((8, 2, 48), (0, 48, 1)))), "overlap"),
                      (lambda: at(c=cache._replace(v=far.as_strided((8, 2, 48), (1 << 24, 48, 1)))), "strides"),
                      (lambda: at(scale=0.0), "scale"), (lambda: at(cap=-1.0), "cap"), (lambda: at(k[:, :1].expand(4, 3, 40)), "multiple"),
                      (lambda: at(out=torch.empty(2, 40, device="cuda").expand(4, 2, 40)), "overlap"),
                      (lambda: r(out=(k.clone(), torch.empty(2, 40, device="cuda").expand(4, 2, 40))), "overlap")):
        with pytest.raises(native.KdecError, match=why):
            call()
    wide = torch.ones(2, 1, 129, device="cuda")
    with pytest.raises(native.KdecError, match="width"):
        tokens.cache_write(ctx, wide, wide, tokens.new_cache(ctx, 2, 1, 129), ints([0, 2]), ints([0, 2]))
    none = tokens.new_cache(ctx, 0, 2, 40)
    o, lse = tokens.cache_attention(ctx, k, none, q_off, ints([0, 0]))
    assert not o.any() and (lse == -math.inf).all()
    tokens.cache_write(ctx, k, k, none, q_off, ints([0, 0]))
    assert not tokens.cache_read(ctx, none, q_off, ints([0, 0]), rows=4, width=40)[0].any()
    assert tokens.cache_attention(ctx, k[:0], cache, ints([0]), ints([0]))[0].shape == (0, 2, 40)
    assert not tokens.cache_attention(ctx, k, cache, ints([0]), ints([0]))[0].any()  # rows that no document holds
