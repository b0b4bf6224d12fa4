"""Attention over packed documents (kdec_attn_fwd / kdec_attn_bwd) against the
definition in 64 bits, document by document.

Tolerances, per element, from the roundings that the kernels make; u is the
type's unit roundoff (2^-p at p bits of precision: 2^-8 bf16, 2^-24 float), e the float sums' share:
  e  = 2^-24 (4 sqrt(D) max_j sum_d |q k| scale + 4 sqrt(keys) + 16)
  o  : one rounding of every p and one of o:       (2 u + e) sum_j p |v|
  dq : one of every ds, one of dq, and o's in delta: scale sum_j ((2 u + 4 e) |ds|
       + (u + 4 e) p (|do| |o| + sum_d |do v|)) |k|, u's part of the last only from |do| |o|
  dk : the same over the rows, dv : (2 u + 4 e) sum_i p |do|
(float: u is below e's 16 2^-24). lse: e (1 + |lse|).
"""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


@pytest.fixture(scope="module")
def ctx():
    from brosoundml_amd import native
    return native.Context(0)


def oracle(q, k, v, do, q_off, k_off, k_len, causal, prefix, scale, cap, slopes):
    """o, lse, dq, dk, dv in float64 and the element tolerances' weights, by the definition."""
    q, k, v, do = (t.double().cpu() for t in (q, k, v, do))
    tq, hq, D = q.shape
    tk, hkv, _ = k.shape
    g = hq // hkv
    r = {n: torch.zeros_like(t) for n, t in (("o", q), ("dq", q), ("dk", k), ("dv", v))}
    lse = torch.full((hq, tq), -math.inf, dtype=torch.float64)
    wt = {n: torch.zeros_like(t) for n, t in r.items()}   # u's weights
    we = {n: torch.zeros_like(t) for n, t in r.items()}   # e's
    reach = 0.0
    for d in range(len(q_off) - 1):
        a, b, k0 = q_off[d], q_off[d + 1], k_off[d]
        lk = k_off[d + 1] - k0 if k_len is None else k_len[d]
        lq = b - a
        if lq == 0 or lk == 0:
            continue
        pos = torch.arange(lq)[:, None] + lk - lq
        key = torch.arange(lk)[None]
        see = torch.ones(lq, lk, dtype=torch.bool)
        if causal:
            see = key <= pos
            if prefix is not None:
                see = see | (key < prefix[d])
        for h in range(hq):
            Q, K, V, G = q[a:b, h], k[k0:k0 + lk, h // g], v[k0:k0 + lk, h // g], do[a:b, h]
            s = scale * Q @ K.T
            reach = max(reach, float((scale * Q.abs() @ K.abs().T).where(see, torch.zeros(())).max()))
            dt = torch.ones_like(s)
            if cap:
                th = torch.tanh(s / cap)
                s, dt = cap * th, 1 - th * th
            if slopes is not None:
                s = s - float(slopes[h]) * (pos - key).abs()
            s = s.masked_fill(~see, -math.inf)
            L = torch.logsumexp(s, -1)
            p = torch.where(see, torch.exp(s - torch.where(L == -math.inf, torch.zeros(()).double(), L)[:, None]), torch.zeros(()).double())
            o = p @ V
            dp = G @ V.T
            ds = p * (dp - (G * o).sum(-1, keepdim=True)) * dt
            r["o"][a:b, h], lse[h, a:b] = o, L
            r["dq"][a:b, h] = scale * ds @ K
            r["dk"][k0:k0 + lk, h // g] += scale * ds.T @ Q
            r["dv"][k0:k0 + lk, h // g] += p.T @ G
            wt["o"][a:b, h] = we["o"][a:b, h] = p @ V.abs()
            go = (G.abs() * o.abs()).sum(-1, keepdim=True)
            du, de = 2 * ds.abs() + p * go, 4 * ds.abs() + 4 * p * (go + G.abs() @ V.abs().T)
            wt["dq"][a:b, h], we["dq"][a:b, h] = scale * du @ K.abs(), scale * de @ K.abs()
            wt["dk"][k0:k0 + lk, h // g] += scale * du.T @ Q.abs()
            we["dk"][k0:k0 + lk, h // g] += scale * de.T @ Q.abs()
            wt["dv"][k0:k0 + lk, h // g] += 2 * p.T @ G.abs()
            we["dv"][k0:k0 + lk, h // g] += 4 * p.T @ G.abs()
    wt["o"] = 2 * wt["o"]
    return r, lse, wt, we, reach


def tensors(rng, ty, tq, tk, hq, hkv, D, layout):
    def t(n, h):
        a = torch.from_numpy(rng.standard_normal((n, h, D)).astype(np.float32)).to(ty)
        if layout == "heads":      # (heads, rows, width) storage
            return a.permute(1, 0, 2).contiguous().cuda().permute(1, 0, 2)
        if layout == "odd":        # rows that start anywhere
            s = torch.zeros(n, h * D + 3, dtype=ty)
            s[:, 1:1 + h * D] = a.view(n, h * D)
            return s.cuda().as_strided((n, h, D), (h * D + 3, D, 1), 1)
        return a.cuda()
    return t(tq, hq), t(tk, hkv), t(tk, hkv), t(tq, hq)


def compare(ctx, ty, lq, lk, hq, hkv, D, *, slots=None, causal=False, prefix=None, cap=0.0, slopes=False, pad=0,
            layout="packed", seed=0, scale=None, spoil=False):
    from brosoundml_amd import tokens
    rng = np.random.default_rng([seed, sum(lq), sum(lk), hq, D])
    q_off = np.concatenate([[0], np.cumsum(lq)]).tolist()
    k_off = np.concatenate([[0], np.cumsum(slots or lk)]).tolist()
    k_len = None if slots is None else list(lk)
    tq, tk = q_off[-1] + pad, k_off[-1] + pad
    q, k, v, do = tensors(rng, ty, tq, tk, hq, hkv, D, layout)
    if spoil:  # what no document holds must not matter
        for t, off, n in ((q, q_off, lq), (do, q_off, lq), (k, k_off, lk), (v, k_off, lk)):
            keep = torch.zeros(t.shape[0], dtype=torch.bool)
            for a, m in zip(off, n):
                keep[a:a + m] = True
            t[~keep.cuda()] = spoil
    clean = [torch.nan_to_num(t.float(), 0.0, 0.0, 0.0) for t in (q, k, v, do)]
    sl = torch.tensor([2.0 ** (-8.0 * (h + 1) / hq) for h in range(hq)]).cuda() if slopes else None
    sc = D ** -0.5 if scale is None else scale
    I = lambda a: None if a is None else torch.tensor(a, dtype=torch.int32).cuda()  # noqa: E731
    mask = dict(causal=causal, prefix=I(prefix), cap=cap, slopes=sl, scale=scale)
    o, lse = tokens.attention(ctx, q, k, v, I(q_off), I(k_off), I(k_len), **mask)
    dq, dk, dv = tokens.attention_bwd(ctx, q, k, v, o, lse, do, I(q_off), I(k_off), I(k_len), **mask)
    r, L, wt, we, reach = oracle(*clean, q_off, k_off, k_len, causal, prefix, sc, cap, sl)
    e = 2.0 ** -24 * (4 * math.sqrt(D) * max(reach, 1.0) + 4 * math.sqrt(max(max(lk), 1)) + 16)
    u = U[ty]
    lse = lse.cpu().double()
    assert torch.equal(lse == -math.inf, L == -math.inf)
    fin = L > -math.inf
    assert ((lse - L)[fin].abs() <= e * (1 + L[fin].abs())).all()
    for n, got in (("o", o), ("dq", dq), ("dk", dk), ("dv", dv)):
        tol = u * wt[n] + e * we[n] + 1e-30
        off = (got.cpu().double() - r[n]).abs()
        assert torch.isfinite(off).all(), n
        worst = float((off / tol).max()) if off.numel() else 0.0
        assert worst <= 1.0, (n, worst)
    return q, k, v, o, lse


TYPES = [torch.float32, torch.bfloat16]


@pytest.mark.parametrize("ty", TYPES, ids=["f32", "bf16"])
@pytest.mark.parametrize("case", [
    dict(lq=[1], lk=[1], hq=1, hkv=1, D=64),
    dict(lq=[37], lk=[37], hq=2, hkv=2, D=64),
    dict(lq=[64, 0, 1, 130, 5], lk=[64, 0, 1, 130, 5], hq=4, hkv=2, D=64, pad=7),
    dict(lq=[129, 63], lk=[129, 63], hq=3, hkv=1, D=128, causal=True),
    dict(lq=[40, 200], lk=[70, 200], hq=2, hkv=2, D=96, causal=True, prefix=[50, 3]),
    dict(lq=[50, 9], lk=[20, 40], hq=2, hkv=1, D=40, causal=True),               # rows before the first key see none
    dict(lq=[50, 9, 3], lk=[20, 0, 90], hq=2, hkv=1, D=40),                      # a document without keys
    dict(lq=[100, 31], lk=[100, 31], hq=5, hkv=5, D=64, cap=2.0),
    dict(lq=[300], lk=[300], hq=4, hkv=4, D=64, slopes=True),
    dict(lq=[300, 20], lk=[300, 20], hq=14, hkv=2, D=128, slopes=True, cap=30.0, causal=True, prefix=[17, 20]),
    dict(lq=[33, 65], lk=[33, 65], hq=2, hkv=2, D=1),
    dict(lq=[33, 65], lk=[90, 65], hq=2, hkv=1, D=77, causal=True),
    dict(lq=[33, 65], lk=[33, 60], slots=[40, 100], hq=2, hkv=1, D=64),
    dict(lq=[70, 40], lk=[70, 40], hq=4, hkv=2, D=64, layout="heads"),
    dict(lq=[70, 40], lk=[70, 40], hq=4, hkv=2, D=64, layout="odd", causal=True),
    dict(lq=[31, 200], lk=[31, 200], hq=2, hkv=2, D=64, scale=3.0),               # sharp softmax
    dict(lq=[40], lk=[3000], hq=2, hkv=2, D=64, causal=True),                     # the keys split over blocks
], ids=lambda c: "-".join(f"{k}{v}" for k, v in c.items()).replace(" ", ""))
def test_against_definition(ctx, ty, case):
    case = dict(case)
    lq, lk, hq, hkv, D = (case.pop(n) for n in ("lq", "lk", "hq", "hkv", "D"))
    compare(ctx, ty, lq, lk, hq, hkv, D, **case)


@pytest.mark.parametrize("ty", TYPES, ids=["f32", "bf16"])
@pytest.mark.parametrize("case", [
    dict(lq=[1], lk=[1000], hq=4, hkv=4, D=64),
    dict(lq=[1, 1, 1], lk=[700, 1, 33], slots=[800, 90, 64], hq=8, hkv=2, D=128, causal=True),
    dict(lq=[1, 0, 1], lk=[700, 5, 0], slots=[800, 90, 64], hq=40, hkv=1, D=64, causal=True),  # 40 heads on one key head
    dict(lq=[3, 1], lk=[2, 515], slots=[300, 520], hq=6, hkv=2, D=64, causal=True),            # a row before the first key
    dict(lq=[1, 1], lk=[2049, 4000], hq=2, hkv=2, D=64, slopes=True, cap=20.0),
    dict(lq=[1], lk=[300], hq=3, hkv=1, D=33, layout="odd"),
], ids=lambda c: "-".join(f"{k}{v}" for k, v in c.items()).replace(" ", ""))
def test_few_rows_over_long_keys(ctx, ty, case):
    case = dict(case)
    lq, lk, hq, hkv, D = (case.pop(n) for n in ("lq", "lk", "hq", "hkv", "D"))
    compare(ctx, ty, lq, lk, hq, hkv, D, **case)


@pytest.mark.parametrize("ty", TYPES, ids=["f32", "bf16"])
@pytest.mark.parametrize("case", [
    dict(lq=[300, 0, 200], lk=[290, 130, 10], slots=[320, 140, 400], pad=150, causal=True, hq=2, hkv=1, D=64),
    dict(lq=[300, 1, 200], lk=[290, 0, 201], slots=[320, 140, 400], pad=3, hq=2, hkv=2, D=128, cap=4.0),
    dict(lq=[257, 128, 129], lk=[257, 128, 129], hq=3, hkv=1, D=128, causal=True, prefix=[130, 0, 129], slopes=True),
    dict(lq=[64, 190] * 33, lk=[64, 190] * 33, hq=1, hkv=1, D=64),                # more documents than a wave has lanes
], ids=lambda c: "-".join(f"{k}{str(v)[:24]}" for k, v in c.items()).replace(" ", ""))
def test_blocks_that_end_with_their_document(ctx, ty, case):
    case = dict(case)
    lq, lk, hq, hkv, D = (case.pop(n) for n in ("lq", "lk", "hq", "hkv", "D"))
    compare(ctx, ty, lq, lk, hq, hkv, D, spoil=math.nan if "slots" in case else False, **case)


@pytest.mark.parametrize("ty", TYPES, ids=["f32", "bf16"])
def test_rows_before_the_first_document(ctx, ty):
    """Rows that offsets leave out at either end get zeros, and the documents between them what they get alone."""
    from brosoundml_amd import tokens
    rng = np.random.default_rng(9)
    q, k, v, do = tensors(rng, ty, 700, 700, 2, 2, 64, "packed")
    for t in (q, k, v, do):
        t[:150] = math.nan
        t[680:] = math.nan

    def run(off, *t):
        off = torch.tensor(off, dtype=torch.int32).cuda()
        o, lse = tokens.attention(ctx, *t[:3], off)
        return (o, *tokens.attention_bwd(ctx, *t[:3], o, lse, t[3], off))

    want = run([0, 330, 530], *(t[150:680].contiguous() for t in (q, k, v, do)))
    for a, b in zip(run([150, 480, 680], q, k, v, do), want):
        assert torch.equal(a[150:680], b) and not a[:150].any() and not a[680:].any()


@pytest.mark.parametrize("ty", TYPES, ids=["f32", "bf16"])
@pytest.mark.parametrize("spoil", [math.nan, math.inf])
def test_rows_of_no_document_do_not_matter(ctx, ty, spoil):
    compare(ctx, ty, [20, 70], [17, 64], 2, 2, 64, slots=[40, 100], pad=11, causal=True, spoil=spoil)
    compare(ctx, ty, [1, 1], [17, 300], 2, 1, 64, slots=[200, 400], pad=11, causal=True, spoil=spoil)


@pytest.mark.parametrize("ty", TYPES, ids=["f32", "bf16"])
def test_nan_stays_in_its_document(ctx, ty):
    """A document with a NaN in q, k, v or do leaves its neighbours' results as they are without it, bit for bit."""
    from brosoundml_amd import tokens
    rng = np.random.default_rng(5)
    q, k, v, do = tensors(rng, ty, 90, 90, 2, 2, 64, "packed")
    off = torch.tensor([0, 30, 50, 90], dtype=torch.int32).cuda()

    def run(*t):
        o, lse = tokens.attention(ctx, *t[:3], off)
        return (o, *tokens.attention_bwd(ctx, *t[:3], o, lse, t[3], off))

    want = run(q, k, v, do)
    for i in range(4):
        t = [x.clone() for x in (q, k, v, do)]
        t[i][35, 1, 7] = math.nan
        for n, (a, b) in enumerate(zip(run(*t), want)):
            assert torch.equal(a[:30], b[:30]) and torch.equal(a[50:], b[50:]), (i, n)
            assert torch.equal(a[30:50, 0], b[30:50, 0]), (i, n)
        got = run(*t)
        assert torch.isnan(got[1 if i != 1 else 2][30:50, 1]).any()


def test_later_keys_that_are_not_finite(ctx):
    """Under the causal mask a row is as if the keys behind it did not exist."""
    from brosoundml_amd import tokens
    rng = np.random.default_rng(6)
    q, k, v, _ = tensors(rng, torch.bfloat16, 100, 100, 2, 2, 64, "packed")
    off = torch.tensor([0, 100], dtype=torch.int32).cuda()
    want, _ = tokens.attention(ctx, q, k, v, off, causal=True)
    for t in (k, v):
        t[60] = math.inf
    got, _ = tokens.attention(ctx, q, k, v, off, causal=True)
    assert torch.equal(got[:60], want[:60]) and torch.isnan(got[60:].float()).any(-1).all()


@pytest.mark.parametrize("ty", TYPES, ids=["f32", "bf16"])
def test_same_bits_again_and_on_another_stream(ctx, ty):
    from brosoundml_amd import native, tokens
    rng = np.random.default_rng(7)
    q, k, v, do = tensors(rng, ty, 333, 333, 6, 2, 64, "packed")
    off = torch.tensor([0, 33, 333], dtype=torch.int32).cuda()

    def run(c):
        o, lse = tokens.attention(c, q, k, v, off, causal=True)
        return (o, lse, *tokens.attention_bwd(c, q, k, v, o, lse, do, off, causal=True))

    want = run(ctx)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    c2 = native.Context(0, stream=side)
    for _ in range(2):
        got = run(c2)
        side.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)


def test_gradients_against_differences(ctx):
    """d(sum(o * do)) along a direction, by a central difference of the float forward in steps of 2^-8:
    the remainder is a third derivative's share of 2^-16 and the forward's rounding over the step, both
    within 2e-3 of the gradients' norm for these inputs of order one."""
    from brosoundml_amd import tokens
    rng = np.random.default_rng(8)
    q, k, v, do = tensors(rng, torch.float32, 60, 60, 4, 2, 64, "packed")
    off = torch.tensor([0, 21, 60], dtype=torch.int32).cuda()
    sl = torch.tensor([0.1, 0.2, 0.3, 0.4]).cuda()
    m = dict(causal=True, cap=5.0, slopes=sl, prefix=torch.tensor([4, 9], dtype=torch.int32).cuda())
    o, lse = tokens.attention(ctx, q, k, v, off, **m)
    grads = tokens.attention_bwd(ctx, q, k, v, o, lse, do, off, **m)
    h = 2.0 ** -8
    for i in range(3):
        t = [q, k, v]
        dr = torch.from_numpy(rng.standard_normal(tuple(t[i].shape)).astype(np.float32)).cuda()
        f = []
        for s in (1, -1):
            t2 = list(t)
            t2[i] = t[i] + s * h * dr
            f.append((tokens.attention(ctx, *t2, off, **m)[0].double() * do.double()).sum())
        num, ana = float(f[0] - f[1]) / (2 * h), float((grads[i].double() * dr.double()).sum())
        assert abs(num - ana) <= 2e-3 * float(grads[i].double().norm() * 2), (i, num, ana)


def test_refusals(ctx):
    from brosoundml_amd import native, tokens
    x = torch.zeros(8, 4, 64, device="cuda")
    off = torch.tensor([0, 8], dtype=torch.int32).cuda()
    with pytest.raises(ValueError):
        tokens.attention(ctx, x, x.bfloat16(), x.bfloat16(), off)
    with pytest.raises(ValueError):
        tokens.attention(ctx, x, x[:4], x[:4], off)
    with pytest.raises(ValueError):
        tokens.attention(ctx, x, x, x, off.long())
    with pytest.raises(ValueError):
        tokens.attention(ctx, x.cpu(), x, x, off)
    with pytest.raises(ValueError):
        tokens.attention(ctx, x.transpose(1, 2), x, x, off)
    for bad in (dict(scale=0.0), dict(scale=math.nan), dict(cap=-1.0)):
        with pytest.raises(native.KdecError):
            tokens.attention(ctx, x, x, x, off, **bad)
    with pytest.raises(native.KdecError, match="multiple"):
        tokens.attention(ctx, x, x[:, :3], x[:, :3], off)
    wide = torch.zeros(8, 1, 129, device="cuda")
    with pytest.raises(native.KdecError, match="width"):
        tokens.attention(ctx, wide, wide, wide, off)
    # nothing to do
    o, lse = tokens.attention(ctx, x[:0], x[:0], x[:0], torch.zeros(1, dtype=torch.int32, device="cuda"))
    assert o.shape == (0, 4, 64) and lse.shape == (4, 0)
    o, lse = tokens.attention(ctx, x, x[:0], x[:0], off, torch.zeros(2, dtype=torch.int32, device="cuda"))
    assert not o.any() and (lse == -math.inf).all()
