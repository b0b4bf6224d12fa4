"""Attention (kdec_attn_fwd / kdec_attn_bwd) where tensors hold values that are not finite in places that rows see:
what a row gets does not depend on the kernel or the tile in which a key comes up. A value that is not finite makes
the rows that see it NaN, o and lse; a key that is not finite enters the scores by the formula (the oracle in 64 bits
tells which) and makes every gradient NaN that the rows seeing it reach, and so does a query or an output gradient."""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16]
INF = math.inf


@pytest.fixture(scope="module")
def ctx():
    from brosoundml_amd import native
    return native.Context(0)


def inputs(ty, tq, tk, hq, hkv, D, seed):
    rng = np.random.default_rng([seed, tq, tk, D])
    return [torch.from_numpy(rng.standard_normal(s).astype(np.float32)).to(ty).cuda() for s in ((tq, hq, D), (tk, hkv, D), (tk, hkv, D), (tq, hq, D))]


def visible(lq, lk, causal):
    pos = torch.arange(lq)[:, None] + lk - lq
    return (torch.arange(lk)[None] <= pos) if causal else torch.ones(lq, lk, dtype=torch.bool)


def forward(q, k, v, see, cap):
    """o and lse of one head in 64 bits (no value of v is used where a row sees one that is not finite: NaN)."""
    q, k, v = (t.double().cpu() for t in (q, k, v))
    s = q @ k.T * q.shape[1] ** -0.5
    if cap:
        s = cap * torch.tanh(s / cap)
    s = torch.where(see, s, torch.tensor(-INF, dtype=torch.float64))
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(m == -INF, torch.zeros_like(m), m))
    lse = torch.log(p.sum(-1)) + m[:, 0]
    wild = see & ~torch.isfinite(v).all(-1)[None]
    o = (p / p.sum(-1, keepdim=True)) @ torch.nan_to_num(v, 0.0, 0.0, 0.0)
    bad = wild.any(-1) | torch.isnan(lse)
    o[bad], lse[bad] = math.nan, math.nan
    return o, lse, wild


CASES = {  # name: rows, keys, causal, cap; what holds which value
    "value-masked-tile": (200, 200, False, 0.0, "v", 170, INF),
    "value-whole-tile": (200, 200, False, 0.0, "v", 5, INF),
    "value-causal": (200, 200, True, 0.0, "v", 5, -INF),
    "value-nan-whole-tile": (200, 200, False, 0.0, "v", 70, math.nan),
    "value-one-row": (1, 3000, False, 0.0, "v", 1234, INF),
    "value-one-row-short": (1, 100, False, 0.0, "v", 99, INF),
    "key-low-masked-tile": (200, 200, False, 0.0, "k", 170, -INF),
    "key-low-whole-tile": (200, 200, False, 0.0, "k", 5, -INF),
    "key-low-causal-last": (200, 200, True, 0.0, "k", 199, -INF),
    "key-low-causal": (200, 200, True, 0.0, "k", 20, -INF),
    "key-high-masked-tile": (200, 200, False, 0.0, "k", 170, INF),
    "key-high-whole-tile": (200, 200, False, 0.0, "k", 5, INF),
    "key-capped-masked-tile": (200, 200, False, 5.0, "k", 170, INF),
    "key-capped-whole-tile": (200, 200, False, 5.0, "k", 5, -INF),
    "key-nan": (200, 200, True, 0.0, "k", 150, math.nan),
    "query-capped": (200, 200, False, 5.0, "q", 150, INF),
    "query-capped-causal": (200, 200, True, 5.0, "q", 90, -INF),
    "query": (200, 200, True, 0.0, "q", 90, INF),
    "grad": (200, 200, True, 0.0, "do", 90, INF),
    "key-low-one-row": (1, 2500, False, 0.0, "k", 700, -INF),
}


@pytest.mark.parametrize("ty", TYPES, ids=["f32", "bf16"])
@pytest.mark.parametrize("name", CASES)
@pytest.mark.parametrize("D,heads", [(64, 1), (128, 2)])
@pytest.mark.parametrize("many", [False, True], ids=["", "many"])
def test_rows_that_see_values_not_finite(ctx, ty, name, D, heads, many):
    """Two documents and two key heads; the first document's second key head is spoilt. `many`: enough rows of further
    documents behind them that the blocks fill the device."""
    from brosoundml_amd import tokens
    lq, lk, causal, cap, which, at, value = CASES[name]
    hkv, hq = 2, 2 * heads
    more = 60 if many and lq > 1 else 0
    lqs, lks = [lq, 40] + [300] * more, [lk, 40] + [300] * more
    t = dict(zip(("q", "k", "v", "do"), inputs(ty, sum(lqs), sum(lks), hq, hkv, D, at)))
    t["q"][:, :, 3] = t["q"][:, :, 3].abs() + 0.25  # so that an infinite key's score has the infinity's sign
    t["k"][:, :, 3] = t["k"][:, :, 3].abs() + 0.25
    clean = {n: x.clone() for n, x in t.items()}
    h = 1 if which in "kv" else hq - 1
    t[which][at, h, 3] = value
    q_off, k_off = (torch.tensor(np.concatenate([[0], np.cumsum(a)]), dtype=torch.int32).cuda() for a in (lqs, lks))
    mask = dict(causal=causal, cap=cap)

    def run(x):
        o, lse = tokens.attention(ctx, x["q"], x["k"], x["v"], q_off, k_off, **mask)
        return dict(zip(("o", "lse", "dq", "dk", "dv"), (o, lse.t(), *tokens.attention_bwd(ctx, x["q"], x["k"], x["v"], o, lse, x["do"], q_off, k_off, **mask))))

    got, want = run(t), run(clean)
    see = visible(lq, lk, causal)
    reached = {n: torch.zeros(got[n].shape[:2], dtype=torch.bool) for n in got}  # rows and heads that may differ from the clean run
    for hh in range(hq):
        kv = hh // heads
        q, k, v, do = (t[n][:(lq if n in ("q", "do") else lk), hh if n in ("q", "do") else kv] for n in ("q", "k", "v", "do"))
        o, lse, _ = forward(q, k, v, see, cap)
        # the forward: NaN where the formula has it, and near it elsewhere
        go, gl = got["o"][:lq, hh].double().cpu(), got["lse"][:lq, hh].double().cpu()
        assert torch.equal(torch.isnan(gl), torch.isnan(lse)), hh
        assert torch.equal(torch.isnan(go), torch.isnan(o)) and torch.isfinite(go[~torch.isnan(lse)]).all(), hh
        fine = ~torch.isnan(lse)
        # (p and o rounded to the type, each by 2^-8 or 2^-24 of values of at most 5; float sums of 3000 terms)
        tol = 5 * (2.0 ** -7 if ty == torch.bfloat16 else 2.0 ** -24 * (4 * math.sqrt(lk) + 4 * math.sqrt(D) * 16))
        assert ((go - o)[fine].abs() <= tol).all() and ((gl - lse)[fine].abs() <= 2.0 ** -24 * (4 * math.sqrt(lk) + 4 * math.sqrt(D) * 16) * 8).all(), hh
        # the backward: rows marked, and the keys that they see
        fin = lambda x: torch.isfinite(x.double().cpu()).all(-1)  # noqa: E731
        marked = ~fin(q) | ~fin(do) | torch.isnan(lse) | (see & ~fin(k)[None]).any(-1)
        reached["dq"][:lq, hh] |= marked
        reached["o"][:lq, hh] = reached["lse"][:lq, hh] = True
        keys = (see & marked[:, None]).any(0)
        reached["dk"][:lk, kv] |= keys
        reached["dv"][:lk, kv] |= keys
    for n in ("dq", "dk", "dv"):
        g, w, r = got[n].cpu(), want[n].cpu(), reached[n]
        assert r.any() and torch.isnan(g[r].float()).all(), n
        assert torch.equal(g[~r], w[~r]), n
    for n in ("o", "lse"):
        assert torch.equal(got[n].cpu()[~reached[n]], want[n].cpu()[~reached[n]]), n


@pytest.mark.parametrize("D", [64, 128])
def test_more_requests_than_a_wave_has_lanes(ctx, D):
    """One row each for 70 requests, one request's cache with an infinite value: its row is NaN, the others keep their bits."""
    from brosoundml_amd import tokens
    q, k, v, _ = inputs(torch.bfloat16, 70, 70 * 50, 4, 1, D, 1)
    q_off, k_off = torch.arange(71, dtype=torch.int32).cuda(), (torch.arange(71) * 50).int().cuda()
    k_len = torch.from_numpy(np.random.default_rng(4).integers(30, 50, 70)).int().cuda()
    want, wl = tokens.attention(ctx, q, k, v, q_off, k_off, k_len, causal=True)
    v[33 * 50 + 20, 0, 9] = INF
    v[34 * 50 + 49] = math.nan  # past what is filled
    got, gl = tokens.attention(ctx, q, k, v, q_off, k_off, k_len, causal=True)
    other = torch.arange(70) != 33
    assert torch.isnan(got[33].float()).all() and torch.isnan(gl[:, 33]).all()
    assert torch.equal(got.cpu()[other], want.cpu()[other]) and torch.equal(gl.cpu()[:, other], wl.cpu()[:, other])
