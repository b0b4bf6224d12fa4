"""The token operators' workloads: attention over packed utterances, the projections with low-rank adapters of
many voices, and dropout, as the text front end of the decoder and the decoder's own style projection run them.

A case says which operator it calls and at which sizes; lengths and adapter choices are drawn from the seed.
``run`` computes the operators in their plain form (32-bit torch operations on utterances padded to the longest)
where ``own`` is false, and calls the package where it is true.
"""
import math

import numpy as np
import torch

own = False

STYLE_C = [514, 1024] + [1090, 1024] * 3 + [1090, 512] + [256] * 24 + [128] * 24  # channels of the decoder's AdaIN units


def listed():
    return [
        # one word through one attention layer: the smallest call, where latency counts
        {"name": "attn_word", "kind": "attn", "type": "bf16", "docs": 1, "lmin": 37, "lmax": 37, "pad": 0, "hq": 8, "hkv": 8,
         "d": 64, "causal": False, "prefix": False, "cap": 0.0, "bias": False, "train": False},
        # a training batch of phoneme sequences packed without padding, every token sees its own utterance
        {"name": "attn_text_train", "kind": "attn", "type": "bf16", "docs": 32, "lmin": 20, "lmax": 510, "pad": 19, "hq": 12, "hkv": 12,
         "d": 64, "causal": False, "prefix": False, "cap": 0.0, "bias": False, "train": True},
        # the same in float, as the decoder's tensors are, with a bias that falls with distance
        {"name": "attn_text_float_train", "kind": "attn", "type": "f32", "docs": 7, "lmin": 11, "lmax": 333, "pad": 5, "hq": 8, "hkv": 8,
         "d": 64, "causal": False, "prefix": False, "cap": 0.0, "bias": True, "train": True},
        # long texts with a voice prompt that every token sees, shared key heads, capped scores
        {"name": "attn_prefix_cap", "kind": "attn", "type": "bf16", "docs": 4, "lmin": 1900, "lmax": 4099, "pad": 0, "hq": 16, "hkv": 4,
         "d": 128, "causal": True, "prefix": True, "cap": 30.0, "bias": False, "train": False},
        # one long recording, causal: the largest call
        {"name": "attn_long_train", "kind": "attn", "type": "bf16", "docs": 1, "lmin": 8192, "lmax": 8192, "pad": 0, "hq": 16, "hkv": 4,
         "d": 128, "causal": True, "prefix": False, "cap": 0.0, "bias": False, "train": True},
        # one new token for each of many requests, each over its own cache slot
        {"name": "attn_step", "kind": "step", "type": "bf16", "docs": 48, "slot": 4096, "lmin": 90, "hq": 16, "hkv": 4,
         "d": 128, "rows": 1, "cap": 0.0, "bias": False},
        # one new token of one request over a long cache, in float
        {"name": "attn_step_one", "kind": "step", "type": "f32", "docs": 1, "slot": 6001, "lmin": 5999, "hq": 12, "hkv": 12,
         "d": 64, "rows": 1, "cap": 0.0, "bias": True},
        # one step of a batch of requests, a voice each: fused query, key and value rows
        {"name": "proj_step", "kind": "proj", "type": "bf16", "t": 16, "voices": 12, "in": 1024, "units": "1024,256,256", "rank": 16,
         "bias": False, "p": 0.0, "train": False},
        # packed texts of many voices through the same rows
        {"name": "proj_text", "kind": "proj", "type": "bf16", "t": 4093, "voices": 24, "in": 1024, "units": "1024,1024,1024,1024", "rank": 16,
         "bias": True, "p": 0.0, "train": False},
        # the adapters' training step on packed texts, dropout before the adapters
        {"name": "proj_train", "kind": "proj", "type": "bf16", "t": 8192, "voices": 8, "in": 2048, "units": "2048", "rank": 16,
         "bias": True, "p": 0.1, "train": True},
        # every AdaIN unit's style projection for a batch of utterances in voices of their own
        {"name": "proj_style_train", "kind": "proj", "type": "f32", "t": 32, "voices": 16, "in": 128, "units": "style", "rank": 16,
         "bias": True, "p": 0.0, "train": True},
        # dropout and the residual behind a block's output, a training batch
        {"name": "dropout_text", "kind": "dropout", "type": "bf16", "t": 8191, "c": 2048, "p": 0.1, "residual": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["text", "text", "long", "step", "step", "proj", "proj", "proj_train", "style", "dropout"])
    ty = rng.choice(["bf16", "bf16", "f32"])
    if kind == "text":
        hkv, g = rng.choice([(8, 1), (12, 1), (4, 2), (2, 8), (1, 5)])
        lmax = _log(rng, 8, 512)
        return {"kind": "attn", "type": ty, "docs": _log(rng, 1, 48), "lmin": rng.randint(1, lmax), "lmax": lmax, "pad": rng.choice([0, 0, 13]),
                "hq": hkv * g, "hkv": hkv, "d": rng.choice([40, 64, 64, 96, 128]), "causal": rng.random() < 0.3, "prefix": rng.random() < 0.3,
                "cap": rng.choice([0.0, 0.0, 20.0]), "bias": rng.random() < 0.4, "train": rng.random() < 0.6}
    if kind == "long":
        lmax = _log(rng, 700, 6000)
        return {"kind": "attn", "type": "bf16", "docs": 1 if lmax > 3000 else rng.randint(1, 4), "lmin": max(1, lmax // 2), "lmax": lmax, "pad": 0, "hq": 16,
                "hkv": rng.choice([2, 4, 16]), "d": rng.choice([64, 128]), "causal": rng.random() < 0.8, "prefix": rng.random() < 0.4,
                "cap": rng.choice([0.0, 30.0]), "bias": rng.random() < 0.3, "train": rng.random() < 0.5}
    if kind == "step":
        hkv, g = rng.choice([(4, 4), (12, 1), (1, 8), (2, 7)])
        slot = _log(rng, 64, 8192)
        return {"kind": "step", "type": ty, "docs": _log(rng, 1, max(1, min(128, 200000 // slot))), "slot": slot, "lmin": rng.randint(1, slot), "hq": hkv * g,
                "hkv": hkv, "d": rng.choice([64, 128]), "rows": rng.choice([1, 1, 1, 3]), "cap": rng.choice([0.0, 0.0, 30.0]), "bias": rng.random() < 0.3}
    if kind == "proj":
        w = rng.choice([512, 768, 1024, 2048])
        units = rng.choice(["%d" % w, "%d,%d,%d" % (w, w // 8, w // 8), "%d,%d" % (w, w)])
        return {"kind": "proj", "type": ty, "t": _log(rng, 1, 4096), "voices": _log(rng, 1, 64), "in": w + rng.choice([0, 0, 8]), "units": units,
                "rank": rng.choice([4, 8, 16, 32, 64]), "bias": rng.random() < 0.5, "p": 0.0, "train": False}
    if kind == "proj_train":
        w = rng.choice([512, 768, 1024])
        return {"kind": "proj", "type": ty, "t": _log(rng, 64, 4096), "voices": _log(rng, 1, 32), "in": w, "units": rng.choice(["%d" % w, "%d,%d" % (w, w // 2)]),
                "rank": rng.choice([8, 16, 32]), "bias": rng.random() < 0.5, "p": rng.choice([0.0, 0.05, 0.1]), "train": True}
    if kind == "style":
        return {"kind": "proj", "type": "f32", "t": _log(rng, 1, 64), "voices": _log(rng, 1, 24), "in": 128, "units": "style", "rank": rng.choice([4, 8, 16]),
                "bias": True, "p": 0.0, "train": rng.random() < 0.5}
    return {"kind": "dropout", "type": ty, "t": _log(rng, 1, 8192), "c": rng.choice([512, 768, 1021, 2048]), "p": rng.choice([0.05, 0.1, 0.5]),
            "residual": rng.random() < 0.7}


# ─── inputs ──────────────────────────────────────────────────────────────────

def _type(case):
    return torch.float32 if case["type"] == "f32" else torch.bfloat16


def _lengths(case, seed):
    """Every document's query rows and keys, and its prefix, as the seed draws them."""
    g = np.random.default_rng([seed, 1])
    if case["kind"] == "step":
        lk = g.integers(min(case["lmin"], case["slot"]), case["slot"] + 1, case["docs"])
        return np.full(case["docs"], case["rows"]), lk, None
    same = np.random.default_rng([case["lmin"], case["lmax"], case["docs"]])  # a case's total is its own, the order is the seed's
    lq = g.permutation(same.integers(case["lmin"], case["lmax"] + 1, case["docs"]))
    prefix = g.integers(0, np.maximum(lq // 3, 1) + 1) if case["prefix"] else None
    return lq, lq, prefix


def _unit_sizes(case):
    return [2 * c for c in STYLE_C] if case["units"] == "style" else [int(u) for u in case["units"].split(",")]


def _voices(case, seed):
    """The adapter of every row: runs of one request for texts, a row of its own per request for steps; -1 has none."""
    g = np.random.default_rng([seed, 2])
    t, n = case["t"], case["voices"]
    if t <= 64:
        return g.integers(-1 if n > 1 else 0, n, t).astype(np.int32)
    cuts = np.sort(g.integers(1, t, max(1, min(t // 48, 2 * n))))
    who = g.integers(-1 if n > 1 else 0, n, len(cuts) + 1)
    return np.repeat(who, np.diff(np.concatenate([[0], cuts, [t]]))).astype(np.int32)


def prepare(case, seed):
    dev = "cuda"
    gen = torch.Generator(dev).manual_seed(seed * 7919 + 13)
    ty = _type(case)

    def normal(*shape, std=1.0, to=None):
        return (torch.randn(shape, generator=gen, device=dev) * std).to(to or ty)

    def ints(a):
        return torch.tensor(np.asarray(a), dtype=torch.int32, device=dev)

    if case["kind"] == "dropout":
        s = {"case": case, "x": normal(case["t"], case["c"]), "seed": seed * 1000003 + 17, "offset": seed % 97}
        s["residual"] = normal(case["t"], case["c"]) if case["residual"] else None
        return s
    if case["kind"] == "proj":
        n, t, cin, rank = case["voices"], case["t"], case["in"], case["rank"]
        sizes = _unit_sizes(case)
        units, out = len(sizes), sum(sizes)
        s = {"case": case, "x": normal(t, cin), "w": normal(out, cin, std=cin ** -0.5), "bias": normal(out, std=0.1) if case["bias"] else None,
             "a": normal(n, units * rank, cin, std=cin ** -0.5), "b": normal(n, out, rank, std=0.3 * rank ** -0.5),
             "scale": 0.5 + torch.rand(n, generator=gen, device=dev), "idx": ints(_voices(case, seed)),
             "unit_off": ints(np.concatenate([[0], np.cumsum(sizes)])), "drop": (case["p"], seed * 1000003 + 29, 3) if case["p"] else None}
        if case["train"]:
            s["dy"] = normal(t, out)
        return s
    lq, lk, prefix = _lengths(case, seed)
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    q_off = np.concatenate([[0], np.cumsum(lq)])
    step = case["kind"] == "step"
    tq = int(q_off[-1]) + case.get("pad", 0)
    tk = case["docs"] * case["slot"] if step else tq
    s = {"case": case, "q_off": ints(q_off), "k_off": ints(np.arange(case["docs"] + 1) * case["slot"] if step else q_off),
         "k_len": ints(lk) if step else None, "prefix": None if prefix is None else ints(prefix), "lq": int(lq.max()), "lk": int(lk.max()),
         "slopes": 2.0 ** (-8.0 * torch.arange(1, hq + 1, device=dev) / hq) if case["bias"] else None}
    if step or hq != hkv:
        s["q"], s["k"], s["v"] = normal(tq, hq, d), normal(tk, hkv, d), normal(tk, hkv, d)
    else:  # the three parts of one fused projection's rows
        s["q"], s["k"], s["v"] = normal(tq, 3, hq, d).unbind(1)
    if case.get("train"):
        s["do"] = normal(tq, hq, d)
    return s


# ─── the operators ───────────────────────────────────────────────────────────

_context = None


def _ctx():
    global _context
    if _context is None:
        from brosoundml_amd import native
        _context = native.Context(0)
    return _context


def run(s):
    kind = s["case"]["kind"]
    if own:
        return {"attn": _own_attn, "step": _own_attn, "proj": _own_proj, "dropout": _own_dropout}[kind](s)
    return {"attn": _plain_attn, "step": _plain_attn, "proj": _plain_proj, "dropout": _plain_dropout}[kind](s)


def _own_attn(s):
    from brosoundml_amd import tokens
    c = s["case"]
    mask = dict(causal=c.get("causal", True), prefix=s["prefix"], cap=c["cap"], slopes=s["slopes"])
    o, lse = tokens.attention(_ctx(), s["q"], s["k"], s["v"], s["q_off"], s["k_off"], s["k_len"], **mask)
    if not c.get("train"):
        return {"o": o, "lse": lse}
    dq, dk, dv = tokens.attention_bwd(_ctx(), s["q"], s["k"], s["v"], o, lse, s["do"], s["q_off"], s["k_off"], s["k_len"], **mask)
    return {"o": o, "lse": lse, "dq": dq, "dk": dk, "dv": dv}


def _own_proj(s):
    from brosoundml_amd import tokens
    args = (s["x"], s["w"], s["a"], s["b"], s["scale"], s["idx"], s["unit_off"])
    if "dy" not in s:
        return {"y": tokens.adapter_proj(_ctx(), *args, bias=s["bias"], drop=s["drop"])}
    y, h = tokens.adapter_proj(_ctx(), *args, bias=s["bias"], drop=s["drop"], keep_h=True)
    dx, da, db = tokens.adapter_proj_bwd(_ctx(), *args, h, s["dy"], drop=s["drop"])
    return {"y": y, "dx": dx, "da": da, "db": db}


def _own_dropout(s):
    from brosoundml_amd import tokens
    return {"y": tokens.dropout(_ctx(), s["x"], s["case"]["p"], s["seed"], s["offset"], residual=s["residual"])}


def _plain_attn(s):
    c, q, k, v = s["case"], s["q"], s["k"], s["v"]
    hq, hkv, d, n, lq, lk = c["hq"], c["hkv"], c["d"], c["docs"], s["lq"], s["lk"]
    g, dev = hq // hkv, q.device
    q_off, k_off = s["q_off"].long(), s["k_off"].long()
    nq = q_off[1:] - q_off[:-1]
    nk = k_off[1:] - k_off[:-1] if s["k_len"] is None else s["k_len"].long()
    iq, ik = torch.arange(lq, device=dev), torch.arange(lk, device=dev)
    at_q = (q_off[:-1, None] + iq).clamp_(max=q.shape[0] - 1)
    at_k = (k_off[:-1, None] + ik).clamp_(max=k.shape[0] - 1)

    def padded_q(t):  # (rows, hq, d) -> (n, hkv, g * lq, d)
        return t[at_q].float().view(n, lq, hkv, g, d).permute(0, 2, 3, 1, 4).reshape(n, hkv, g * lq, d)

    def padded_k(t):  # (rows, hkv, d) -> (n, hkv, lk, d)
        return t[at_k].float().permute(0, 2, 1, 3).contiguous()

    Q, K, V = padded_q(q), padded_k(k), padded_k(v)
    pos = iq + (nk - nq)[:, None]                                     # (n, lq)
    see = (ik < nk[:, None])[:, None, :] & (iq < nq[:, None])[:, :, None]
    if c.get("causal", True):
        near = ik <= pos[:, :, None]
        see = see & (near if s["prefix"] is None else near | (ik < s["prefix"][:, None])[:, None, :])
    scale = d ** -0.5
    x = torch.matmul(Q, K.transpose(2, 3)).view(n, hkv, g, lq, lk).mul_(scale)
    if c["cap"]:
        th = x.div_(c["cap"]).tanh_()
        x = th * c["cap"]
    if s["slopes"] is not None:
        x = x - s["slopes"].view(hkv, g, 1, 1) * (ik - pos[:, :, None]).abs().float()[:, None, None]
    x = x.masked_fill_(~see[:, None, None], -math.inf)
    m = x.amax(-1, keepdim=True)
    p = x.sub_(torch.where(m == -math.inf, torch.zeros_like(m), m)).exp_()
    l = p.sum(-1, keepdim=True)
    lse = (m + l.log()).view(n, hq, lq)
    p = p.div_(torch.where(l == 0, torch.ones_like(l), l)).view(n, hkv, g * lq, lk)
    O = torch.matmul(p, V)

    rows = torch.arange(q.shape[0], device=dev)
    doc = torch.searchsorted(q_off[1:].contiguous(), rows, right=True)
    real = doc < n
    doc = doc.clamp_(max=n - 1)
    at = (rows - q_off[doc]).clamp_(max=lq - 1)

    def packed_q(t):  # (n, hkv, g * lq, d) -> (rows, hq, d)
        t = t.view(n, hq, lq, d)[doc, :, at]
        return torch.where(real[:, None, None], t, torch.zeros_like(t)).to(q.dtype)

    res = {"o": packed_q(O), "lse": torch.where(real[:, None], lse[doc, :, at], torch.full_like(lse[0, 0, :1], -math.inf)).t().contiguous()}
    if not c.get("train"):
        return res
    dO = padded_q(s["do"])
    dv = torch.matmul(p.transpose(2, 3), dO)
    ds = torch.matmul(dO, V.transpose(2, 3)).sub_((dO * O).sum(-1, keepdim=True)).mul_(p)
    if c["cap"]:
        ds = ds.mul_((1.0 - th * th).view_as(ds))
    ds = ds.mul_(scale)
    rows_k = torch.arange(k.shape[0], device=dev)
    doc_k = torch.searchsorted(k_off[1:].contiguous(), rows_k, right=True)
    doc_c = doc_k.clamp(max=n - 1)
    at_c = rows_k - k_off[doc_c]
    real_k = (doc_k < n) & (at_c < nk[doc_c])
    at_c = at_c.clamp_(max=lk - 1)

    def packed_k(t):
        t = t[doc_c, :, at_c]
        return torch.where(real_k[:, None, None], t, torch.zeros_like(t)).to(q.dtype)

    res["dq"] = packed_q(torch.matmul(ds, K))
    res["dk"] = packed_k(torch.matmul(ds.transpose(2, 3), Q))
    res["dv"] = packed_k(dv)
    return res


def _plain_kept(rows, cols, drop, dev):
    """0 where dropped, 1 / (1 - p) where kept: the halves of Philox4x32-10's words (column / 8, row, offset) under the seed."""
    p, seed, offset = drop
    thr = int(math.floor(p * 65536 + 0.5))
    c0 = torch.arange((cols + 7) // 8, device=dev).expand(rows, -1)
    c1 = torch.arange(rows, device=dev)[:, None].expand_as(c0)
    c2, c3 = torch.full_like(c0, offset & 0xFFFFFFFF), torch.full_like(c0, offset >> 32 & 0xFFFFFFFF)
    k0, k1 = seed & 0xFFFFFFFF, seed >> 32 & 0xFFFFFFFF

    def mul(a, m):  # the high and the low 32 bits of a product of two 32-bit numbers
        hi = (a * (m >> 16) + ((a * (m & 0xFFFF)) >> 16)) >> 16
        return hi, (a * m) & 0xFFFFFFFF

    for _ in range(10):
        h0, l0 = mul(c0, 0xD2511F53)
        h1, l1 = mul(c2, 0xCD9E8D57)
        c0, c1, c2, c3 = h1 ^ c1 ^ k0, l1, h0 ^ c3 ^ k1, l0
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    words = torch.stack([c0, c1, c2, c3], -1)
    halves = torch.stack([words & 0xFFFF, words >> 16], -1).view(rows, -1)[:, :cols]
    return (halves >= thr).float() * (65536.0 / (65536 - thr))


def _plain_dropout(s):
    x, c = s["x"], s["case"]
    y = x.float() * _plain_kept(*x.shape, (c["p"], s["seed"], s["offset"]), x.device)
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return {"y": y.to(x.dtype)}


def _plain_proj(s):
    c, ty = s["case"], s["x"].dtype
    x, w, a, b, scale = s["x"].float(), s["w"].float(), s["a"].float(), s["b"].float(), s["scale"]
    t, cin = x.shape
    n, rank, out = c["voices"], c["rank"], w.shape[0]
    units = a.shape[1] // rank
    idx = s["idx"].long()
    has = idx >= 0
    who = idx.clamp(min=0)
    unit = torch.searchsorted(s["unit_off"][1:].long(), torch.arange(out, device=x.device), right=True)
    kept = _plain_kept(t, cin, s["drop"], x.device) if s["drop"] else None
    xd = x * kept if kept is not None else x
    sc = torch.where(has, scale[who], torch.zeros_like(scale[who]))
    few = t * rank <= n * units * rank  # few rows: every row fetches its adapter; else all adapters, then every row its own
    y = torch.matmul(x, w.t())
    if s["bias"] is not None:
        y = y + s["bias"].float()
    mine = (idx[:, None] == torch.arange(n, device=x.device)).float()[:, :, None]
    if few:
        ra, rb = a[who], b[who]
        h = torch.matmul(ra, xd[:, :, None])[:, :, 0] * has[:, None]
        hu = h.view(t, units, rank)[:, unit]                               # (t, out, rank)
        y = y + sc[:, None] * (rb * hu).sum(-1)
    else:
        h = (torch.matmul(xd, a.view(n * units * rank, cin).t()).view(t, n, units * rank) * mine).view(t, -1)
        own_unit = (unit[:, None] == torch.arange(units, device=x.device)).float()
        wide = (b[:, :, None, :] * own_unit[None, :, :, None]).permute(0, 2, 3, 1).reshape(n * units * rank, out)
        y = y + torch.matmul(h * sc[:, None], wide)
    res = {"y": y.to(ty)}
    if not c["train"]:
        return res
    dy = s["dy"].float()
    if few:
        part = torch.zeros(t, units, rank, device=x.device).index_add_(1, unit, rb * dy[:, :, None])
        dh = part.view(t, -1) * sc[:, None]
        low = torch.matmul(dh[:, None, :], ra)[:, 0]
        da = torch.zeros_like(a).index_add_(0, who, dh[:, :, None] * xd[:, None, :])
        db = torch.zeros_like(b).index_add_(0, who, (sc[:, None] * dy)[:, :, None] * hu)
    else:
        dh = (torch.matmul(dy, wide.t()).view(t, n, units * rank) * mine * sc[:, None, None]).view(t, -1)
        low = torch.matmul(dh, a.view(n * units * rank, cin))
        da = torch.matmul(dh.t(), xd).view_as(a)
        db = torch.matmul((h * sc[:, None]).t(), dy).view(n, units, rank, out)
        db = (db * own_unit.t()[None, :, None, :]).sum(1).transpose(1, 2).contiguous()
    if kept is not None:
        low = low * kept
    res.update(dx=(torch.matmul(dy, w) + low).to(ty), da=da, db=db)
    return res


# ─── work ────────────────────────────────────────────────────────────────────

def work(case):
    e = 4 if case["type"] == "f32" else 2
    if case["kind"] == "dropout":
        return {"bytes": e * case["t"] * case["c"] * (3 if case["residual"] else 2), "flops": 2 * case["t"] * case["c"]}
    if case["kind"] == "proj":
        t, n, cin, r = case["t"], case["voices"], case["in"], case["rank"]
        sizes = _unit_sizes(case)
        out, units = sum(sizes), len(sizes)
        used = min(t, n) if t <= 64 else n
        low = used * r * (units * cin + out)
        size = e * (t * cin + out * cin + t * out + low + (out if case["bias"] else 0))
        ops = 2 * t * cin * out + 2 * t * r * (units * cin + out)
        if case["train"]:  # forward, input grad and the two adapter grads (float)
            size += e * (t * out + t * cin) + 4 * n * r * (units * cin + out)
            ops += 2 * t * cin * out + 4 * t * r * (units * cin + out)
        return {"bytes": size, "flops": ops}
    hq, hkv, d, docs = case["hq"], case["hkv"], case["d"], case["docs"]
    if case["kind"] == "step":
        mean = (case["lmin"] + case["slot"]) / 2
        pairs, rows, keys = docs * case["rows"] * mean, docs * case["rows"], docs * mean
    else:
        lo, hi = case["lmin"], case["lmax"]
        mean, square = (lo + hi) / 2, (lo * lo + lo * hi + hi * hi) / 3
        pairs, rows, keys = docs * square * (0.5 if case["causal"] else 1.0), docs * mean, docs * mean
    size, ops = e * d * (2 * rows * hq + 2 * keys * hkv), 4 * pairs * hq * d
    if case.get("train"):
        size += e * d * (2 * rows * hq + 2 * keys * hkv)
        ops += 10 * pairs * hq * d
    return {"bytes": int(size), "flops": int(ops)}


# ─── the definitions in 64 bits ──────────────────────────────────────────────

def exact(case, seed):
    s = prepare(case, seed)
    return {"attn": _exact_attn, "step": _exact_attn, "proj": _exact_proj, "dropout": _exact_dropout}[case["kind"]](case, s, seed)


def _exact_attn(case, s, seed):
    lq, lk, prefix = _lengths(case, seed)
    q, k, v = (s[x].double() for x in "qkv")
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    g, causal = hq // hkv, case.get("causal", True)
    o, lse = torch.zeros_like(q), torch.full((hq, q.shape[0]), -math.inf, dtype=torch.float64, device=q.device)
    train = bool(case.get("train"))
    if train:
        do, dq, dk, dv = s["do"].double(), torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    qs = np.concatenate([[0], np.cumsum(lq)])
    for i in range(case["docs"]):
        a, b = int(qs[i]), int(qs[i + 1])
        k0 = i * case["slot"] if case["kind"] == "step" else a
        k1 = k0 + int(lk[i])
        spot = torch.arange(b - a, device=q.device)[:, None] + (k1 - k0) - (b - a)
        key = torch.arange(k1 - k0, device=q.device)[None]
        hide = torch.zeros(b - a, k1 - k0, dtype=torch.bool, device=q.device)
        if causal:
            hide = key > spot
            if prefix is not None:
                hide = hide & (key >= int(prefix[i]))
        together = max(1, min(hq, (1 << 28) // max(1, (b - a) * (k1 - k0))))
        for h0 in range(0, hq, together):
            hs = torch.arange(h0, min(hq, h0 + together), device=q.device)
            Q, K, V = q[a:b, hs].transpose(0, 1), k[k0:k1, hs // g].transpose(0, 1), v[k0:k1, hs // g].transpose(0, 1)
            z = Q @ K.transpose(1, 2) / math.sqrt(d)
            slope = torch.ones_like(z[:, :1, :1])
            if case["cap"]:
                t = torch.tanh(z / case["cap"])
                z, slope = case["cap"] * t, 1 - t * t
            if s["slopes"] is not None:
                z = z - s["slopes"].double()[hs][:, None, None] * (spot - key).abs()
            z = z.masked_fill(hide, -math.inf)
            n = torch.logsumexp(z, -1, keepdim=True)
            p = torch.where(n == -math.inf, torch.zeros_like(z), torch.exp(z - n))
            out = p @ V
            o[a:b, hs], lse[hs, a:b] = out.transpose(0, 1), n[:, :, 0]
            if train:
                G = do[a:b, hs].transpose(0, 1)
                z = p * (G @ V.transpose(1, 2) - (G * out).sum(-1, keepdim=True)) * slope / math.sqrt(d)
                dq[a:b, hs] = (z @ K).transpose(0, 1)
                dk[k0:k1].index_add_(1, hs // g, (z.transpose(1, 2) @ Q).transpose(0, 1))
                dv[k0:k1].index_add_(1, hs // g, (p.transpose(1, 2) @ G).transpose(0, 1))
    return {"o": o, "lse": lse, "dq": dq, "dk": dk, "dv": dv} if train else {"o": o, "lse": lse}


def _exact_kept(rows, cols, p, seed, offset, dev):
    low = np.uint64(0xFFFFFFFF)
    thr = int(math.floor(p * 65536 + 0.5))
    x = np.zeros((4, rows, (cols + 7) // 8), np.uint64)
    x[0] += np.arange(x.shape[2], dtype=np.uint64)
    x[1] += np.arange(rows, dtype=np.uint64)[:, None]
    x[2] += np.uint64(offset % 2 ** 32)
    x[3] += np.uint64(offset // 2 ** 32)
    for r in range(10):
        key = [(seed % 2 ** 32 + r * 0x9E3779B9) % 2 ** 32, (seed // 2 ** 32 + r * 0xBB67AE85) % 2 ** 32]
        u, w = x[0] * np.uint64(0xD2511F53), x[2] * np.uint64(0xCD9E8D57)
        x = np.stack([(w >> np.uint64(32)) ^ x[1] ^ np.uint64(key[0]), w & low, (u >> np.uint64(32)) ^ x[3] ^ np.uint64(key[1]), u & low])
    bits = np.ascontiguousarray(x.transpose(1, 2, 0).astype("<u4")).view("<u2").reshape(rows, -1)[:, :cols]
    return torch.from_numpy(np.where(bits < thr, 0.0, 65536 / (65536 - thr))).to(dev)


def _exact_dropout(case, s, seed):
    y = s["x"].double() * _exact_kept(*s["x"].shape, case["p"], s["seed"], s["offset"], s["x"].device)
    return {"y": y if s["residual"] is None else y + s["residual"].double()}


def _exact_proj(case, s, seed):
    x, w, a, b = (s[i].double() for i in ("x", "w", "a", "b"))
    rank, who = case["rank"], _voices(case, seed)
    edges = np.concatenate([[0], np.cumsum(_unit_sizes(case))])
    y = x @ w.t()
    if s["bias"] is not None:
        y += s["bias"].double()
    kept = _exact_kept(*x.shape, *s["drop"], x.device) if s["drop"] else torch.ones_like(x)
    xd = x * kept
    if case["train"]:
        dy, da, db = s["dy"].double(), torch.zeros_like(a), torch.zeros_like(b)
        dx = dy @ w
    for v in np.unique(who[who >= 0]):
        rows = torch.from_numpy(np.flatnonzero(who == v)).to(x.device)
        f = float(s["scale"][int(v)])
        X = xd[rows]
        for u in range(len(edges) - 1):
            e0, e1, A, B = int(edges[u]), int(edges[u + 1]), a[v, u * rank:(u + 1) * rank], b[v, int(edges[u]):int(edges[u + 1])]
            h = X @ A.t()
            y[rows, e0:e1] += f * (h @ B.t())
            if case["train"]:
                G = f * dy[rows, e0:e1]
                dx[rows] += (G @ B @ A) * kept[rows]
                da[v, u * rank:(u + 1) * rank] = (G @ B).t() @ X
                db[v, e0:e1] = G.t() @ h
    return {"y": y, "dx": dx, "da": da, "db": db} if case["train"] else {"y": y}
