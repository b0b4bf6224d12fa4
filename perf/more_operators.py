"""More of the token operators' workloads: a text block's entry (embedding and its gradient), its norms with gate and
residual, and the 8-bit cache that its step writes, reads back and attends to.

A case says which operator it calls and at which sizes; lengths, ids and values are drawn from the seed. ``run``
computes the operators in their plain form (32-bit torch operations; caches padded to the longest) where ``own`` is
false, and calls the package where it is true.
"""
import math

import numpy as np
import torch

own = False


def listed():
    return [
        # one word's phonemes become rows: the smallest call, where latency counts
        {"name": "embed_word", "kind": "embed", "type": "bf16", "t": 37, "vocab": 181, "c": 512, "scale": 1.0, "train": False},
        # a training batch of phonemes: few ids, each of them very often
        {"name": "embed_text_train", "kind": "embed", "type": "f32", "t": 8190, "vocab": 181, "c": 768, "scale": 1.0, "train": True},
        # a training batch of word pieces: most ids of a large table do not occur, the gradient's table is the work
        {"name": "embed_pieces_train", "kind": "embed", "type": "bf16", "t": 16381, "vocab": 32000, "c": 1024, "scale": 32.0, "train": True},
        # between two blocks of one step of 16 requests
        {"name": "norm_step", "kind": "norm", "type": "bf16", "t": 16, "c": 1024, "layer": False, "post": True, "pre": True, "gate": "none", "bias": False,
         "scale": 1.0, "x_scale": 1.0, "train": False},
        # packed texts in float with layer norms and a learned gate for each column
        {"name": "norm_text_train", "kind": "norm", "type": "f32", "t": 4093, "c": 768, "layer": True, "post": True, "pre": True, "gate": "column", "bias": True,
         "scale": 1.0, "x_scale": 1.0, "train": True},
        # a training batch with gates that a projection made for each row
        {"name": "norm_batch_train", "kind": "norm", "type": "bf16", "t": 8192, "c": 2048, "layer": False, "post": True, "pre": True, "gate": "row", "bias": False,
         "scale": 0.5, "x_scale": 1.0, "train": True},
        # wide rows of a prompt, the residual scaled up, no norm behind the block
        {"name": "norm_wide", "kind": "norm", "type": "bf16", "t": 2050, "c": 5120, "layer": True, "post": False, "pre": True, "gate": "column", "bias": True,
         "scale": 1.0, "x_scale": 1.25, "train": False},
        # one new token for each of many requests goes into the cache (and comes back, as a check of it does)
        {"name": "store_step", "kind": "store", "type": "bf16", "docs": 48, "slot": 4096, "rmin": 1, "rmax": 1, "h": 4, "d": 128},
        # the keys and values of a batch of prompts are written, and read back for the attention of a whole prompt
        {"name": "store_text", "kind": "store", "type": "bf16", "docs": 32, "slot": 1024, "rmin": 77, "rmax": 1000, "h": 12, "d": 64},
        # one new token for each of many requests over its own slot
        {"name": "attend_step", "kind": "attend", "type": "bf16", "docs": 48, "slot": 4096, "lmin": 90, "rmin": 1, "rmax": 1, "hq": 16, "hkv": 4, "d": 128,
         "prefix": False, "cap": 0.0, "bias": False},
        # one new token of one request over a long cache, in float, with a bias that falls with distance
        {"name": "attend_one", "kind": "attend", "type": "f32", "docs": 1, "slot": 6001, "lmin": 5999, "rmin": 1, "rmax": 1, "hq": 12, "hkv": 12, "d": 64,
         "prefix": False, "cap": 0.0, "bias": True},
        # pieces of new text behind caches that are filled already, a voice prompt that every token sees, capped scores
        {"name": "attend_piece", "kind": "attend", "type": "bf16", "docs": 5, "slot": 4100, "lmin": 1500, "rmin": 90, "rmax": 301, "hq": 16, "hkv": 4, "d": 128,
         "prefix": True, "cap": 30.0, "bias": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["embed", "embed", "norm", "norm", "norm", "store", "store", "attend", "attend", "attend", "piece"])
    ty = rng.choice(["bf16", "bf16", "f32"])
    if kind == "embed":
        c = rng.choice([128, 512, 640, 768, 1021, 1024])
        return {"kind": "embed", "type": ty, "t": _log(rng, 1, 8190 if ty == "f32" else 16381), "vocab": _log(rng, 30, 32000), "c": c, "scale": rng.choice([1.0, round(c ** 0.5, 3)]),
                "train": rng.random() < 0.7}
    if kind == "norm":
        c = rng.choice([256, 512, 768, 1000, 1021, 1024, 1536, 2048, 4096, 5120])
        post, pre = rng.choice([(True, True), (True, True), (False, True), (True, False)])
        return {"kind": "norm", "type": ty, "t": _log(rng, 1, max(1, (1 << 24) // c // (2 if ty == "f32" else 1))), "c": c, "layer": rng.random() < 0.5, "post": post,
                "pre": pre, "gate": rng.choice(["none", "column", "row"]), "bias": rng.random() < 0.5, "scale": rng.choice([1.0, 0.5]),
                "x_scale": rng.choice([1.0, 1.25]), "train": rng.random() < 0.6}
    if kind == "store":
        docs, slot, h, d = _log(rng, 1, 64), _log(rng, 16, 4096), rng.choice([1, 2, 4, 8, 12]), rng.choice([40, 64, 64, 96, 128])
        rmax = min(rng.choice([1, 4, slot]), 12_000_000 // (docs * h * d))
        return {"kind": "store", "type": ty, "docs": docs, "slot": slot, "rmin": rng.randint(1 if docs < 8 else 0, rmax), "rmax": rmax, "h": h, "d": d}
    cap, bias = rng.choice([0.0, 0.0, 30.0]), rng.random() < 0.3
    if kind == "attend":
        hkv, g = rng.choice([(4, 4), (12, 1), (1, 8), (2, 7)])
        slot, d = _log(rng, 64, 8192), rng.choice([40, 64, 96, 128, 128])
        return {"kind": "attend", "type": ty, "docs": _log(rng, 1, max(1, min(128, 100_000_000 // (slot * hkv * d)))), "slot": slot, "lmin": rng.randint(1, slot),
                "rmin": 1, "rmax": rng.choice([1, 1, 1, 4]), "hq": hkv * g, "hkv": hkv, "d": d, "prefix": rng.random() < 0.2, "cap": cap, "bias": bias}
    hkv, g = rng.choice([(4, 4), (12, 1), (2, 7)])
    slot = _log(rng, 300, 4096)
    rmax = _log(rng, 8, 256)
    return {"kind": "attend", "type": ty, "docs": rng.randint(1, 5), "slot": slot, "lmin": rng.randint(slot // 2, slot), "rmin": rng.randint(1, rmax), "rmax": rmax,
            "hq": hkv * g, "hkv": hkv, "d": rng.choice([64, 128]), "prefix": rng.random() < 0.4, "cap": cap, "bias": bias}


# ─── inputs ──────────────────────────────────────────────────────────────────

def _type(case):
    return torch.float32 if case["type"] == "f32" else torch.bfloat16


def _ids(case, seed):
    """Ids as texts have them (the n-th most frequent about 1 / n as often as the first), some places of padding."""
    g = np.random.default_rng([seed, 3])
    p = 1.0 / (np.arange(case["vocab"]) + 2.0)
    ids = g.permutation(case["vocab"])[np.searchsorted(np.cumsum(p / p.sum()), g.random(case["t"])).clip(max=case["vocab"] - 1)]
    ids[g.random(case["t"]) < 0.03] = -1
    return ids


def _lengths(case, seed):
    """Every request's new rows, filled keys (the new ones among them) and prefix, as the seed draws them."""
    g = np.random.default_rng([seed, 4])
    n, slot = case["docs"], case["slot"]
    lq = np.random.default_rng([case["rmin"], case["rmax"], n]).integers(case["rmin"], case["rmax"] + 1, n)  # a case's total is its own
    lq = np.minimum(g.permutation(lq), slot)
    low = np.maximum(lq, min(case.get("lmin", 1), slot))
    lk = g.integers(low, slot + 1)
    prefix = g.integers(0, np.maximum(lk // 3, 1) + 1) if case.get("prefix") else None
    return lq, lk, prefix


def _wide(d):
    return (d + 15) // 16 * 16


def _coded(x):
    """A cache's codes and scales of float rows (rows, heads, width): largest magnitude 127, nearest code, ties to the even one."""
    s = (x.double().abs().amax(-1) / 127.0).float().clamp(min=2.0 ** -126)
    return torch.round(x.double() / s.double()[..., None]).to(torch.int8), s


def prepare(case, seed):
    dev = "cuda"
    gen = torch.Generator(dev).manual_seed(seed * 7919 + 31)
    ty = _type(case)

    def normal(*shape, std=1.0, to=None):
        return (torch.randn(shape, generator=gen, device=dev) * std).to(to or ty)

    def ints(a):
        return torch.tensor(np.asarray(a), dtype=torch.int32, device=dev)

    if case["kind"] == "embed":
        s = {"case": case, "table": normal(case["vocab"], case["c"], std=0.5), "ids": ints(_ids(case, seed))}
        if case["train"]:
            s["dy"] = normal(case["t"], case["c"], std=0.01)
        return s
    if case["kind"] == "norm":
        t, c = case["t"], case["c"]
        loud = 1.0 + 20.0 * (torch.rand(c, generator=gen, device=dev) < 0.01).float()  # a residual stream has columns that stand out
        s = {"case": case, "x": ((torch.randn((t, c), generator=gen, device=dev) + 0.1) * loud).to(ty), "z": normal(t, c, std=0.7)}
        vec = lambda mid, std: (mid + torch.randn(c, generator=gen, device=dev) * std).to(ty)  # noqa: E731
        s["post"] = (vec(1.0, 0.2), vec(0.0, 0.1) if case["bias"] else None) if case["post"] else None
        s["pre"] = (vec(1.0, 0.2), vec(0.0, 0.1) if case["bias"] else None) if case["pre"] else None
        s["gate"] = {"none": None, "column": vec(0.5, 0.3), "row": torch.sigmoid(torch.randn((t, c), generator=gen, device=dev)).to(ty)}[case["gate"]]
        if case["train"]:
            s["dr"] = normal(t, c, std=0.02)
            s["dy"] = normal(t, c, std=0.05) if case["pre"] else None
        return s
    lq, lk, prefix = _lengths(case, seed)
    n, slot, d = case["docs"], case["slot"], case["d"]
    tq, tk = int(lq.sum()), n * slot
    s = {"case": case, "q_off": ints(np.concatenate([[0], np.cumsum(lq)])), "k_off": ints(np.arange(n + 1) * slot), "k_len": ints(lk), "lq": int(lq.max()),
         "lk": int(lk.max())}
    if case["kind"] == "store":
        h = case["h"]
        s["k"], s["v"] = normal(tq, 3, h, d).unbind(1)[1:]  # two parts of a fused projection's rows
        s["cache"] = tuple(torch.zeros(tk, h, _wide(d), dtype=torch.int8, device=dev) for _ in range(2)) + tuple(torch.zeros(h, tk, device=dev) for _ in range(2))
        return s
    hq, hkv = case["hq"], case["hkv"]
    s["q"] = normal(tq, hq, d)
    codes, scales = [], []
    for std in (1.0, 0.8):
        c, f = _coded(normal(tk, hkv, d, std=std, to=torch.float32))
        codes.append(torch.nn.functional.pad(c, (0, _wide(d) - d)))
        scales.append(f.t().contiguous())
    s["cache"] = (*codes, *scales)
    s["prefix"] = None if prefix is None else ints(prefix)
    s["slopes"] = 2.0 ** (-8.0 * torch.arange(1, hq + 1, device=dev) / hq) if case["bias"] else None
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
        return {"embed": _own_embed, "norm": _own_norm, "store": _own_store, "attend": _own_attend}[kind](s)
    return {"embed": _plain_embed, "norm": _plain_norm, "store": _plain_store, "attend": _plain_attend}[kind](s)


def _own_embed(s):
    from brosoundml_amd import tokens
    c = s["case"]
    y = tokens.embedding(_ctx(), s["table"], s["ids"], scale=c["scale"])
    if not c["train"]:
        return {"y": y}
    return {"y": y, "dtable": tokens.embedding_bwd(_ctx(), s["ids"], s["dy"], c["vocab"], scale=c["scale"])}


def _own_norm(s):
    from brosoundml_amd import tokens
    c = s["case"]
    rule = dict(gate=s["gate"], post=s["post"], pre=s["pre"], kind="layer" if c["layer"] else "rms", eps=1e-5, scale=c["scale"], x_scale=c["x_scale"])
    if not c["train"]:
        r, y = tokens.residual_norm(_ctx(), s["x"], s["z"], **rule)
        return {"r": r, "y": y}
    r, y, stats = tokens.residual_norm(_ctx(), s["x"], s["z"], keep=True, **rule)
    dx, dz, dgate, dpost, dpre = tokens.residual_norm_bwd(_ctx(), s["x"], s["z"], s["dr"], s["dy"], stats, **rule)
    return {"r": r, "y": y, "dx": dx, "dz": dz, "dgate": dgate, "dpost": dpost, "dpre": dpre}


def _own_store(s):
    from brosoundml_amd import tokens
    cache = tokens.Cache(*s["cache"])
    tokens.cache_write(_ctx(), s["k"], s["v"], cache, s["q_off"], s["k_off"], s["k_len"])
    k, v = tokens.cache_read(_ctx(), cache, s["q_off"], s["k_off"], s["k_len"], rows=s["k"].shape[0], width=s["case"]["d"], dtype=s["k"].dtype)
    return {"k": k, "v": v, "k_scale": cache.k_scale, "v_scale": cache.v_scale}


def _own_attend(s):
    from brosoundml_amd import tokens
    o, lse = tokens.cache_attention(_ctx(), s["q"], tokens.Cache(*s["cache"]), s["q_off"], s["k_off"], s["k_len"], causal=True, prefix=s["prefix"],
                                    cap=s["case"]["cap"], slopes=s["slopes"])
    return {"o": o, "lse": lse}


def _plain_embed(s):
    c, ids = s["case"], s["ids"].long()
    has = (ids >= 0) & (ids < c["vocab"])
    at = torch.where(has, ids, torch.zeros_like(ids))
    y = torch.where(has[:, None], s["table"][at].float() * c["scale"], 0.0).to(s["table"].dtype)
    if not c["train"]:
        return {"y": y}
    dy = torch.where(has[:, None], s["dy"].float(), 0.0)
    return {"y": y, "dtable": torch.zeros(c["vocab"], c["c"], device=ids.device).index_add_(0, at, dy).mul_(c["scale"])}


def _plain_centred(u, layer):
    """u normalised along its rows, and one over its deviation."""
    if layer:
        u = u - u.mean(1, keepdim=True)
    rs = torch.rsqrt((u * u).mean(1, keepdim=True) + 1e-5)
    return u * rs, rs


def _plain_back(e, hat, rs, layer):
    """The normalisation's gradient from that of its normalised rows."""
    d = e - hat * (e * hat).mean(1, keepdim=True)
    return rs * (d - e.mean(1, keepdim=True) if layer else d)


def _plain_norm(s):
    c, ty = s["case"], s["x"].dtype
    a, layer = c["scale"], c["layer"]
    x, u = s["x"].float(), s["z"].float()
    (w1, b1), (w2, b2) = ([None if v is None else v.float() for v in p or (None, None)] for p in (s["post"], s["pre"]))
    g = None if s["gate"] is None else s["gate"].float()
    if s["post"]:
        zh, s1 = _plain_centred(u, layer)
        u = zh * w1 if b1 is None else zh * w1 + b1
    r = x * c["x_scale"] + (u if g is None else g * u) * a
    y = None
    if s["pre"]:
        rh, s2 = _plain_centred(r, layer)
        y = (rh * w2 if b2 is None else rh * w2 + b2).to(ty)
    res = {"r": r.to(ty), "y": y}
    if not c["train"]:
        return res
    top, dpre, dpost, dgate = s["dr"].float(), None, None, None
    if s["pre"]:
        dy = s["dy"].float()
        top = top + _plain_back(dy * w2, rh, s2, layer)
        dpre = ((dy * rh).sum(0), None if b2 is None else dy.sum(0))
    du = top * a if g is None else g * top * a
    if g is not None:
        dgate = u * top * a
        dgate = dgate.sum(0) if g.dim() == 1 else dgate.to(ty)
    dz = du
    if s["post"]:
        dpost = ((du * zh).sum(0), None if b1 is None else du.sum(0))
        dz = _plain_back(du * w1, zh, s1, layer)
    res.update(dx=(top * c["x_scale"]).to(ty), dz=dz.to(ty), dgate=dgate, dpost=dpost, dpre=dpre)
    return res


def _plain_store(s):
    d, (kc, vc, ks, vs) = s["case"]["d"], s["cache"]
    q_off = s["q_off"].long()
    rows = torch.arange(s["k"].shape[0], device=kc.device)
    doc = torch.searchsorted(q_off[1:].contiguous(), rows, right=True)
    at = s["k_off"].long()[doc] + s["k_len"][doc] - (q_off[doc + 1] - rows)

    def one(x, codes, scales):
        f = torch.clamp((x.double().abs().amax(-1) / 127.0).float(), min=2.0 ** -126)
        codes[at, :, :d] = torch.round(x.double() / f.double()[..., None]).to(torch.int8)
        scales[:, at] = f.t()
        return (codes[at, :, :d].float() * scales[:, at].t()[..., None]).to(x.dtype)

    return {"k": one(s["k"], kc, ks), "v": one(s["v"], vc, vs), "k_scale": ks, "v_scale": vs}


def _plain_attend(s):
    c, q = s["case"], s["q"]
    hq, hkv, d, n, lq, lk = c["hq"], c["hkv"], c["d"], c["docs"], s["lq"], s["lk"]
    g, dev = hq // hkv, q.device
    q_off, nk = s["q_off"].long(), s["k_len"].long()
    nq = q_off[1:] - q_off[:-1]
    iq, ik = torch.arange(lq, device=dev), torch.arange(lk, device=dev)
    at_q = (q_off[:-1, None] + iq).clamp_(max=q.shape[0] - 1)
    at_k = s["k_off"].long()[:-1, None] + ik
    kc, vc, ks, vs = s["cache"]
    Q = q[at_q].float().view(n, lq, hkv, g, d).permute(0, 2, 3, 1, 4).reshape(n, hkv, g * lq, d)

    def padded(codes, scales):
        return (codes[at_k][..., :d].float() * scales.t()[at_k][..., None]).permute(0, 2, 1, 3).contiguous()

    x = torch.matmul(Q, padded(kc, ks).transpose(2, 3)).view(n, hkv, g, lq, lk).mul_(d ** -0.5)
    pos = iq + (nk - nq)[:, None]
    see = ik <= pos[:, :, None]
    if s["prefix"] is not None:
        see = see | (ik < s["prefix"][:, None])[:, None, :]
    see = see & (ik < nk[:, None])[:, None, :] & (iq < nq[:, None])[:, :, None]
    if c["cap"]:
        x = x.div_(c["cap"]).tanh_().mul_(c["cap"])
    if s["slopes"] is not None:
        x = x - s["slopes"].view(hkv, g, 1, 1) * (ik - pos[:, :, None]).abs().float()[:, None, None]
    x = x.masked_fill_(~see[:, None, None], -math.inf)
    m = x.amax(-1, keepdim=True)
    p = x.sub_(torch.where(m == -math.inf, torch.zeros_like(m), m)).exp_()
    l = p.sum(-1, keepdim=True)
    lse = (m + l.log()).view(n, hq, lq)
    p = p.div_(torch.where(l == 0, torch.ones_like(l), l)).view(n, hkv, g * lq, lk)
    o = torch.matmul(p, padded(vc, vs)).view(n, hq, lq, d)
    rows = torch.arange(q.shape[0], device=dev)
    doc = torch.searchsorted(q_off[1:].contiguous(), rows, right=True)
    at = rows - q_off[doc]
    return {"o": o[doc, :, at].to(q.dtype), "lse": lse[doc, :, at].t().contiguous()}


# ─── work ────────────────────────────────────────────────────────────────────

def work(case):
    e = 4 if case["type"] == "f32" else 2
    if case["kind"] == "embed":
        t, v, c = case["t"], case["vocab"], case["c"]
        p = 1.0 / (np.arange(v) + 2.0)
        used = float((1.0 - (1.0 - 0.97 * p / p.sum()) ** t).sum())  # how many ids occur
        size, ops = 4 * t + e * c * (t + used), t * c
        if case["train"]:
            size, ops = size + e * t * c + 4 * v * c, ops + 2 * t * c
        return {"bytes": int(size), "flops": int(ops)}
    if case["kind"] == "norm":
        n, gate = case["t"] * case["c"], case["gate"] == "row"
        size, ops = e * n * (3 + case["pre"] + gate), 16 * n
        if case["train"]:
            size, ops = size + e * n * (5 + case["pre"] + 2 * gate), ops + 30 * n
        return {"bytes": size, "flops": ops}
    if case["kind"] == "store":
        mean = (min(case["rmin"], case["slot"]) + min(case["rmax"], case["slot"])) / 2
        rows = 2 * case["docs"] * mean * case["h"]  # keys and values: read, coded, and the values that come back
        return {"bytes": int(rows * (2 * e * case["d"] + case["d"] + 4)), "flops": int(rows * case["d"] * 4)}
    hq, hkv, d, docs = case["hq"], case["hkv"], case["d"], case["docs"]
    rows = docs * (case["rmin"] + case["rmax"]) / 2
    keys = docs * (min(case["lmin"], case["slot"]) + case["slot"]) / 2
    return {"bytes": int(keys * hkv * 2 * (d + 4) + 2 * e * rows * hq * d), "flops": int(4 * rows * keys / docs * hq * d)}


# ─── the definitions in 64 bits ──────────────────────────────────────────────

def exact(case, seed):
    s = prepare(case, seed)
    return {"embed": _exact_embed, "norm": _exact_norm, "store": _exact_store, "attend": _exact_attend}[case["kind"]](case, s, seed)


def _exact_embed(case, s, seed):
    ids = _ids(case, seed)
    dev, v, c = s["table"].device, case["vocab"], case["c"]
    y = torch.zeros(case["t"], c, dtype=torch.float64, device=dev)
    real = np.flatnonzero(ids >= 0)
    y[torch.from_numpy(real).to(dev)] = s["table"].double()[torch.from_numpy(ids[real]).to(dev)] * case["scale"]
    if not case["train"]:
        return {"y": y}
    order = real[np.argsort(ids[real], kind="stable")]  # runs of equal ids: differences of the running sum at their ends
    total = torch.cat([torch.zeros(1, c, dtype=torch.float64, device=dev), s["dy"].double()[torch.from_numpy(order).to(dev)].cumsum(0)])
    ends = torch.from_numpy(np.searchsorted(ids[order], np.arange(v + 1))).to(dev)
    return {"y": y, "dtable": (total[ends[1:]] - total[ends[:-1]]) * case["scale"]}


def _exact_norm(case, s, seed):
    f = lambda v: None if v is None else v.double().requires_grad_(case["train"])  # noqa: E731
    x, z, gate = f(s["x"]), f(s["z"]), f(s["gate"])
    post, pre = ([f(v) for v in p] if p else None for p in (s["post"], s["pre"]))

    def normed(u, wb):
        centre = u.mean(1, keepdim=True) if case["layer"] else 0.0
        h = (u - centre) / torch.sqrt(((u - centre) ** 2).mean(1, keepdim=True) + 1e-5) * wb[0]
        return h if wb[1] is None else h + wb[1]

    u = normed(z, post) if post else z
    r = case["x_scale"] * x + case["scale"] * (u if gate is None else gate * u)
    y = normed(r, pre) if pre else None
    out = {"r": r.detach(), "y": None if y is None else y.detach()}
    if not case["train"]:
        return out
    total = (r * s["dr"].double()).sum()
    if y is not None:
        total = total + (y * s["dy"].double()).sum()
    total.backward()
    g = lambda v: None if v is None else v.grad  # noqa: E731
    out.update(dx=g(x), dz=g(z), dgate=g(gate), dpost=tuple(map(g, post)) if post else None, dpre=tuple(map(g, pre)) if pre else None)
    return out


def _exact_store(case, s, seed):
    lq, lk, _ = _lengths(case, seed)
    ends = np.concatenate([[0], np.cumsum(lq)])
    res = {}
    for name, x in (("k", s["k"]), ("v", s["v"])):
        f = (x.double().abs().amax(-1, keepdim=True) / 127).float().double().clamp(min=2.0 ** -126)  # held in 32 bits
        q = x.double() / f
        low = torch.floor(q)
        up = (q - low > 0.5) | ((q - low == 0.5) & (low % 2 != 0))
        res[name] = (low + up.double()) * f
        held = torch.zeros(case["h"], case["docs"] * case["slot"], dtype=torch.float64, device=x.device)
        for i in range(case["docs"]):
            a = i * case["slot"] + int(lk[i]) - int(lq[i])
            held[:, a:a + int(lq[i])] = f[ends[i]:ends[i + 1], :, 0].t()
        res[name + "_scale"] = held
    return res


def _exact_attend(case, s, seed):
    lq, lk, prefix = _lengths(case, seed)
    q, (kc, vc, ks, vs) = s["q"].double(), s["cache"]
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    g, dev = hq // hkv, q.device
    o, lse = torch.zeros_like(q), torch.full((hq, q.shape[0]), -math.inf, dtype=torch.float64, device=dev)
    a = 0
    for i in range(case["docs"]):
        rows, keys, k0 = int(lq[i]), int(lk[i]), i * case["slot"]
        b = a + rows
        K, V = (codes[k0:k0 + keys, :, :d].double() * scales[:, k0:k0 + keys].double().t()[:, :, None] for codes, scales in ((kc, ks), (vc, vs)))
        spot = torch.arange(rows, device=dev)[:, None] + keys - rows
        key = torch.arange(keys, device=dev)[None]
        hide = key > spot
        if prefix is not None:
            hide = hide & (key >= int(prefix[i]))
        for h in range(hq):
            z = q[a:b, h] @ K[:, h // g].t() / math.sqrt(d)
            if case["cap"]:
                z = case["cap"] * torch.tanh(z / case["cap"])
            if s["slopes"] is not None:
                z = z - float(s["slopes"][h]) * (spot - key).abs()
            z = z.masked_fill(hide, -math.inf)
            norm = torch.logsumexp(z, -1)
            lse[h, a:b] = norm
            o[a:b, h] = torch.exp(z - norm[:, None]) @ V[:, h // g]
        a = b
    return {"o": o, "lse": lse}
