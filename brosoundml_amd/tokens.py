"""Token operators on torch tensors: attention over packed documents and over
a cache in 8 bits, the projection with low-rank adapters chosen per row,
dropout, embedding, and the norms around a block with gate and residual (the
last section of kdec.h). Each call checks its tensors, allocates what it returns
and makes one C ABI call on the context's stream; nothing synchronises. A
tensor made on another stream has to be ordered before the context's by the
caller, as for every call of the library.

The calls make no autograd graph: a gradient is its own call. So a tensor that
requires grad is refused where grad mode is on; pass ``t.detach()``, or call
under ``torch.no_grad()`` or from an autograd function.

Tensors are float32 or bfloat16 (one type per call), on the context's device;
offsets and adapter choices are int32 tensors there. Errors are
``native.KdecError`` (what the library refuses) and ``ValueError`` (tensors
that do not fit each other)."""
from __future__ import annotations

from typing import NamedTuple

import torch

from .native import Context

try:  # the current stream's address without an object around it
    from torch._C import _cuda_getCurrentRawStream as _raw_stream
except ImportError:
    def _raw_stream(device):
        return torch.cuda.current_stream(device).cuda_stream

_INT_MAX = 0x7FFFFFFF
_TYPES = {torch.float32: 0, torch.bfloat16: 1}


# A single token's kernels take a few microseconds, about what these checks
# do: each reads what it needs of a tensor once, and forms no message that it
# does not raise. Sizes that become ints of the C ABI are checked together, by
# their bits: where one is past 2^31 - 1, so is (a | b).

def _fail(what):
    raise ValueError("brosoundml: " + what)


def _large():
    _fail("sizes past 2^31 - 1: more than the C ABI's ints hold")


def _no_graph(x):
    if x.requires_grad and torch.is_grad_enabled():
        _fail("a tensor requires grad, and these calls make no autograd graph: detach it or call under torch.no_grad()")


def _dtype(ctx, x, *others):
    """The C ABI's type of x, which the others must share, all on the context's device."""
    ty, dev = x.dtype, ctx.device
    if ty not in _TYPES:
        _fail("tensors must be float32 or bfloat16")
    if x.get_device() != dev:
        _fail("tensors must be on the context's HIP device")
    if x.requires_grad:
        _no_graph(x)
    for t in others:
        if t.requires_grad:
            _no_graph(t)
        if t.dtype != ty or t.get_device() != dev:
            _fail("tensors must share one type and device")
    return _TYPES[ty]


def _ints(ctx, x, n, what):
    """Address of an int32 tensor of n values on the device (None passes)."""
    if x is None:
        return None
    if x.dtype != torch.int32 or x.get_device() != ctx.device or x.numel() != n or not x.is_contiguous():
        _fail(f"{what} must hold {n} contiguous int32 values on the device")
    return x.data_ptr()


def _floats(ctx, x, shape, what):
    if x is None:
        return None
    if x.dtype != torch.float32 or x.get_device() != ctx.device or x.shape != shape or not x.is_contiguous():
        _fail(f"{what} must be a contiguous float32 tensor of shape {tuple(shape)}")
    if x.requires_grad:
        _no_graph(x)
    return x.data_ptr()


def _heads(x, what):
    """Address, row stride and head stride of a (rows, heads, width) tensor with contiguous width."""
    s = x.stride()
    if len(s) != 3:
        _fail(f"{what} must be (rows, heads, width)")
    if s[2] != 1 and x.shape[2] > 1:
        _fail(f"{what}: the width must be contiguous")
    return x.data_ptr(), s[0], s[1]


def _rows(x, what):
    """Address and row stride of a (rows, columns) tensor with contiguous columns."""
    s = x.stride()
    if len(s) != 2:
        _fail(f"{what} must be (rows, columns)")
    if s[1] != 1 and x.shape[1] > 1:
        _fail(f"{what}: the columns must be contiguous")
    return x.data_ptr(), s[0]


def _whole(x, shape, what):
    if x.shape != shape or not x.is_contiguous():
        _fail(f"{what} must be contiguous, of shape {tuple(shape)}")
    return x.data_ptr()


def _empty(ctx, x, shape, dtype=None):
    """A new tensor of x's type (or dtype) and device that belongs to the context's stream."""
    if _raw_stream(ctx.device) == ctx.stream.cuda_stream:
        return x.new_empty(shape) if dtype is None else x.new_empty(shape, dtype=dtype)
    with torch.cuda.stream(ctx.stream):
        return x.new_empty(shape, dtype=dtype)


def _attn_args(ctx, q, k, v, q_off, k_off, k_len, causal, prefix, scale, cap, slopes):
    dt = _dtype(ctx, q, k, v)
    Q, K, V = _heads(q, "q"), _heads(k, "k"), _heads(v, "v")
    tq, hq, d = q.shape
    tk, hkv, _ = k.shape
    if not (v.shape == k.shape and k.shape[2] == d):
        _fail("k and v must share their shape, and q their width")
    docs = q_off.numel() - 1
    if not (docs >= 0):
        _fail("q_off must hold one offset more than there are documents")
    if (tq | tk | hq | hkv | d | docs) > _INT_MAX:
        _large()
    if k_off is None:
        if not (tq == tk):
            _fail("without k_off the keys are the query rows' own")
        k_off = q_off
    # where / length / mask arguments, in the C ABI's order
    mask = (_ints(ctx, q_off, docs + 1, "q_off"), _ints(ctx, k_off, docs + 1, "k_off"), _ints(ctx, k_len, docs, "k_len"),
            _ints(ctx, prefix, docs, "prefix"), docs, int(causal), _floats(ctx, slopes, (hq,), "slopes"),
            float(d ** -0.5 if scale is None else scale), float(cap), tq, tk, hq, hkv, d)
    return dt, Q, K, V, mask


def attention(ctx: Context, q, k, v, q_off, k_off=None, k_len=None, *, causal=False, prefix=None, scale=None,
              cap=0.0, slopes=None, out=None):
    """Attention of packed documents (kdec_attn_fwd): q (Tq, Hq, D), k and v
    (Tk, Hkv, D) with any row and head strides; document d holds the query
    rows q_off[d]:q_off[d+1] and the keys k_off[d]:k_off[d+1] (the query rows'
    own without k_off), of which the first k_len[d] are filled. ``causal``
    rows see the keys up to their own position, counted from the document's
    end, and its first prefix[d]. ``cap`` caps the scores by cap * tanh(s /
    cap), ``slopes`` (Hq floats) lowers them by slope * distance; ``scale``
    is 1 / sqrt(D) by default. Returns (o, lse): o as q, lse (Hq, Tq) float.
    Single tokens over long caches take a kernel of their own in this call."""
    dt, Q, K, V, mask = _attn_args(ctx, q, k, v, q_off, k_off, k_len, causal, prefix, scale, cap, slopes)
    tq, hq, _ = q.shape
    o = _empty(ctx, q, q.shape) if out is None else out
    lse = _empty(ctx, q, (hq, tq), torch.float32)
    if out is not None and (o.shape != q.shape or o.dtype != q.dtype or o.device != q.device):
        _fail("out must be as q")
    ctx.call("kdec_attn_fwd", dt, *Q, *K, *V, *mask, *_heads(o, "out"), lse.data_ptr())
    return o, lse


def attention_bwd(ctx: Context, q, k, v, o, lse, do, q_off, k_off=None, k_len=None, *, causal=False, prefix=None,
                  scale=None, cap=0.0, slopes=None, dq=None, dk=None, dv=None):
    """The gradients (dq, dk, dv) of ``attention`` from ``do``, with its o and
    lse and the same mask arguments (kdec_attn_bwd). dq, dk and dv may be
    given, for example as the parts of a fused projection's gradient."""
    dt, Q, K, V, mask = _attn_args(ctx, q, k, v, q_off, k_off, k_len, causal, prefix, scale, cap, slopes)
    _dtype(ctx, q, o, do)
    if not (o.shape == q.shape and do.shape == q.shape):
        _fail("o and do must be as q")
    dq = _empty(ctx, q, q.shape) if dq is None else dq
    dk = _empty(ctx, k, k.shape) if dk is None else dk
    dv = _empty(ctx, v, v.shape) if dv is None else dv
    _dtype(ctx, q, dq, dk, dv)
    if not (dq.shape == q.shape and dk.shape == k.shape and dv.shape == v.shape):
        _fail("dq, dk and dv must be as q, k and v")
    ctx.call("kdec_attn_bwd", dt, *Q, *K, *V, *_heads(o, "o"), _floats(ctx, lse, (q.shape[1], q.shape[0]), "lse"),
             *_heads(do, "do"), *mask, *_heads(dq, "dq"), *_heads(dk, "dk"), *_heads(dv, "dv"))
    return dq, dk, dv


def _adapter_args(ctx, x, w, a, b, scale, idx, unit_off):
    t, cin = x.shape
    out = w.shape[0]
    n, units = a.shape[0], unit_off.numel() - 1
    if not (b.dim() == 3 and units >= 1):
        _fail("b must be (adapters, out, rank), unit_off units + 1 offsets")
    rank = b.shape[2]
    if (t | cin | out | n | units | rank) > _INT_MAX:
        _large()
    return (_whole(w, (out, cin), "w"), _whole(a, (n, units * rank, cin), "a"), _whole(b, (n, out, rank), "b"),
            _floats(ctx, scale, (n,), "scale"), _ints(ctx, idx, t, "idx"), _ints(ctx, unit_off, units + 1, "unit_off"), t, cin, out,
            n, units, rank)


def adapter_proj(ctx: Context, x, w, a, b, scale, idx, unit_off, *, bias=None, drop=None, keep_h=False, out=None):
    """x W^T + bias with row t's own low-rank adapter idx[t] beside it
    (kdec_adapter_fwd): x (T, in), w (out, in), a (adapters, units * rank,
    in), b (adapters, out, rank), scale (adapters floats); rows whose idx is
    outside [0, adapters) take none. unit_off (units + 1) cuts the output rows
    into units with adapters of their own. ``drop`` = (p, seed, offset) drops
    inputs of the adapters. Returns y (T, out), and with ``keep_h`` the pair
    (y, h) whose h the backward takes."""
    dt = _dtype(ctx, x, w, a, b)
    X = _rows(x, "x")
    W, A, B, S, I, U, t, cin, cout, n, units, rank = _adapter_args(ctx, x, w, a, b, scale, idx, unit_off)
    p, seed, offset = drop if drop is not None else (0.0, 0, 0)
    y = _empty(ctx, x, (t, cout)) if out is None else out
    h = _empty(ctx, x, (t, units * rank), torch.float32) if keep_h else None
    if not (y.shape == (t, cout)):
        _fail("out must be (T, out)")
    _dtype(ctx, x, y)
    if bias is not None:
        _dtype(ctx, x, bias)
        _whole(bias, (cout,), "bias")
    ctx.call("kdec_adapter_fwd", dt, *X, W, None if bias is None else bias.data_ptr(), A, B, S, I, U, t, cin, cout,
             n, units, rank, p, seed, offset, None if h is None else h.data_ptr(), *_rows(y, "out"))
    return (y, h) if keep_h else y


def adapter_proj_bwd(ctx: Context, x, w, a, b, scale, idx, unit_off, h, dy, *, drop=None, need_dx=True, da=None,
                     db=None, beta=0.0):
    """The gradients (dx, da, db) of ``adapter_proj`` from ``dy`` and its h,
    w and bias frozen (kdec_adapter_bwd). dx is of x's type (None without
    ``need_dx``); da and db are float and, where given, become beta times
    what they held plus the gradient."""
    dt = _dtype(ctx, x, w, a, b, dy)
    X = _rows(x, "x")
    W, A, B, S, I, U, t, cin, cout, n, units, rank = _adapter_args(ctx, x, w, a, b, scale, idx, unit_off)
    p, seed, offset = drop if drop is not None else (0.0, 0, 0)
    if not (dy.shape == (t, cout)):
        _fail("dy must be (T, out)")
    if not (beta == 0.0 or (da is not None and db is not None)):
        _fail("beta without da and db to add to")
    dx = _empty(ctx, x, (t, cin)) if need_dx else None
    da = _empty(ctx, x, a.shape, torch.float32) if da is None else da
    db = _empty(ctx, x, b.shape, torch.float32) if db is None else db
    ctx.call("kdec_adapter_bwd", dt, *X, W, A, B, S, I, U, t, cin, cout, n, units, rank, p, seed, offset,
             _floats(ctx, h, (t, units * rank), "h"), *_rows(dy, "dy"), None if dx is None else dx.data_ptr(), cin,
             _floats(ctx, da, a.shape, "da"), _floats(ctx, db, b.shape, "db"), beta)
    return dx, da, db


def dropout(ctx: Context, x, p, seed, offset=0, *, residual=None, out=None):
    """residual + x with values dropped with probability p and the kept ones
    scaled by 1 / (1 - p) (kdec_dropout; p in steps of 1 / 65536). The mask is
    the seed's, the offset's and the place's alone: the backward is this call on
    the gradient with the same seed and offset and no residual, and dropouts
    whose masks are to differ, ``drop`` of ``adapter_proj`` among them, take
    offsets of their own. ``out`` may be x."""
    dt = _dtype(ctx, x)
    X = _rows(x, "x")
    if x.shape[1] > _INT_MAX:  # the rows are a long
        _large()
    y = _empty(ctx, x, x.shape) if out is None else out
    _dtype(ctx, x, y)
    if not (y.shape == x.shape):
        _fail("out must be as x")
    R = (None, 0)
    if residual is not None:
        _dtype(ctx, x, residual)
        if not (residual.shape == x.shape):
            _fail("residual must be as x")
        R = _rows(residual, "residual")
    ctx.call("kdec_dropout", dt, *X, *R, *_rows(y, "out"), x.shape[0], x.shape[1], p, seed, offset)
    return y


def embedding(ctx: Context, table, ids, *, scale=1.0, out=None):
    """scale * table[ids] (kdec_embed_fwd): table (vocab, columns), ids (T
    int32); an id outside the table gives a row of zeros."""
    dt = _dtype(ctx, table)
    W = _rows(table, "table")
    vocab, cols = table.shape
    t = ids.numel()
    if (vocab | cols | t) > _INT_MAX:
        _fail("a table has from 0 to 2^31 - 1 rows and columns, and as many ids")
    if ids.dim() != 1:
        _fail("ids must be (T)")
    if out is None:
        y = _empty(ctx, table, (t, cols))
        Y = y.data_ptr(), cols
    else:
        y, Y = out, _as(ctx, out, table.dtype, (t, cols), "out must be (T, columns)")
    ctx.call("kdec_embed_fwd", dt, *W, _ints(ctx, ids, t, "ids"), t, vocab, cols, float(scale), *Y)
    return y


def embedding_bwd(ctx: Context, ids, dy, vocab, *, scale=1.0, dtable=None, beta=0.0):
    """The gradient of ``embedding``'s table from ``dy`` (kdec_embed_bwd), float
    (vocab, columns): beta times what ``dtable`` held, where it is given, plus
    scale times the sum of every id's rows, in one order."""
    dt = _dtype(ctx, dy)
    Y = _rows(dy, "dy")
    t, cols = dy.shape
    if ids.dim() != 1:
        _fail("ids must be (T)")
    if vocab < 0 or (vocab | cols | t) > _INT_MAX:
        _fail("a table has from 0 to 2^31 - 1 rows and columns, and as many ids")
    I = _ints(ctx, ids, t, "ids")  # noqa: E741
    if not (beta == 0.0 or dtable is not None):
        _fail("beta without dtable to add to")
    g = _empty(ctx, dy, (vocab, cols), torch.float32) if dtable is None else dtable
    ctx.call("kdec_embed_bwd", dt, *Y, I, t, vocab, cols, float(scale), _floats(ctx, g, (vocab, cols), "dtable"), float(beta))
    return g


def _as(ctx, t, ty, shape, what):
    """Address and row stride of a (rows, columns) tensor that must have this type and shape."""
    if t.dtype != ty or t.get_device() != ctx.device:
        _fail("tensors must share one type and device")
    if t.requires_grad:
        _no_graph(t)
    if t.shape != shape:
        _fail(what)
    return _rows(t, what)


def _norm_vectors(ctx, wb, ty, c, what):
    """A norm's flag and the addresses of its weight and bias."""
    if wb is None:
        return 0, None, None
    if not isinstance(wb, (tuple, list)):
        wb = (wb, None)
    if len(wb) != 2:
        _fail(f"{what} must be a weight or (weight, bias)")
    return 1, _vector(ctx, wb[0], ty, c, what), _vector(ctx, wb[1], ty, c, what)


def _vector(ctx, v, ty, c, what):
    if v is None:
        return None
    if v.dtype != ty or v.get_device() != ctx.device:
        _fail("tensors must share one type and device")
    if v.requires_grad:
        _no_graph(v)
    if v.shape != (c,) or not v.is_contiguous():
        _fail(f"{what} must be contiguous, of shape {(c,)}")
    return v.data_ptr()


def _norm_args(ctx, x, z, gate, post, pre, kind, eps, scale, x_scale):
    """The arguments that both directions share, and x's type and shape."""
    dt, X, ty, shape = _dtype(ctx, x), _rows(x, "x"), x.dtype, x.shape
    t, c = shape
    if (t | c) > _INT_MAX:
        _large()
    if kind != "rms" and kind != "layer":
        _fail("kind must be 'rms' or 'layer'")
    G = None, 0
    if z is None:
        Z = None, 0
        if post is not None or gate is not None or x_scale != 1.0 or pre is None:
            _fail("without z there is the norm of x alone")
    else:
        Z = _as(ctx, z, ty, shape, "z must be as x")
        if gate is not None:
            if gate.dim() == 1:
                G = _vector(ctx, gate, ty, c, "gate"), 0
            else:
                G = _as(ctx, gate, ty, shape, "gate must be (columns) or as x")
                if G[1] == 0:  # which the C ABI takes for one gate for all rows
                    if t > 1:
                        _fail("one gate for all rows must be (columns)")
                    G = G[0], c
    return (dt, int(kind == "layer"), *X, *Z, *G, *_norm_vectors(ctx, post, ty, c, "post"), *_norm_vectors(ctx, pre, ty, c, "pre"), float(eps),
            float(scale), float(x_scale), t, c), ty, (t, c)


def residual_norm(ctx: Context, x, z=None, *, gate=None, post=None, pre=None, kind="rms", eps=1e-5, scale=1.0, x_scale=1.0, keep=False,
                  out=None):
    """What stands between two blocks, in one pass (kdec_resnorm_fwd): the
    block's output z (T, C) through its norm ``post``, its ``gate`` ((C), or
    (T, C) with a gate for each row) and ``scale`` onto the residual x, and the
    next block's norm ``pre``:

        r = x_scale x + scale gate N_post(z),   y = N_pre(r)

    ``post`` and ``pre`` are None (no norm), a weight, or (weight, bias) of
    which either may be None; ``kind`` is "rms" or "layer". Without z it is y =
    N_pre(x), and r is x. ``out`` may give r and y, (r, y). Returns (r, y), y
    None without ``pre``, and with ``keep`` also the statistics that the
    backward takes."""
    args, ty, shape = _norm_args(ctx, x, z, gate, post, pre, kind, eps, scale, x_scale)
    r, y = out if out is not None else (None, None)
    R = Y = None, 0
    if z is None:
        r = x
    elif r is None:
        r = _empty(ctx, x, shape)
        R = r.data_ptr(), shape[1]
    else:
        R = _as(ctx, r, ty, shape, "r must be as x")
    if pre is None:
        y = None
    elif y is None:
        y = _empty(ctx, x, shape)
        Y = y.data_ptr(), shape[1]
    else:
        Y = _as(ctx, y, ty, shape, "y must be as x")
    stats = _empty(ctx, x, (shape[0], 4), torch.float32) if keep else None
    ctx.call("kdec_resnorm_fwd", *args, *R, *Y, None if stats is None else stats.data_ptr())
    return (r, y, stats) if keep else (r, y)


def residual_norm_bwd(ctx: Context, x, z, dr, dy, stats, *, gate=None, post=None, pre=None, kind="rms", eps=1e-5, scale=1.0, x_scale=1.0):
    """The gradients (dx, dz, dgate, dpost, dpre) of ``residual_norm`` from
    those of r (None: none) and y, with its inputs, arguments and statistics
    (kdec_resnorm_bwd). dx, dz and the gate's of each row are of x's type; the
    gradients of (C) vectors are float, dpost and dpre (weight's, bias's) with
    None where there is none."""
    args, ty, shape = _norm_args(ctx, x, z, gate, post, pre, kind, eps, scale, x_scale)
    t, c = shape
    if (dy is None) != (pre is None):
        _fail("dy comes with pre")
    st = _floats(ctx, stats, (t, 4), "stats")
    DR = (None, 0) if dr is None else _as(ctx, dr, ty, shape, "dr must be as x")
    DY = (None, 0) if dy is None else _as(ctx, dy, ty, shape, "dy must be as x")
    dx, dz = _empty(ctx, x, shape), None if z is None else _empty(ctx, x, shape)
    wide = gate is not None and gate.dim() == 2
    wb = [v if isinstance(v, (tuple, list)) else (v, None) for v in (post, pre)]
    want = (wb[0][0], wb[0][1], wb[1][0], wb[1][1], None if wide else gate)
    n = sum(v is not None for v in want)
    parts = iter(_empty(ctx, x, (n, c), torch.float32).unbind(0) if n else ())  # one allocation for the vectors' gradients
    got = [None if v is None else next(parts) for v in want]
    if wide:
        got[4] = _empty(ctx, x, shape)
    at = [None if v is None else v.data_ptr() for v in got]
    ctx.call("kdec_resnorm_bwd", *args, st, *DR, *DY, dx.data_ptr(), None if dz is None else dz.data_ptr(), at[4], *at[:4])
    return dx, dz, got[4], None if post is None else (got[0], got[1]), None if pre is None else (got[2], got[3])


class Cache(NamedTuple):
    """A key and value cache in 8 bits (kdec_cache_write): codes k and v (rows,
    heads, width rounded up to 16), int8, and their scales (heads, rows), float."""
    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor
    v_scale: torch.Tensor


def new_cache(ctx: Context, rows, heads, width):
    """An empty ``Cache`` of `rows` tokens (of all requests' slots together)."""
    with torch.cuda.stream(ctx.stream):
        codes = torch.zeros(rows, 2, heads, (width + 15) // 16 * 16, dtype=torch.int8, device=f"cuda:{ctx.device}")
        scales = torch.zeros(2, heads, rows, device=codes.device)
    return Cache(codes[:, 0], codes[:, 1], scales[0], scales[1])


def _cache_args(ctx, cache, width):
    """A cache's codes and scales as the C ABI takes them, its rows and heads."""
    k, v, ks, vs = cache
    dev, shape, wide = ctx.device, k.shape, (width + 15) // 16 * 16
    if k.dtype != torch.int8 or v.dtype != torch.int8 or k.get_device() != dev or v.get_device() != dev:
        _fail("the cache's k and v must be int8 on the device")
    if len(shape) != 3 or v.shape != shape or shape[2] != wide:
        _fail(f"the cache's k and v must be (rows, heads, {wide})")
    heads = shape[1], shape[0]
    if (shape[0] | shape[1] | wide) > _INT_MAX:
        _large()
    return (*_heads(k, "the cache's k"), *_heads(v, "the cache's v"), _floats(ctx, ks, heads, "k_scale"), _floats(ctx, vs, heads, "v_scale")), \
        shape[0], shape[1]


def _places(ctx, q_off, k_off, k_len):
    docs = q_off.numel() - 1
    if docs < 0:
        _fail("q_off must hold one offset more than there are documents")
    if docs > _INT_MAX:
        _large()
    return _ints(ctx, q_off, docs + 1, "q_off"), _ints(ctx, k_off, docs + 1, "k_off"), _ints(ctx, k_len, docs, "k_len"), docs


def cache_write(ctx: Context, k, v, cache, q_off, k_off, k_len=None):
    """Writes new tokens' k and v (T, heads, width) into ``cache``
    (kdec_cache_write): the rows q_off[d]:q_off[d+1] become the last of the
    k_len[d] filled tokens in the slot k_off[d]:k_off[d+1] (of the whole slot
    without k_len), where ``cache_attention`` with the same arguments expects
    them. Rows outside a document or before its slot are left out."""
    dt = _dtype(ctx, k, v)
    K, V = _heads(k, "k"), _heads(v, "v")
    t, h, d = k.shape
    C, rows, heads = _cache_args(ctx, cache, d)
    if v.shape != k.shape or heads != h:
        _fail("k and v must share their shape, and the cache's heads")
    if t > _INT_MAX:
        _large()
    ctx.call("kdec_cache_write", dt, *K, *V, *_places(ctx, q_off, k_off, k_len), t, rows, h, d, *C)


def cache_read(ctx: Context, cache, q_off, k_off, k_len=None, *, rows, width, dtype=torch.bfloat16, out=None):
    """The tokens that ``cache_write`` with the same arguments wrote, as (k, v)
    of `rows` rows: (rows, heads, width) of ``dtype`` (kdec_cache_read). Rows
    that it would not have written are zeros."""
    C, tk, heads = _cache_args(ctx, cache, width)
    if not 0 <= rows <= _INT_MAX:
        _fail("rows must be from 0 to 2^31 - 1")
    if out is None:
        if dtype not in _TYPES:
            _fail("tensors must be float32 or bfloat16")
        shape = rows, heads, width
        k, v = _empty(ctx, cache.k, shape, dtype), _empty(ctx, cache.k, shape, dtype)
        dt, K, V = _TYPES[dtype], (k.data_ptr(), heads * width, width), (v.data_ptr(), heads * width, width)
    else:
        k, v = out
        dt, K, V = _dtype(ctx, k, v), _heads(k, "k"), _heads(v, "v")
        if k.shape != (rows, heads, width) or v.shape != k.shape:
            _fail("out must be two tensors (rows, heads, width)")
    ctx.call("kdec_cache_read", dt, *C, *_places(ctx, q_off, k_off, k_len), rows, tk, heads, width, *K, *V)
    return k, v


def cache_attention(ctx: Context, q, cache, q_off, k_off, k_len=None, *, causal=False, prefix=None, scale=None, cap=0.0, slopes=None,
                    out=None):
    """``attention`` over a ``Cache`` (kdec_attn_cache_fwd): q (Tq, Hq, D) and
    the documents' keys and values k_off, k_len in the cache, the same masks,
    scores and results (o, lse). One row for a request or many."""
    dt = _dtype(ctx, q)
    Q = _heads(q, "q")
    tq, hq, d = q.shape
    C, tk, hkv = _cache_args(ctx, cache, d)
    if (tq | hq) > _INT_MAX:
        _large()
    qo, ko, kl, docs = _places(ctx, q_off, k_off, k_len)
    if out is None:
        o = _empty(ctx, q, (tq, hq, d))
        O = o.data_ptr(), hq * d, d  # noqa: E741
    else:
        _dtype(ctx, q, out)
        if out.shape != q.shape:
            _fail("out must be as q")
        o, O = out, _heads(out, "out")  # noqa: E741
    lse = _empty(ctx, q, (hq, tq), torch.float32)
    ctx.call("kdec_attn_cache_fwd", dt, *Q, *C, qo, ko, kl, _ints(ctx, prefix, docs, "prefix"), docs, int(causal),
             _floats(ctx, slopes, (hq,), "slopes"), float(d ** -0.5 if scale is None else scale), float(cap), tq, tk, hq, hkv, d, *O, lse.data_ptr())
    return o, lse
