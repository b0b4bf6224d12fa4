"""Token operators on torch tensors: attention over packed documents, the
projection with low-rank adapters chosen per row, and dropout (the last
section of kdec.h). Each call checks its tensors, allocates what it returns
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

import torch

from .native import Context

try:  # the current stream's address without an object around it
    from torch._C import _cuda_getCurrentRawStream as _raw_stream
except ImportError:
    def _raw_stream(device):
        return torch.cuda.current_stream(device).cuda_stream

_TYPES = {torch.float32: 0, torch.bfloat16: 1}


# A single token's kernels take a few microseconds, about what these checks
# do: each reads what it needs of a tensor once, and forms no message that it
# does not raise.

def _fail(what):
    raise ValueError("brosoundml: " + what)


def _no_graph(x):
    if x.requires_grad and torch.is_grad_enabled():
        _fail("a tensor requires grad, and these calls make no autograd graph: detach it or call under torch.no_grad()")


def _dtype(ctx, x, *others):
    """The C ABI's type of x, which the others must share, all on the context's device."""
    ty, dev = x.dtype, x.device
    if ty not in _TYPES:
        _fail("tensors must be float32 or bfloat16")
    if dev.type != "cuda" or dev.index != ctx.device:
        _fail("tensors must be on the context's HIP device")
    if x.requires_grad:
        _no_graph(x)
    for t in others:
        if t.requires_grad:
            _no_graph(t)
        if t.dtype != ty or t.device != dev:
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
        return x.new_empty(shape, dtype=dtype)
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
