"""Token operators on torch tensors: attention over packed documents, the
projection with low-rank adapters chosen per row, and dropout (the last
section of kdec.h). Each call checks its tensors, allocates what it returns
and makes one C ABI call on the context's stream; nothing synchronises. A
tensor made on another stream has to be ordered before the context's by the
caller, as for every call of the library.

Tensors are float32 or bfloat16 (one type per call), on the context's device;
offsets and adapter choices are int32 tensors there. Errors are
``native.KdecError`` (what the library refuses) and ``ValueError`` (tensors
that do not fit each other)."""
from __future__ import annotations

import torch

from .native import Context

_TYPES = {torch.float32: 0, torch.bfloat16: 1}


def _need(cond, what):
    if not cond:
        raise ValueError("brosoundml: " + what)


def _dtype(x, *others):
    """The C ABI's type of x, which the others must share, all on one HIP device."""
    _need(x.dtype in _TYPES, "tensors must be float32 or bfloat16")
    _need(x.is_cuda, "tensors must be on the HIP device")
    for t in others:
        _need(t.dtype == x.dtype and t.device == x.device, "tensors must share one type and device")
    return _TYPES[x.dtype]


def _ints(x, n, what):
    """Address of an int32 tensor of n values on the device (None passes)."""
    if x is None:
        return None
    _need(x.dtype == torch.int32 and x.is_cuda and x.is_contiguous() and x.numel() == n,
          f"{what} must hold {n} contiguous int32 values on the device")
    return x.data_ptr()


def _floats(x, shape, what):
    if x is None:
        return None
    _need(x.dtype == torch.float32 and x.is_cuda and x.is_contiguous() and tuple(x.shape) == tuple(shape),
          f"{what} must be a contiguous float32 tensor of shape {tuple(shape)}")
    return x.data_ptr()


def _heads(x, what):
    """Address, row stride and head stride of a (rows, heads, width) tensor with contiguous width."""
    _need(x.dim() == 3, f"{what} must be (rows, heads, width)")
    _need(x.stride(2) == 1 or x.shape[2] <= 1, f"{what}: the width must be contiguous")
    return x.data_ptr(), x.stride(0), x.stride(1)


def _rows(x, what):
    """Address and row stride of a (rows, columns) tensor with contiguous columns."""
    _need(x.dim() == 2, f"{what} must be (rows, columns)")
    _need(x.stride(1) == 1 or x.shape[1] <= 1, f"{what}: the columns must be contiguous")
    return x.data_ptr(), x.stride(0)


def _whole(x, shape, what):
    _need(tuple(x.shape) == tuple(shape) and x.is_contiguous(), f"{what} must be contiguous, of shape {tuple(shape)}")
    return x.data_ptr()


class _on:
    """Allocations inside belong to the context's stream."""

    def __init__(self, ctx: Context):
        self.cm = None if torch.cuda.current_stream(ctx.device) == ctx.stream else torch.cuda.stream(ctx.stream)

    def __enter__(self):
        if self.cm is not None:
            self.cm.__enter__()

    def __exit__(self, *a):
        if self.cm is not None:
            self.cm.__exit__(*a)


def _attn_args(q, k, v, q_off, k_off, k_len, causal, prefix, scale, cap, slopes):
    dt = _dtype(q, k, v)
    Q, K, V = _heads(q, "q"), _heads(k, "k"), _heads(v, "v")
    tq, hq, d = q.shape
    tk, hkv, _ = k.shape
    _need(v.shape == k.shape and k.shape[2] == d, "k and v must share their shape, and q their width")
    docs = q_off.numel() - 1
    _need(docs >= 0, "q_off must hold one offset more than there are documents")
    if k_off is None:
        _need(tq == tk, "without k_off the keys are the query rows' own")
        k_off = q_off
    # where / length / mask arguments, in the C ABI's order
    mask = (_ints(q_off, docs + 1, "q_off"), _ints(k_off, docs + 1, "k_off"), _ints(k_len, docs, "k_len"),
            _ints(prefix, docs, "prefix"), docs, int(causal), _floats(slopes, (hq,), "slopes"),
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
    dt, Q, K, V, mask = _attn_args(q, k, v, q_off, k_off, k_len, causal, prefix, scale, cap, slopes)
    tq, hq, _ = q.shape
    with _on(ctx):
        o = torch.empty(q.shape, dtype=q.dtype, device=q.device) if out is None else out
        lse = torch.empty((hq, tq), dtype=torch.float32, device=q.device)
    _need(o.shape == q.shape and o.dtype == q.dtype, "out must be as q")
    ctx.call("kdec_attn_fwd", dt, *Q, *K, *V, *mask, *_heads(o, "out"), lse.data_ptr())
    return o, lse


def attention_bwd(ctx: Context, q, k, v, o, lse, do, q_off, k_off=None, k_len=None, *, causal=False, prefix=None,
                  scale=None, cap=0.0, slopes=None, dq=None, dk=None, dv=None):
    """The gradients (dq, dk, dv) of ``attention`` from ``do``, with its o and
    lse and the same mask arguments (kdec_attn_bwd). dq, dk and dv may be
    given, for example as the parts of a fused projection's gradient."""
    dt, Q, K, V, mask = _attn_args(q, k, v, q_off, k_off, k_len, causal, prefix, scale, cap, slopes)
    _dtype(q, o, do)
    _need(o.shape == q.shape and do.shape == q.shape, "o and do must be as q")
    with _on(ctx):
        dq = torch.empty(q.shape, dtype=q.dtype, device=q.device) if dq is None else dq
        dk = torch.empty(k.shape, dtype=k.dtype, device=k.device) if dk is None else dk
        dv = torch.empty(v.shape, dtype=v.dtype, device=v.device) if dv is None else dv
    _dtype(q, dq, dk, dv)
    _need(dq.shape == q.shape and dk.shape == k.shape and dv.shape == v.shape, "dq, dk and dv must be as q, k and v")
    ctx.call("kdec_attn_bwd", dt, *Q, *K, *V, *_heads(o, "o"), _floats(lse, (q.shape[1], q.shape[0]), "lse"),
             *_heads(do, "do"), *mask, *_heads(dq, "dq"), *_heads(dk, "dk"), *_heads(dv, "dv"))
    return dq, dk, dv


def _adapter_args(x, w, a, b, scale, idx, unit_off):
    t, cin = x.shape
    out = w.shape[0]
    n, units = a.shape[0], unit_off.numel() - 1
    _need(b.dim() == 3 and units >= 1, "b must be (adapters, out, rank), unit_off units + 1 offsets")
    rank = b.shape[2]
    return (_whole(w, (out, cin), "w"), _whole(a, (n, units * rank, cin), "a"), _whole(b, (n, out, rank), "b"),
            _floats(scale, (n,), "scale"), _ints(idx, t, "idx"), _ints(unit_off, units + 1, "unit_off"), t, cin, out,
            n, units, rank)


def adapter_proj(ctx: Context, x, w, a, b, scale, idx, unit_off, *, bias=None, drop=None, keep_h=False, out=None):
    """x W^T + bias with row t's own low-rank adapter idx[t] beside it
    (kdec_adapter_fwd): x (T, in), w (out, in), a (adapters, units * rank,
    in), b (adapters, out, rank), scale (adapters floats); rows whose idx is
    outside [0, adapters) take none. unit_off (units + 1) cuts the output rows
    into units with adapters of their own. ``drop`` = (p, seed, offset) drops
    inputs of the adapters. Returns y (T, out), and with ``keep_h`` the pair
    (y, h) whose h the backward takes."""
    dt = _dtype(x, w, a, b)
    X = _rows(x, "x")
    W, A, B, S, I, U, t, cin, cout, n, units, rank = _adapter_args(x, w, a, b, scale, idx, unit_off)
    p, seed, offset = drop if drop is not None else (0.0, 0, 0)
    with _on(ctx):
        y = torch.empty((t, cout), dtype=x.dtype, device=x.device) if out is None else out
        h = torch.empty((t, units * rank), dtype=torch.float32, device=x.device) if keep_h else None
    _need(y.shape == (t, cout), "out must be (T, out)")
    _dtype(x, y)
    if bias is not None:
        _dtype(x, bias)
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
    dt = _dtype(x, w, a, b, dy)
    X = _rows(x, "x")
    W, A, B, S, I, U, t, cin, cout, n, units, rank = _adapter_args(x, w, a, b, scale, idx, unit_off)
    p, seed, offset = drop if drop is not None else (0.0, 0, 0)
    _need(dy.shape == (t, cout), "dy must be (T, out)")
    _need(beta == 0.0 or (da is not None and db is not None), "beta without da and db to add to")
    with _on(ctx):
        dx = torch.empty((t, cin), dtype=x.dtype, device=x.device) if need_dx else None
        da = torch.empty(a.shape, dtype=torch.float32, device=x.device) if da is None else da
        db = torch.empty(b.shape, dtype=torch.float32, device=x.device) if db is None else db
    ctx.call("kdec_adapter_bwd", dt, *X, W, A, B, S, I, U, t, cin, cout, n, units, rank, p, seed, offset,
             _floats(h, (t, units * rank), "h"), *_rows(dy, "dy"), None if dx is None else dx.data_ptr(), cin,
             _floats(da, a.shape, "da"), _floats(db, b.shape, "db"), beta)
    return dx, da, db


def dropout(ctx: Context, x, p, seed, offset=0, *, residual=None, out=None):
    """residual + x with values dropped with probability p and the kept ones
    scaled by 1 / (1 - p) (kdec_dropout; p in steps of 1 / 65536). The mask is
    the seed's and offset's alone: the backward is this call on the gradient
    with the same seed and offset and no residual. ``out`` may be x."""
    dt = _dtype(x)
    X = _rows(x, "x")
    with _on(ctx):
        y = torch.empty(x.shape, dtype=x.dtype, device=x.device) if out is None else out
    _dtype(x, y)
    _need(y.shape == x.shape, "out must be as x")
    R = (None, 0)
    if residual is not None:
        _dtype(x, residual)
        _need(residual.shape == x.shape, "residual must be as x")
        R = _rows(residual, "residual")
    ctx.call("kdec_dropout", dt, *X, *R, *_rows(y, "out"), x.shape[0], x.shape[1], p, seed, offset)
    return y
