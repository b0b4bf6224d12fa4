"""The adapters' gradients (kdec_adapter_bwd) where an adapter's rows lie in several chunks of sorted rows, that begin
and end inside them: dA and dB against the definition in 64 bits, and the room that many rows take."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_adapter import TYPES, ctx, make  # noqa: E402, F401


def definition(d, idx, keep=None):
    """h, da, db by adapter in 64 bits, and the root of the summed squares of their products (dH's and H's own too)."""
    x, a, b, dy = (d[k].double() for k in ("x", "a", "b", "dy"))
    n, out, rank = b.shape
    if keep is not None:
        x = x * keep
    units = len(d["edges"]) - 1
    h = torch.zeros(x.shape[0], units * rank, dtype=torch.float64, device=x.device)
    da, db = torch.zeros_like(a), torch.zeros_like(b)
    for v in range(n):
        r = torch.from_numpy(np.flatnonzero(idx == v)).to(x.device)
        s = float(d["scale"][v])
        for u in range(units):
            c, e = slice(u * rank, (u + 1) * rank), slice(d["edges"][u], d["edges"][u + 1])
            h[r, c] = s * x[r] @ a[v, c].T
            da[v, c] = (s * dy[r, e] @ b[v, e]).T @ x[r]
            db[v, e] = dy[r, e].T @ h[r, c]
    return h, da, db


def check(got, want, longest):
    # float sums whose products are exact to 24 bits: relative to the norm, 2^-24 by the sums' root length and a few more
    assert float((got.double() - want).norm()) <= 2.0 ** -24 * (longest ** 0.5 + 16) * float(want.norm())


@pytest.mark.parametrize("ty", TYPES, ids=["f32", "bf16"])
@pytest.mark.parametrize("case", [
    dict(T=700, cin=72, sizes=[64, 40], n=5, rank=16),
    dict(T=257, cin=40, sizes=[48], n=2, rank=4),
    dict(T=768, cin=130, sizes=[33, 31], n=3, rank=8, odd=True),
    dict(T=1500, cin=64, sizes=[24], n=40, rank=33),                 # several adapters to a chunk, some without rows
    dict(T=5000, cin=56, sizes=[200, 24], n=3, rank=8, drop=(0.25, 77, 3)),
    dict(T=140001, cin=24, sizes=[16, 8], n=4, rank=4),              # chunks of 512
], ids=lambda c: "-".join(f"{k}{v}" for k, v in c.items()).replace(" ", "")[:60])
def test_gradients_over_chunks(ctx, ty, case):  # noqa: F811
    from brosoundml_amd import tokens
    case = dict(case)
    drop = case.pop("drop", None)
    d = make(ty, **case)
    T, n, cin = case["T"], case["n"], case["cin"]
    idx = np.random.default_rng(T).integers(-1, n, T)
    idx[idx == 17] = 18
    idx[T // 3:T // 2] = 0  # a run that fills chunks of its own
    I = torch.from_numpy(idx.astype(np.int32)).cuda()
    edges = torch.tensor(d["edges"], dtype=torch.int32).cuda()
    args = (ctx, d["x"], d["w"], d["a"], d["b"], d["scale"], I, edges)
    _, h = tokens.adapter_proj(*args, drop=drop, keep_h=True)
    _, da, db = tokens.adapter_proj_bwd(*args, h, d["dy"], drop=drop, need_dx=False)
    keep = tokens.dropout(ctx, torch.ones(T, cin, device="cuda"), *drop).double() if drop else None
    wh, wa, wb = definition(d, idx, keep)
    check(h, wh, cin)
    check(da, wa, T)
    check(db, wb, T)
    # added to what is there, and the same bits again
    base_a, base_b = torch.full_like(da, 3.0), torch.full_like(db, -2.0)
    _, a2, b2 = tokens.adapter_proj_bwd(*args, h, d["dy"], drop=drop, need_dx=False, da=base_a, db=base_b, beta=0.5)
    check(a2, wa + 1.5, T)
    check(b2, wb - 1.0, T)
    _, a3, b3 = tokens.adapter_proj_bwd(*args, h, d["dy"], drop=drop, need_dx=False)
    assert torch.equal(a3, da) and torch.equal(b3, db)


def test_room_for_many_rows():
    """A million rows of 1024 columns: the gradients' shares took 0.54 GB, one for every 256 rows; with the rows' own
    64 MB of dH it is less than a third of that now."""
    from brosoundml_amd import native, tokens
    c = native.Context(0)
    T, w, rank = 1 << 20, 1024, 16
    x = torch.randn(T, w, device="cuda", dtype=torch.bfloat16)
    wt, a, b = (torch.randn(*s, device="cuda", dtype=torch.bfloat16) for s in ((w, w), (4, rank, w), (4, w, rank)))
    idx, edges = torch.randint(-1, 4, (T,), device="cuda").int(), torch.tensor([0, w], dtype=torch.int32).cuda()
    h = torch.randn(T, rank, device="cuda")
    da, db = torch.empty(4, rank, w, device="cuda"), torch.empty(4, w, rank, device="cuda")
    torch.cuda.synchronize()
    before = torch.cuda.mem_get_info()[0]
    tokens.adapter_proj_bwd(c, x, wt, a, b, torch.ones(4, device="cuda"), idx, edges, h, x, need_dx=False, da=da, db=db)
    torch.cuda.synchronize()
    assert before - torch.cuda.mem_get_info()[0] < 200 << 20
