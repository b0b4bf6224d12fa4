"""Embedding and its table's gradient (kdec_embed_fwd / kdec_embed_bwd) against their definition in 64 bits.

Tolerances, u the type's unit roundoff and e = 2^-24: a lookup is one float product, rounded once, (u + e) |y|. A
gradient is the float sum of n rows in some order, scaled: n e scale sum |dy| for the additions, and with beta one
product and one addition more, 3 e (|beta| |old| + |dtable|).
"""
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


def values(rng, ty, *shape, odd=False):
    if not odd:
        return torch.from_numpy(rng.standard_normal(shape).astype(np.float32)).to(ty).cuda()
    rows, cols = shape  # rows that start anywhere
    a = torch.from_numpy(rng.standard_normal((rows, cols + 5)).astype(np.float32)).to(ty).cuda()
    return a[:, 1:1 + cols]


def ints(a):
    return torch.tensor(np.asarray(a), dtype=torch.int32).cuda()


def check_lookup(ctx, table, ids, scale, **kw):
    from brosoundml_amd import tokens
    y = tokens.embedding(ctx, table, ints(ids), scale=scale, **kw)
    ids = torch.from_numpy(np.asarray(ids)).long()
    has = (ids >= 0) & (ids < table.shape[0])
    want = torch.zeros(len(ids), table.shape[1], dtype=torch.float64)
    want[has] = table.double().cpu()[ids[has]] * float(np.float32(scale))
    assert ((y.double().cpu() - want).abs() <= (U[table.dtype] + E) * want.abs()).all()
    return y


def check_grad(ctx, ids, dy, vocab, scale, old=None, beta=0.0):
    from brosoundml_amd import tokens
    given = None if old is None else old.clone()
    g = tokens.embedding_bwd(ctx, ints(ids), dy, vocab, scale=scale, dtable=given, beta=beta)
    assert g.dtype == torch.float32 and g.shape == (vocab, dy.shape[1])
    assert given is None or g is given
    at = torch.from_numpy(np.asarray(ids)).long()
    has = (at >= 0) & (at < vocab)
    d = dy.double().cpu()[has] * scale
    want = torch.zeros(vocab, dy.shape[1], dtype=torch.float64).index_add_(0, at[has], d)
    size = torch.zeros_like(want).index_add_(0, at[has], d.abs())
    n = torch.bincount(at[has], minlength=vocab).double()[:, None]
    tol = (n + 2) * E * size
    if beta:
        want += beta * old.double().cpu()
        tol += 3 * E * (abs(beta) * old.double().cpu().abs() + want.abs())
    off = (g.double().cpu() - want).abs()
    assert (off <= tol).all(), float((off - tol).max())
    return g


@pytest.mark.parametrize("ty", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("t,vocab,cols,odd", [(1, 1, 1, False), (1, 181, 512, False), (37, 181, 512, False), (65, 30, 77, True), (5, 9, 40, True),
                                              (300, 1000, 1021, False), (129, 7, 768, False)])
def test_lookup(ctx, ty, t, vocab, cols, odd):
    rng = np.random.default_rng([t, cols])
    table = values(rng, ty, vocab, cols, odd=odd)
    ids = rng.integers(-1, vocab + 1, t)
    ids[-1:] = [2 ** 31 - 1]
    check_lookup(ctx, table, ids, 1.0)
    check_lookup(ctx, table, ids, 22.627)
    out = torch.full((t, cols + 3), 7.0, dtype=ty, device="cuda")
    check_lookup(ctx, table, ids, 0.5, out=out[:, 1:1 + cols])
    assert (out[:, 0] == 7).all() and (out[:, 1 + cols:] == 7).all()


@pytest.mark.parametrize("ty", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("t,vocab,cols,odd", [
    (1, 1, 1, False), (1, 181, 512, False), (31, 181, 100, True), (32, 5, 512, False), (33, 2, 8, False), (64, 1, 520, False),  # pieces and their ends
    (257, 254, 64, False), (257, 255, 64, False), (257, 256, 64, False),      # one digit of 8 bits, and the first sizes past it
    (1023, 3, 128, False), (1025, 400, 1021, False), (5000, 70000, 24, True),   # two digits, three
    (16384, 181, 72, False), (16385, 181, 72, False), (40000, 9, 16, False), (33000, 66000, 16, True)])  # one sorting block, more
def test_gradient(ctx, ty, t, vocab, cols, odd):
    rng = np.random.default_rng([t, vocab, cols])
    ids = rng.integers(-1, vocab + 1, t) if vocab > 3 else rng.integers(0, vocab, t)
    dy = values(rng, ty, t, cols, odd=odd)
    a = check_grad(ctx, ids, dy, vocab, 1.0)
    b = check_grad(ctx, ids, dy, vocab, 1.0)
    assert torch.equal(a, b)  # the same bits every time
    old = values(rng, torch.float32, vocab, cols)
    check_grad(ctx, ids, dy, vocab, 22.627, old, 1.0)
    check_grad(ctx, ids, dy, vocab, 0.25, old, -0.5)


@pytest.mark.parametrize("which", ["all the same", "sorted", "backwards", "none", "two ends", "every 32nd"])
@pytest.mark.parametrize("t", [96, 3333, 20000])
def test_gradient_orders(ctx, which, t):
    rng = np.random.default_rng([t, len(which)])
    vocab, cols = 600, 40
    ids = {"all the same": np.full(t, 77), "sorted": np.sort(rng.integers(0, vocab, t)), "backwards": np.sort(rng.integers(0, vocab, t))[::-1].copy(),
           "none": np.full(t, -5), "two ends": np.where(np.arange(t) < t // 2, vocab - 1, 0), "every 32nd": np.arange(t) // 32 % vocab}[which]
    check_grad(ctx, ids, values(rng, torch.bfloat16, t, cols), vocab, 1.0)


def test_sums_take_ascending_tokens(ctx):
    """Rows of one id inside a piece are added in the tokens' order: 2^24 + 1 + 1 - 2^24 is 0 from the left in float."""
    from brosoundml_amd import tokens
    dy = torch.tensor([2.0 ** 24, 5.0, 1.0, 7.0, 1.0, -2.0 ** 24], device="cuda")[:, None].repeat(1, 8)
    g = tokens.embedding_bwd(ctx, ints([3, 1, 3, 0, 3, 3]), dy, 5)
    assert g[:, 0].tolist() == [7.0, 5.0, 0.0, 0.0, 0.0]


def test_values_that_are_not_finite_stay_with_their_id(ctx):
    from brosoundml_amd import tokens
    rng = np.random.default_rng(5)
    ids = rng.integers(0, 50, 4000)
    dy = values(rng, torch.float32, 4000, 24)
    clean = tokens.embedding_bwd(ctx, ints(ids), dy, 50)
    spoilt = dy.clone()
    spoilt[torch.from_numpy(np.flatnonzero(ids == 7)).cuda()] = float("nan")
    ids2 = ids.copy()
    ids2[ids == 9] = -1
    spoilt[torch.from_numpy(np.flatnonzero(ids == 9)).cuda()] = float("inf")  # rows outside the table
    g = tokens.embedding_bwd(ctx, ints(ids2), spoilt, 50)
    rest = [i for i in range(50) if i not in (7, 9)]
    clean2 = tokens.embedding_bwd(ctx, ints(ids2), dy, 50)  # the same ids: where pieces end decides how a sum is grouped
    assert torch.isnan(g[7]).all() and (g[9] == 0).all() and torch.equal(g[rest], clean2[rest])
    held = torch.full_like(clean, float("nan"))  # beta = 0 does not read what the table held
    assert torch.equal(tokens.embedding_bwd(ctx, ints(ids), dy, 50, dtable=held), clean)


def test_gradient_is_the_lookups(ctx):
    """<embedding(table + h d) - embedding(table - h d), dy> / 2h = <d, dtable>; the lookup is linear, so the step may be one."""
    from brosoundml_amd import tokens
    rng = np.random.default_rng(8)
    ids = rng.integers(-1, 40, 700)
    table, d, dy = values(rng, torch.float32, 40, 65), values(rng, torch.float32, 40, 65), values(rng, torch.float32, 700, 65)
    y = [tokens.embedding(ctx, table + s * d, ints(ids), scale=3.0).double() for s in (1, -1)]
    left = ((y[0] - y[1]) / 2 * dy.double()).sum()
    right = (d.double() * tokens.embedding_bwd(ctx, ints(ids), dy, 40, scale=3.0).double()).sum()
    size = 3.0 * float((d.double().abs()[torch.from_numpy(np.maximum(ids, 0)).cuda()] * dy.double().abs()).sum())
    # table +- d rounds by e |table| each, the rows and sums by n e: 700 of them at most
    assert abs(float(left - right)) <= 800 * E * (size + 3.0 * float(table.abs().max()) * float(dy.abs().sum()))


def test_offsets_past_32_bits(ctx):
    """A table of more than 2^31 values, and a gradient of rows that far apart."""
    from brosoundml_amd import tokens
    vocab, cols = 2100000, 1024
    table = torch.empty(vocab, cols, dtype=torch.bfloat16, device="cuda")
    table[:3], table[-3:] = 2.0, 5.0
    y = tokens.embedding(ctx, table, ints([vocab - 1, 0, vocab, vocab - 3]), scale=0.5)
    assert y[:, 0].tolist() == [2.5, 1.0, 0.0, 2.5] and (y == y[:, :1]).all()
    del table
    far = torch.empty(3, (1 << 30) + 8, dtype=torch.bfloat16, device="cuda")[:, :cols]
    far.copy_(torch.tensor([1.0, 2.0, 4.0])[:, None].expand(3, cols))
    g = tokens.embedding_bwd(ctx, ints([4, 4, 1]), far, 6)
    assert g[:, 0].tolist() == [0.0, 4.0, 0.0, 0.0, 3.0, 0.0] and (g == g[:, :1]).all()


def test_refusals(ctx):
    from brosoundml_amd import native, tokens
    table, ids, dy = torch.ones(9, 16, device="cuda"), ints([1, 2, 3]), torch.ones(3, 16, device="cuda")
    for call in (lambda: tokens.embedding(ctx, table.half(), ids), lambda: tokens.embedding(ctx, table, ids.long()),
                 lambda: tokens.embedding(ctx, table.cpu(), ids), lambda: tokens.embedding(ctx, table, ids.view(1, 3)),
                 lambda: tokens.embedding(ctx, table, ids, out=torch.ones(3, 15, device="cuda")), lambda: tokens.embedding(ctx, table.t(), ids),
                 lambda: tokens.embedding(ctx, table.clone().requires_grad_(), ids), lambda: tokens.embedding_bwd(ctx, ids[:2], dy, 9),
                 lambda: tokens.embedding_bwd(ctx, ids, dy, 9, beta=1.0), lambda: tokens.embedding_bwd(ctx, ids, dy, 9, dtable=table.bfloat16()),
                 lambda: tokens.embedding_bwd(ctx, ids, dy, 9, dtable=torch.ones(9, 17, device="cuda")[:, :16])):
        with pytest.raises(ValueError, match="brosoundml"):
            call()
    with pytest.raises(native.KdecError, match="too small"):
        tokens.embedding(ctx, table, ids, out=torch.empty(16, device="cuda").expand(3, 16))
    assert tokens.embedding(ctx, table, ids[:0]).shape == (0, 16)
    assert (tokens.embedding_bwd(ctx, ids[:0], dy[:0], 9) == 0).all()
    assert tokens.embedding(ctx, table[:0], ids).abs().sum() == 0
    with torch.no_grad():
        assert torch.equal(tokens.embedding(ctx, table.clone().requires_grad_(), ids), table[:3])


@pytest.mark.parametrize("vocab", [9, 600001])
def test_gradient_of_no_tokens(ctx, vocab):
    """The table is cleared, scaled or left as it was, however many ids it has."""
    from brosoundml_amd import tokens
    ids, dy = ints([]), torch.empty(0, 3, device="cuda")
    assert (tokens.embedding_bwd(ctx, ids, dy, vocab) == 0).all()
    for beta, want in ((1.0, 7.0), (0.5, 3.5), (0.0, 0.0)):
        held = torch.full((vocab, 3), 7.0, device="cuda")
        assert (tokens.embedding_bwd(ctx, ids, dy, vocab, dtable=held, beta=beta) == want).all(), beta


def test_tables_past_what_a_call_takes(ctx):
    """Sizes that do not fit the C ABI's int are refused, not cut to it."""
    from brosoundml_amd import tokens
    ids = ints([1, 2, 3])
    for vocab in (2 ** 31, 2 ** 32 + 5):
        with pytest.raises(ValueError, match="rows"):
            tokens.embedding(ctx, torch.ones(1, 8, device="cuda").expand(vocab, 8), ids)
        with pytest.raises(ValueError, match="rows"):
            tokens.embedding_bwd(ctx, ids, torch.ones(3, 8, device="cuda"), vocab)
    with pytest.raises(ValueError, match="rows"):
        tokens.embedding_bwd(ctx, ids, torch.ones(3, 8, device="cuda"), -1)
