"""Sizes that the C ABI's ints do not hold: every token operator refuses them before it allocates or calls anything. On the
CPU, with a context that only notes the calls made: rows of stride 0 take no memory."""
import pytest

torch = pytest.importorskip("torch")

from brosoundml_amd import tokens  # noqa: E402

FAR = 2 ** 32 + 5  # its low 32 bits are 5: cut to an int it would be a size that fits


class Context:
    device = -1  # torch's number for tensors of the CPU

    def __init__(self):
        self.calls = []

    def call(self, name, *args):
        self.calls.append(name)


def far(*shape, at=0, dtype=torch.float32):
    """Ones of FAR rows (or heads, or columns: axis `at`), repeated."""
    shape = list(shape)
    shape.insert(at, 1)
    t = torch.ones(shape, dtype=dtype)
    shape[at] = FAR
    return t.expand(shape)


def wide():
    """No rows of FAR columns."""
    return torch.empty(0, FAR)


def ints(n):
    return torch.zeros(n, dtype=torch.int32)


def cache(rows, heads=2, width=16, k=None, scales=None):
    codes = torch.zeros(rows, heads, width, dtype=torch.int8) if k is None else k
    scales = torch.zeros(heads, rows) if scales is None else scales
    return tokens.Cache(codes, codes, scales, scales)


ROWS = torch.ones(3, 8)
HEADS = torch.ones(3, 2, 16)
OFF = torch.tensor([0, 3], dtype=torch.int32)

CASES = {
    "embedding, table": lambda c: tokens.embedding(c, far(8), ints(3)),
    "embedding, columns": lambda c: tokens.embedding(c, wide(), ints(3)),
    "embedding_bwd, tokens": lambda c: tokens.embedding_bwd(c, ints(3), far(8), 9),
    "embedding_bwd, columns": lambda c: tokens.embedding_bwd(c, ints(0), wide(), 9),
    "residual_norm, rows": lambda c: tokens.residual_norm(c, far(8), pre=torch.ones(8)),
    "residual_norm, rows with z": lambda c: tokens.residual_norm(c, far(8), far(8), pre=torch.ones(8)),
    "residual_norm, columns": lambda c: tokens.residual_norm(c, wide(), pre=(None, None)),
    "residual_norm_bwd, rows": lambda c: tokens.residual_norm_bwd(c, far(8), None, None, far(8), torch.ones(1, 4).expand(FAR, 4), pre=torch.ones(8)),
    "cache_write, tokens": lambda c: tokens.cache_write(c, far(2, 16), far(2, 16), cache(8), OFF, OFF),
    "cache_write, heads": lambda c: tokens.cache_write(c, far(3, 16, at=1), far(3, 16, at=1), cache(8, k=far(8, 16, at=1, dtype=torch.int8)), OFF, OFF),
    "cache_write, cache rows": lambda c: tokens.cache_write(c, HEADS, HEADS, cache(FAR, k=far(2, 16, dtype=torch.int8), scales=far(2, at=1)), OFF, OFF),
    "cache_read, cache rows": lambda c: tokens.cache_read(c, cache(FAR, k=far(2, 16, dtype=torch.int8), scales=far(2, at=1)), OFF, OFF, rows=3, width=16),
    "cache_read, rows": lambda c: tokens.cache_read(c, cache(8), OFF, OFF, rows=FAR, width=16),
    "cache_read, rows into tensors": lambda c: tokens.cache_read(c, cache(8), OFF, OFF, rows=FAR, width=16, out=(far(2, 16), far(2, 16))),
    "cache_read, negative rows": lambda c: tokens.cache_read(c, cache(8), OFF, OFF, rows=-1, width=16),
    "cache_attention, rows": lambda c: tokens.cache_attention(c, far(2, 16), cache(8), OFF, OFF),
    "cache_attention, heads": lambda c: tokens.cache_attention(c, far(3, 16, at=1), cache(8), OFF, OFF),
    "cache_attention, cache rows": lambda c: tokens.cache_attention(c, HEADS, cache(FAR, k=far(2, 16, dtype=torch.int8), scales=far(2, at=1)), OFF, OFF),
    "attention, rows": lambda c: tokens.attention(c, far(2, 16), far(2, 16), far(2, 16), OFF),
    "attention, keys": lambda c: tokens.attention(c, HEADS, far(2, 16), far(2, 16), OFF, OFF),
    "attention_bwd, rows": lambda c: tokens.attention_bwd(c, far(2, 16), far(2, 16), far(2, 16), far(2, 16), HEADS, far(2, 16), OFF),
    "adapter_proj, rows": lambda c: tokens.adapter_proj(c, far(8), torch.ones(4, 8), torch.ones(2, 3, 8), torch.ones(2, 4, 3), torch.ones(2), ints(3), ints(2)),
    "dropout, columns": lambda c: tokens.dropout(c, wide(), 0.1, 1),
}


@pytest.mark.parametrize("name", CASES)
def test_refused(name):
    ctx = Context()
    with pytest.raises(ValueError, match="2\\^31"):
        CASES[name](ctx)
    assert not ctx.calls


def test_dropout_takes_as_many_rows_as_a_long_holds():
    ctx, x = Context(), far(8)
    assert tokens.dropout(ctx, x, 0.1, 1, out=x, residual=x) is x and ctx.calls == ["kdec_dropout"]


def test_sizes_that_fit_are_called():
    """The same calls with outputs given, so that nothing is allocated on a device."""
    ctx = Context()
    tokens.embedding(ctx, ROWS, ints(3), out=torch.empty(3, 8))
    tokens.embedding_bwd(ctx, ints(3), ROWS, 9, dtable=torch.empty(9, 8))
    tokens.residual_norm(ctx, ROWS, pre=torch.ones(8), out=(None, torch.empty(3, 8)))
    tokens.cache_write(ctx, HEADS, HEADS, cache(8), OFF, OFF)
    tokens.cache_read(ctx, cache(8), OFF, OFF, rows=3, width=16, out=(HEADS, HEADS))
    assert ctx.calls == ["kdec_embed_fwd", "kdec_embed_bwd", "kdec_resnorm_fwd", "kdec_cache_write", "kdec_cache_read"]
