"""Few rows for each of many requests over their caches: results against the definition for more documents than two
turns of 64, with padding rows, and that neither padding nor one document more changes what a call costs."""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_attention import TYPES, compare, ctx  # noqa: E402, F401


@pytest.mark.parametrize("ty", TYPES, ids=["f32", "bf16"])
@pytest.mark.parametrize("case", [
    dict(docs=140, rows=2, keys=400, slot=420, hq=4, hkv=2, D=64),                   # blocks that end with their document
    dict(docs=130, rows=1, keys=300, slot=310, hq=4, hkv=1, D=128, pad=5),           # padded single rows
    dict(docs=260, rows=1, keys=60, slot=64, hq=2, hkv=2, D=64, pad=9),              # too many documents for short caches
    dict(docs=200, rows=3, keys=700, slot=701, hq=2, hkv=1, D=64, cap=5.0, slopes=True),
], ids=lambda c: "-".join(f"{k}{v}" for k, v in c.items()))
def test_many_requests(ctx, ty, case):  # noqa: F811
    case = dict(case)
    docs, rows, keys, slot = (case.pop(n) for n in ("docs", "rows", "keys", "slot"))
    lk = [max(0, keys - 7 * (i % 50) - (keys if i % 41 == 40 else 0)) for i in range(docs)]  # some caches are empty
    compare(ctx, ty, [rows] * docs, lk, case.pop("hq"), case.pop("hkv"), case.pop("D"), slots=[slot] * docs, causal=True,
            spoil=math.nan, **case)


def cost(ctx, docs, rows, pad, keys=1000):  # noqa: F811
    """Microseconds of a forward call, the best of five runs of twenty."""
    from brosoundml_amd import tokens
    q = torch.randn(docs * rows + pad, 16, 128, device="cuda", dtype=torch.bfloat16)
    k, v = (torch.randn(docs * keys, 4, 128, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    q_off, k_off = (torch.arange(docs + 1, device="cuda") * rows).int(), (torch.arange(docs + 1, device="cuda") * keys).int()
    best = math.inf
    for _ in range(5):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        for _ in range(20):
            tokens.attention(ctx, q, k, v, q_off, k_off, causal=True)
        b.record()
        b.synchronize()
        best = min(best, a.elapsed_time(b) * 50)
    return best


def test_padding_rows_cost_nothing(ctx):  # noqa: F811
    """128 requests of one row with four padding rows took three times what they take without."""
    assert cost(ctx, 128, 1, 4) < 1.6 * cost(ctx, 128, 1, 0)


def test_two_rows_of_more_than_two_turns_of_documents(ctx):  # noqa: F811
    """128 requests of two rows took nearly twice what 126 take."""
    assert cost(ctx, 128, 2, 0) < 1.4 * cost(ctx, 126, 2, 0)
