"""Attention where its blocks fill the device (each then has 32 entries to a wave, not two waves to 32 entries), where
blocks hold several documents, and where one document's rows are shared out, against the definition in 64 bits with
test_gpu_attention.py's tolerances."""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_attention import TYPES, compare, ctx  # noqa: E402, F401


def name(c):
    return "-".join(f"{k}{str(v)[:20]}" for k, v in c.items()).replace(" ", "")


def texts(n, lo, hi, seed=0, empty=0):
    """n lengths between lo and hi, every `empty`-th of them zero."""
    a = np.random.default_rng([seed, n]).integers(lo, hi + 1, n).tolist()
    return [0 if empty and i % empty == empty - 1 else x for i, x in enumerate(a)]


def run(ctx, ty, case):  # noqa: F811
    case = dict(case)
    lq, hq, hkv, D = (case.pop(n) for n in ("lq", "hq", "hkv", "D"))
    compare(ctx, ty, lq, case.pop("lk", lq), hq, hkv, D, **case)


@pytest.mark.parametrize("ty", TYPES, ids=["f32", "bf16"])
@pytest.mark.parametrize("case", [
    dict(lq=[1100, 700, 37, 300], hq=16, hkv=4, D=128),
    dict(lq=[1100, 1, 737, 300], hq=16, hkv=4, D=128, causal=True, prefix=[130, 0, 70, 299], cap=20.0),
    dict(lq=[900, 650, 37, 600], hq=16, hkv=4, D=128, causal=True, slopes=True, scale=0.2),
    dict(lq=[900, 650, 637], hq=16, hkv=8, D=128, cap=3.0, slopes=True, pad=5),
    dict(lq=[1300, 700, 100], hq=16, hkv=2, D=64, causal=True),
    dict(lq=[1300, 700, 100], lk=[1200, 900, 30], hq=16, hkv=2, D=64, causal=True, cap=20.0),   # rows before the first key
    dict(lq=[600, 300, 500], lk=[610, 0, 500], slots=[640, 64, 700], hq=24, hkv=12, D=64, slopes=True, spoil=math.nan, pad=40),
    dict(lq=[1000, 500], hq=24, hkv=24, D=40, layout="odd", causal=True),
    dict(lq=[1000, 500], hq=24, hkv=8, D=96, layout="heads", cap=100.0),
], ids=name)
def test_blocks_that_fill_the_device(ctx, ty, case):  # noqa: F811
    run(ctx, ty, case)


@pytest.mark.parametrize("ty", TYPES, ids=["f32", "bf16"])
@pytest.mark.parametrize("case", [
    dict(lq=texts(33, 20, 510), hq=12, hkv=12, D=64),                    # (bf16: four waves to a SIMD)
    dict(lq=texts(33, 20, 510, seed=1), hq=12, hkv=12, D=64, causal=True, pad=19),
    dict(lq=texts(40, 100, 400, seed=2, empty=7), hq=12, hkv=4, D=64, causal=True, prefix=[50] * 40),
], ids=name)
def test_packed_texts(ctx, ty, case):  # noqa: F811
    run(ctx, ty, case)


@pytest.mark.parametrize("ty", TYPES, ids=["f32", "bf16"])
@pytest.mark.parametrize("case", [
    dict(lq=texts(200, 1, 60), hq=6, hkv=6, D=64),
    dict(lq=texts(200, 1, 60, seed=1, empty=5), hq=6, hkv=6, D=64, causal=True, pad=77),
    dict(lq=texts(200, 1, 60, seed=2), hq=2, hkv=1, D=128, causal=True, prefix=texts(200, 0, 40, seed=3), cap=10.0),
    dict(lq=texts(150, 0, 50, seed=4), lk=texts(150, 0, 70, seed=5), slots=[80] * 150, hq=4, hkv=2, D=64, causal=True, spoil=math.nan),
    dict(lq=texts(130, 0, 90, seed=6, empty=3), lk=texts(130, 0, 90, seed=7, empty=4), hq=8, hkv=2, D=128, slopes=True),
    dict(lq=texts(120, 5, 30, seed=8), hq=16, hkv=16, D=64, causal=True),  # few rows each, and blocks that fill the device
    dict(lq=texts(120, 5, 30, seed=9), lk=texts(120, 0, 40, seed=10), slots=[41] * 120, hq=16, hkv=16, D=128, spoil=math.inf, cap=5.0),
], ids=name)
def test_blocks_of_several_documents(ctx, ty, case):  # noqa: F811
    run(ctx, ty, case)


@pytest.mark.parametrize("ty", TYPES, ids=["f32", "bf16"])
@pytest.mark.parametrize("case", [
    dict(lq=[1200], hq=8, hkv=1, D=64, causal=True),
    dict(lq=[1500, 900], hq=4, hkv=1, D=128, cap=30.0),
    dict(lq=[2000], lk=[300], hq=4, hkv=2, D=128, slopes=True),
    dict(lq=[1100, 1000], lk=[60, 200], slots=[100, 300], hq=6, hkv=1, D=96, spoil=math.nan),
], ids=name)
def test_rows_of_a_key_tile_shared_out(ctx, ty, case):  # noqa: F811
    run(ctx, ty, case)


@pytest.mark.parametrize("ty", TYPES, ids=["f32", "bf16"])
@pytest.mark.parametrize("case", [
    dict(lq=[1] * 100, lk=texts(100, 0, 70), slots=[75] * 100, hq=8, hkv=2, D=64, causal=True, spoil=math.nan),
    dict(lq=[1, 0, 1, 0] * 40, lk=texts(160, 0, 300, seed=1), hq=4, hkv=4, D=128, causal=True, cap=10.0, slopes=True),
    dict(lq=[1] * 70, lk=[600] * 69 + [9], hq=3, hkv=1, D=64),
], ids=name)
def test_one_row_each_for_more_documents_than_lanes(ctx, ty, case):  # noqa: F811
    run(ctx, ty, case)
