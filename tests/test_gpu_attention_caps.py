"""Attention under caps far beyond the scores. tanh is then nearly its argument, and the scores have to keep their
bits whatever the cap: tolerances as in test_gpu_attention.py, whose float part (e) knows nothing of the cap."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_attention import TYPES, compare, ctx  # noqa: E402, F401


@pytest.mark.parametrize("ty", TYPES, ids=["f32", "bf16"])
@pytest.mark.parametrize("cap", [50.0, 65.0, 1000.0, 1e5, 1e7])
@pytest.mark.parametrize("D,slopes", [(64, False), (128, True)])
def test_caps_beyond_the_scores(ctx, ty, cap, D, slopes):  # noqa: F811
    compare(ctx, ty, [100, 31, 1], [100, 60, 900], 4, 2, D, causal=True, cap=cap, slopes=slopes)


@pytest.mark.parametrize("ty", TYPES, ids=["f32", "bf16"])
@pytest.mark.parametrize("cap", [1000.0, 1e6])
def test_single_rows(ctx, ty, cap):  # noqa: F811
    compare(ctx, ty, [1, 1, 1], [700, 33, 2500], 8, 2, 64, causal=True, cap=cap)
