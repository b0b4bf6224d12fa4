"""Attention over the 8-bit cache rounds a bf16 output once, whatever a request is called with: probabilities times values'
scales enter the products as two bf16 terms in blocks of any width.

Tolerance per element, u = 2^-8 bf16's unit roundoff: two terms leave u^2 of each product p vs, the float sums e of
w = sum_j p_j |v_j| (as in test_gpu_cache), and o is rounded once: u |o| + (1 + u) (u^2 + e) w. Scores are kept small, so that
e stays near u^2 and one rounding of p vs, u of it, stands out where o is small against w.
"""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_cache import coded, empty, ints, oracle  # noqa: E402

U = 2.0 ** -8


@pytest.fixture(scope="module")
def ctx():
    from brosoundml_amd import native
    return native.Context(0)


@pytest.mark.parametrize("hq,hkv,D", [(16, 4, 128), (12, 12, 64), (40, 1, 40), (17, 1, 128)])
@pytest.mark.parametrize("lq,lk", [([1, 1, 1], [9, 40, 300]), ([1, 90, 33], [40, 290, 33]), ([3], [700]), ([200], [260])],
                         ids=["steps", "a step beside pieces", "few rows", "a piece"])
@pytest.mark.parametrize("cap", [0.0, 5.0])
def test_outputs_are_rounded_once(ctx, hq, hkv, D, lq, lk, cap):
    from brosoundml_amd import tokens
    rng = np.random.default_rng([sum(lq), sum(lk), hq, D])
    mk = lambda n, h, std: torch.from_numpy((std * rng.standard_normal((n, h, D))).astype(np.float32))  # noqa: E731
    k_off = np.concatenate([[0], np.cumsum(lk)]).tolist()
    cache = empty(k_off[-1], hkv, D, "both")
    for codes, scales in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        s, c = coded(mk(k_off[-1], hkv, 1.0))
        codes[..., :D], codes[..., D:] = c.to(torch.int8).cuda(), 0
        scales.copy_(s.t())
    q = mk(sum(lq), hq, 0.02).bfloat16().cuda()
    o, _ = tokens.cache_attention(ctx, q, cache, ints(np.concatenate([[0], np.cumsum(lq)])), ints(k_off), causal=True, cap=cap)
    want, w, _, e = oracle(q, cache, D, lq, k_off, None, True, None, D ** -0.5, cap, None)
    off, tol = (o.double().cpu() - want).abs(), U * want.abs() + (1 + U) * (U * U + e) * w + 1e-30
    assert (off <= tol).all(), (float((off / tol).max()), int((off > tol).sum()))
