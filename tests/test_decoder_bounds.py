"""That the limits on the error of fp32 results (tests/_decoder.py: Q4_NORM, ATTENTION_NORM) are limits: host models of a
linear and an attention that lose bits, which the elementwise bounds let pass, are far outside them."""
import numpy as np
import pytest

import _decoder as D


@pytest.mark.parametrize("M,K,N,group,zeros", ((1, 1024, 64, 32, True), (5, 4096, 40, 64, False), (3, 8200, 24, 128, True)))
def test_q4_with_two_pieces_is_outside(M, K, N, group, zeros):
    rng = np.random.default_rng([M, K])
    x, wt = D.rows(rng, "f32", M, K), D.q4_weight(rng, K, N, group, zeros)
    w = D.q4_values(*wt, K, N, group)
    want = x.astype(np.float64) @ w
    assert np.array_equal(D.pieces(x, 3), x.astype(np.float64))
    off = D.norm_off(D.pieces(x, 2) @ w, want)
    assert off > 4 * D.Q4_NORM, off
    assert (np.abs(D.pieces(x, 2) @ w - want) <= D.q4_bound("f32", x, w, want, 1.0, K)).all()   # why the norm is asked for


@pytest.mark.parametrize("n,Dh", ((1100, 64), (300, 128), (40, 64)))
def test_attention_of_fewer_bits_is_outside(n, Dh):
    rng = np.random.default_rng([n, Dh])
    q, k, v = (D.rows(rng, "f32", m, 2, Dh) for m in (20, n, n))
    seen = np.ones((20, n), bool)
    want, bound = D.attention("f32", *(a.astype(np.float64) for a in (q, k, v)), seen, Dh ** -0.5)
    less = D.attention("f32", *(D.short(a, 16).astype(np.float64) for a in (q, k, v)), seen, Dh ** -0.5)[0]
    assert D.norm_off(less, want) > 8 * D.ATTENTION_NORM and (np.abs(less - want) <= bound).all()
    halved = np.zeros(want.shape)   # the weights rounded to fp16
    for h in range(2):
        s = q[:, h].astype(np.float64) @ k[:, h].T.astype(np.float64) * Dh ** -0.5
        w = np.exp(s - s.max(1, keepdims=True))
        halved[:, h] = (w.astype(np.float16).astype(np.float64) @ v[:, h]) / w.sum(1, keepdims=True)
    assert D.norm_off(halved, want) > 8 * D.ATTENTION_NORM
