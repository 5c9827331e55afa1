"""What pins the oracle of rotary positions and linear attention (CPU)."""

from __future__ import annotations

import numpy as np
import pytest

from oracle import layer_oracle as L


@pytest.mark.parametrize("pairing", ["half", "adjacent"])
@pytest.mark.parametrize("d,rot", [(32, 32), (128, 64), (128, 126), (256, 64)])
def test_rope_fp32_against_complex_64(pairing, d, rot):
    rng = np.random.default_rng(d + rot)
    x = rng.standard_normal((9, 3, d)).astype(np.float16)
    pos = rng.integers(0, 500, (1, 9))
    w = (1 + 0.2 * rng.standard_normal(d)).astype(np.float32)
    table = L.cos_sin_table(512, rot)
    for norm in (None, w):
        got = L.rope(x, pos, table, pairing=pairing, norm=norm)
        want = L.rope_f64(x, pos, table, pairing=pairing, norm=norm)
        # two products and a sum: 3 half steps of 2^-24 of |a| + |b| <= 2 max; the norm's tree (log2 D + 4 roundings)
        assert np.abs(got - want).max() <= (3 + (12 if norm is not None else 0)) * 2.0 ** -24 * 2 * np.abs(want).max()


def test_rope_properties():
    rng = np.random.default_rng(5)
    x = rng.standard_normal((4, 2, 64))
    table = L.cos_sin_table(100, 64).astype(np.float64)
    zero = L.rope_f64(x, np.zeros((1, 4), int), table)
    assert np.array_equal(zero, x)  # position 0 turns nothing
    # a rotation keeps each pair's length, and q.k depends on the positions' difference alone
    a = L.rope_f64(x, np.array([[3, 7, 11, 20]]), table)
    assert np.allclose((a ** 2).sum(-1), (x ** 2).sum(-1), rtol=1e-6)
    y = rng.standard_normal((4, 2, 64))
    dots = [(L.rope_f64(x, np.full((1, 4), p), table) * L.rope_f64(y, np.full((1, 4), p + 5), table)).sum(-1)
            for p in (0, 13, 60)]
    assert np.allclose(dots[0], dots[1], atol=1e-5) and np.allclose(dots[0], dots[2], atol=1e-5)


def test_axes():
    assert L.axis_of_pair((2, 3, 3), False, 8).tolist() == [0, 0, 1, 1, 1, 2, 2, 2]
    assert L.axis_of_pair((4, 2, 2), True, 8).tolist() == [0, 1, 2, 0, 1, 2, 0, 0]
    table = L.cos_sin_table(64, 16)
    x = np.random.default_rng(1).standard_normal((3, 1, 16))
    same = np.array([[4, 9, 30]] * 3)
    # equal positions on every axis are the one-axis rotation
    assert np.array_equal(L.rope(x, same, table, sections=(2, 3, 3)), L.rope(x, same[:1], table))
    moved = same.copy()
    moved[1] += 1
    d = L.rope(x, moved, table, sections=(2, 3, 3)) != L.rope(x, same, table, sections=(2, 3, 3))
    assert d.any(0)[0].nonzero()[0].tolist() == [2, 3, 4, 10, 11, 12]  # the height pairs' dims
    bad = L.rope(x, np.array([[-1, 64, 3]]), table)
    assert np.isnan(bad[:2]).all() and np.isfinite(bad[2]).all()


def test_linear_attention_against_the_masked_product():
    rng = np.random.default_rng(2)
    n, h, d = 40, 4, 8
    q, k, v = (rng.standard_normal((n, hh, d)) for hh in (h, 2, 2))
    g = np.array([0.0, -0.1, -2.0, -np.inf])
    s0 = rng.standard_normal((h, d, d))
    out, s = L.linear_attention(q, k, v, g, s0, 0.5)
    i = np.arange(n)
    ago = i[:, None] - i
    for a in range(h):
        with np.errstate(invalid="ignore"):
            decay = np.where(ago > 0, np.exp(g[a] * np.maximum(ago, 1)), (ago == 0) * 1.0)
        kk, vv = k[:, a // 2], v[:, a // 2]
        want = 0.5 * ((q[:, a] @ kk.T * decay) @ vv + np.exp(g[a] * (i + 1))[:, None] * (q[:, a] @ s0[a]))
        assert np.allclose(out[:, a], want, rtol=1e-10, atol=1e-12)
        assert np.allclose(s[a], np.exp(g[a] * n) * s0[a] + (kk * decay[-1][:, None]).T @ vv, rtol=1e-10, atol=1e-12)
