"""The running reference of the 4-bit attention's kernel for many columns, restated in f32.

Per stage of 128 tokens a column's weights are made against its last reference
and, where the largest exponent passes the slack, once more against the moved reference.  From
2^20 on scores are rounded before the reference is taken off them: below, what
roundings leave of the largest exponent is at most an eighth; above, it would
be octaves."""

import numpy as np
import pytest

F32, F64, EXT = np.float32, np.float64, np.longdouble
SLACK, FAR = F32(8.0), F32(2.0 ** 20)


def fma(x, c, b):
    """x c + b rounded once (a product of f32 has 48 bits; the sum in 64 of them)."""
    return (np.asarray(x, EXT) * EXT(c) + EXT(b)).astype(F32)


def column(stages, c):
    """Scores of one column by stages -> (reference, sum of weights, weights against it)."""
    m, total, weights = None, F64(0), []
    for x in stages:
        base = F32(0) if m is None else m
        exponents = fma(x, c, -base)
        best = exponents.max()
        over = m is None or best > SLACK
        if over or abs(base) >= FAR:
            moved = base + best if over else m
            far = abs(base) >= FAR or abs(moved) >= FAR
            if far:
                scores = x * c
                over = m is None or scores.max() - base > SLACK
                moved = scores.max() if over else m
            by = F64(0) if m is None else np.exp2(F64(m) - F64(moved))
            total, weights, m = total * by, [w * by for w in weights], moved
            exponents = scores - m if far else fma(x, c, -m)
        w = np.exp2(exponents.astype(F64))
        assert w.max() <= 2.0 ** 8  # f16 holds it
        total += w.sum()
        weights.append(w)
    return m, total, np.concatenate(weights)


@pytest.mark.parametrize("octaves", [1.0, 1e3, 1e5, 2.0 ** 20, 1e7, 1e8, 3e8, 8e8, 1e9, 3e9, 1e11, 1e12, 1e20, 1e30])
@pytest.mark.parametrize("sign", [1, -1])
def test_two_passes_agree_with_float64(octaves, sign):
    """Ends, and gives the softmax of scores that are off by their f32 rounding alone."""
    rng = np.random.default_rng(int(np.log2(octaves) * 7) + 2 + sign)
    for trial in range(40):
        c = F32(0.1 + rng.random())
        x = (rng.standard_normal((4, 128)) * octaves * np.array([0.2, 1, 0.5, 2])[:, None]).astype(F32)
        if sign < 0:  # all below zero
            x = x - x.max() - F32(octaves)
        m, total, w = column(list(x), c)
        exact = x.reshape(-1).astype(EXT) * EXT(c)
        off = np.abs(exact).max() * EXT(2.0 ** -23)  # how far a score may be moved by roundings
        gap = exact - exact.max()
        share = (w / total).astype(EXT)
        assert np.isfinite(total) and total >= 2.0 ** -1
        # Weights of scores that lie further below the largest than roundings reach.
        some = share > 1e-290  # normal numbers of float64
        assert (np.log2(share[some]) <= gap[some] + 2 * off + 1e-3).all()
        if off < 1e-3:
            want = np.exp2(gap) / np.exp2(gap).sum()
            assert np.abs(share - want).max() <= 4 * off + 1e-6
        clear = gap < -(2 * off + 60)
        if clear.sum() == clear.size - 1:
            assert share[np.argmax(exact)] > 1 - 1e-6


@pytest.mark.parametrize("score", [1.0, 1e6, 3e8, 1e9, 3e9, 1e12, -1e9, -1e12])
def test_equal_scores_share_alike(score):
    """However far from zero, equal scores have the largest exponent 0 (an eighth at most below 2^20)."""
    rng = np.random.default_rng(3)
    for _ in range(50):
        c, x = F32(0.1 + rng.random()), F32(score * (1 + rng.random()))
        m, total, w = column([np.full(128, x), np.full(128, x)], c)
        assert (w == w[0]).all() and 2.0 ** -0.125 <= w[0] <= 2.0 ** 0.125
