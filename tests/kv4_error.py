"""What the 4-bit attention's f32 outputs should be off by from float64, as a standard deviation.

Rounding x to f16 moves it by an error of mean 0 and a deviation of at most
|x| 2^-11 / sqrt(3) (uniform over a unit in the last place, which is at most
2^-10 |x|).  With weights w and o = sum w v:
  values and weights rounded once each: sqrt(2 sum w^2 v^2) of these,
  keys rounded once: scores are off by scale sqrt(sum q^2 k^2) of these, and
  a score's error moves o by w (v - o).
f32 sums, exponentials and q's exact scaling add less than a hundredth of it."""

import numpy as np

ROUNDING = 2.0 ** -11 / np.sqrt(3.0)


def exact_and_deviation(q, k, v, see, scale, keys_rounded):
    """q [rows, heads, d], k, v [tokens, kv heads, d] in float64, see [rows, tokens] how
    often a row sees a token (a token's errors are alike each time) -> o, deviation."""
    rows, heads, d = q.shape
    g = heads // k.shape[1]
    o, dev = np.zeros_like(q), np.zeros_like(q)
    for h in range(heads):
        kk, vv = k[:, h // g], v[:, h // g]
        s = np.where(see, q[:, h] @ kk.T * scale, -np.inf)
        w = see * np.exp(s - s.max(1, keepdims=True))
        w /= w.sum(1, keepdims=True)
        o[:, h] = w @ vv
        var = 2 * (w ** 2 @ vv ** 2)
        if keys_rounded:
            moved = w ** 2 * (q[:, h] ** 2 @ (kk ** 2).T * scale ** 2)
            # sum of moved (v - o)^2
            var += moved @ vv ** 2 - 2 * o[:, h] * (moved @ vv) + o[:, h] ** 2 * moved.sum(1, keepdims=True)
        dev[:, h] = ROUNDING * np.sqrt(np.maximum(var, 0))
    return o, dev


def in_deviations(got, want, dev):
    """Root mean square error in units of the deviation: below 1 where the roundings are those and no more."""
    at = dev > 0
    return float(np.sqrt(np.mean(((got - want)[at] / dev[at]) ** 2)))
