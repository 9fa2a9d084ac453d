"""The rules of spec_batch_* (include/spec_b200.h) in float64, row by row, on numpy arrays."""

import numpy as np


def probs(logits, t):
    """The row's distribution, or None where it has none."""
    x = np.asarray(logits, np.float64)
    t = float(np.float32(t))
    if not (0 <= t < np.inf) or np.isnan(x).any() or np.isinf(x.max()):
        return None
    if t == 0:
        p = np.zeros_like(x)
        p[int(np.argmax(x))] = 1.0  # the first of them
        return p
    t = min(max(t, 2.0 ** -60), 2.0 ** 60)
    with np.errstate(over="ignore"):
        w = np.exp((x - x.max()) / t)
    return w / w.sum()


def unit(u):
    u = float(u)
    return 0.0 if np.isnan(u) else min(max(u, 0.0), 1.0)


def token(p, u):
    c = np.cumsum(p)
    at = np.flatnonzero(c > unit(u) * c[-1])
    return int(at[0]) if at.size else int(np.flatnonzero(p > 0)[-1])


def sample(logits, us, ts):
    out = []
    for x, u, t in zip(logits, us, ts):
        p = probs(x, t)
        out.append((-1, np.zeros(len(x))) if p is None else (token(p, u), p))
    return [a for a, _ in out], np.stack([b for _, b in out])


def chain(logits, drafts, q, us, ts, first, end, n_rows):
    """(kept drafts, next token) of the sequence with rows first .. end - 1."""
    if not (0 <= first < end <= n_rows):
        return 0, -1
    v = logits.shape[1]
    for r in range(first, end):
        p = probs(logits[r], ts[r])
        n = r - first
        if p is None:
            return n, -1
        d = int(drafts[r]) if r + 1 < end else -1
        if not 0 <= d < v:
            return n, token(p, us[r])
        qx = float(q[r, d])
        if qx <= 0 or unit(us[r]) * qx <= p[d]:
            continue
        rest = np.fmax(p - q[r].astype(np.float64), 0.0)
        return n, token(rest if rest.sum() > 0 else p, us[r + 1])
    raise AssertionError("the last row judges no draft")


def tree(logits, tokens, parents, us, ts, first, end, n_rows):
    """(path, next token)."""
    if not (0 <= first < end <= n_rows):
        return [], -1
    path = [0]
    while True:
        p = probs(logits[first + path[-1]], ts[first + path[-1]])
        if p is None:
            return path, -1
        x = token(p, us[first + path[-1]])
        below = [i for i in range(path[-1] + 1, end - first) if parents[first + i] == path[-1] and tokens[first + i] == x]
        if not below:
            return path, x
        path.append(below[0])
