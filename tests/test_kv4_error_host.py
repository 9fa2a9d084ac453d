"""The error model of kv4_error on the CPU: roundings to f16 stay below it, coarser ones and wrong scales do not."""

import numpy as np
import pytest

from kv4_error import exact_and_deviation, in_deviations


def f16(x):
    return x.astype(np.float16).astype(np.float64)


def bf16(x):
    bits = np.ascontiguousarray(x, np.float32).view(np.uint32)
    bits = (bits + 0x7FFF + ((bits >> 16) & 1)) & np.uint32(0xFFFF0000)
    return bits.view(np.float32).astype(np.float64)


def attend(q, k, v, see, scale, key=f16, value=f16, weight=f16):
    o = np.zeros_like(q)
    g = q.shape[1] // k.shape[1]
    for h in range(q.shape[1]):
        s = np.where(see, q[:, h] @ key(k[:, h // g]).T * scale, -np.inf)
        w = np.exp2((s - s.max(1, keepdims=True)) * 1.4426950408889634)
        o[:, h] = weight(w) @ value(v[:, h // g]) / w.sum(1, keepdims=True)
    return o


@pytest.fixture(scope="module")
def inputs():
    rng = np.random.default_rng(4)
    n, rows, d = 500, 6, 128
    q, k, v = (bf16(rng.standard_normal(s) * x) for s, x in (((rows, 8, d), 1.5), ((n, 2, d), 1.5), ((n, 2, d), 1.0)))
    k, v = k * 0.917, v * 0.917  # values that no format holds
    return q, k, v, np.tri(rows, n, n - rows, dtype=bool), d ** -0.5


def same(x):
    return x


MISTAKES = [
    # keys of which the model is told, what is done, below 1?
    (True, {}, True),
    (False, dict(key=same), True),
    (False, {}, False),  # keys rounded to f16 where they should enter as they are
    (True, dict(key=bf16), False),
    (True, dict(value=bf16), False),
    (True, dict(weight=bf16), False),
    (False, dict(key=same, value=bf16), False),
    (False, dict(key=same, weight=bf16), False),
]


@pytest.mark.parametrize("keys_rounded,how,below", MISTAKES)
def test_model_tells_roundings_apart(inputs, keys_rounded, how, below):
    q, k, v, see, scale = inputs
    want, dev = exact_and_deviation(q, k, v, see, scale, keys_rounded)
    off = in_deviations(attend(q, k, v, see, scale, **how), want, dev)
    assert (off < 1) == below, off


@pytest.mark.parametrize("wrong", [0.998, 1.002, 1.005])
@pytest.mark.parametrize("keys_rounded", [True, False])
def test_model_tells_a_wrong_scale(inputs, wrong, keys_rounded):
    q, k, v, see, scale = inputs
    want, dev = exact_and_deviation(q, k, v, see, scale, keys_rounded)
    assert in_deviations(attend(q, k, v, see, scale * wrong), want, dev) > 1
