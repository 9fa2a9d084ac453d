"""Sampling and verification of a batch on the GPU against float64 (tests/batch_ref.py).

Tokens and counts are equal.  Probabilities: each is a product of 2^x, off by
2^-22 and 3 u (M - l) / T (u = 2^-24), and 1 / Z, off by the bound 2^-18 at worst; the
tests allow 2^-17 of each value and 2^-120 where it is that small."""

import ctypes

import numpy as np
import pytest

import batch_ref as ref

pytestmark = pytest.mark.gpu

TYPES = ["bf16", "f16", "f32"]


def rows(n, v, dtype, seed, spread=2.0, hot=8, pad=0, at=0):
    """Logits [n, v] on the device (columns `at` .. of wider rows), and the same as float64."""
    import torch
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((n, v)) * spread
    for r in range(n):
        x[r, rng.integers(0, v, min(hot, v))] += rng.uniform(2, 12, min(hot, v))
    kind = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}[dtype]
    store = torch.full((n, v + pad + at), 100.0, dtype=kind, device="cuda")
    store[:, at:at + v] = torch.from_numpy(x).cuda()
    got = store[:, at:at + v]
    return got, got.double().cpu().numpy()


def uniforms(n, seed):
    import torch
    u = (np.random.default_rng(seed + 99).integers(0, 1 << 24, n) / (1 << 24)).astype(np.float32)
    return torch.from_numpy(u).cuda(), u


def dev(x, dtype):
    import torch
    return torch.from_numpy(np.ascontiguousarray(x, dtype)).cuda()


def check_sample(pkg, x, host, u, t, want_probs=True):
    import torch
    ts = dev(t, np.float32) if not np.isscalar(t) else t
    q = torch.full(x.shape, 7.0, device="cuda") if want_probs else None
    got = pkg.sample_rows(x, dev(u, np.float32), ts, probs_out=q)
    tokens, p = ref.sample(host, u, np.broadcast_to(t, (len(u),)))
    assert got.dtype == torch.int32 and got.tolist() == tokens
    if want_probs:
        q = q.cpu().numpy().astype(np.float64)
        assert (np.abs(q - p) <= 2.0 ** -17 * p + 2.0 ** -120).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("v", [1, 2, 7, 505, 512, 513, 1031, 4096, 32003, 128256])
def test_sample_sizes(pkg, v, dtype):
    n = 5
    x, host = rows(n, v, dtype, seed=v)
    _, u = uniforms(n, v)
    check_sample(pkg, x, host, u, np.array([1.0, 0.7, 0.0, 1.3, 0.3], np.float32))
    check_sample(pkg, x, host, u, 0.9, want_probs=False)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("pad,at", [(0, 0), (1, 0), (3, 1), (64, 0), (5, 4), (2, 3)])
def test_sample_strides(pkg, pad, at, dtype):
    import torch
    n, v = 9, 2001
    x, host = rows(n, v, dtype, seed=pad * 7 + at, pad=pad, at=at)
    _, u = uniforms(n, 5)
    check_sample(pkg, x, host, u, 1.0)
    # Probability rows of another stride, the columns between them left as they are.
    wide = torch.full((n, v + 6), -3.0, device="cuda")
    token = torch.full((n + 2,), -9, dtype=torch.int32, device="cuda")
    pkg.sample_rows(x, dev(u, np.float32), 1.0, probs_out=wide[:, 3:3 + v], tokens_out=token[:n])
    want, p = ref.sample(host, u, [1.0] * n)
    assert token.tolist() == want + [-9, -9]
    wide = wide.cpu().numpy()
    assert (wide[:, :3] == -3).all() and (wide[:, 3 + v:] == -3).all()
    assert (np.abs(wide[:, 3:3 + v] - p) <= 2.0 ** -17 * p + 2.0 ** -120).all()


@pytest.mark.parametrize("n", [1, 2, 75, 149, 300, 3000])
def test_sample_row_counts(pkg, n):
    x, host = rows(n, 1500, "bf16", seed=n)
    _, u = uniforms(n, n)
    check_sample(pkg, x, host, u, 1.0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("v", [8, 512, 1024, 65536])
def test_sample_borders(pkg, v, dtype):
    """Equal logits: every prefix is a whole number, u = k / v lies on a border and takes the token behind it."""
    import torch
    ks = np.unique(np.linspace(0, v - 1, 40).astype(int))
    kind = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}[dtype]
    x = torch.full((len(ks), v), -2.5, dtype=kind, device="cuda")
    u = (ks / v).astype(np.float32)
    assert pkg.sample_rows(x, dev(u, np.float32), 0.8).tolist() == ks.tolist()
    # One step of u below the border: the token before it.
    below = np.nextafter(u[1:], np.float32(0))
    assert pkg.sample_rows(x[1:], dev(below, np.float32), 0.8).tolist() == (ks[1:] - 1).tolist()


def test_sample_next_to_borders(pkg):
    """Uniforms as near to a cumulative weight as float32 gets, on both sides."""
    v = 3000
    x, host = rows(1, v, "f32", seed=3, spread=1.0)
    p = ref.probs(host[0], 1.0)
    c = np.cumsum(p)
    at = np.argsort(-p)[:60]
    near = c[at].astype(np.float32)
    u = np.concatenate([near, np.nextafter(near, np.float32(0)), np.nextafter(near, np.float32(1))])
    check_sample(pkg, x.expand(len(u), v).contiguous(), np.repeat(host, len(u), 0), u, 1.0, want_probs=False)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("v,spread,t", [(50001, 2.0, 0.7), (50001, 0.3, 1.0), (128256, 4.0, 1.0), (4096, 1.0, 0.3)])
def test_sample_around_borders(pkg, v, spread, t, dtype):
    """Uniforms from 2^-24 to 2^-16 off a cumulative weight, where f32 sums begin to decide."""
    x, host = rows(1, v, dtype, seed=v % 11, spread=spread)
    c = np.cumsum(ref.probs(host[0], t))
    p = np.diff(c, prepend=0.0)
    at = np.unique(np.concatenate([np.argsort(-p)[:6], np.searchsorted(c, [0.01, 0.1, 0.5, 0.9, 0.99])]))
    u = np.concatenate([c[at] + s * 2.0 ** -e for s in (-1, 1) for e in range(16, 25)]).astype(np.float32)
    check_sample(pkg, x.expand(len(u), v), np.broadcast_to(host, (len(u), v)), u, t, want_probs=False)


def test_sample_flat_rows_and_odd_uniforms(pkg):
    """A flat distribution, where f32 sums decide little; uniforms at and outside the ends."""
    x, host = rows(12, 50001, "f32", seed=11, spread=0.05, hot=0)
    u = np.array([0.0, 1.0, 1 - 2.0 ** -24, 2.0 ** -24, -0.5, 1.5, np.nan, np.inf, 0.5, 0.25, 0.999, 1e-6], np.float32)
    check_sample(pkg, x, host, u, 1.0)


@pytest.mark.parametrize("dtype", TYPES)
def test_sample_masked_values(pkg, dtype):
    import torch
    x, _ = rows(12, 1111, dtype, seed=4)
    low = float(torch.finfo(x.dtype).min)
    x[0] = -float("inf")
    x[1, 3:] = -float("inf")
    x[2] = low
    x[3, :-1] = low
    x[4, 700] = float("nan")
    x[5, 1] = float("inf")
    x[6, ::2] = -float("inf")
    x[7] = float("nan")
    x[8, 512:] = -float("inf")
    x[9, :1000] = -float("inf")
    x[10, :] = float(torch.finfo(x.dtype).max)
    x[11, 5] = float(torch.finfo(x.dtype).max)
    host = x.double().cpu().numpy()
    _, u = uniforms(12, 8)
    check_sample(pkg, x, host, u, 1.0)
    check_sample(pkg, x, host, np.zeros(12, np.float32), 0.7)
    check_sample(pkg, x, host, u, 0.0)


def test_sample_temperatures(pkg):
    t = np.array([0, 1e-45, 1e-30, 1e-3, 0.05, 1, 30, 1e8, 1e38, -1, np.nan, np.inf, -0.0], np.float32)
    x, host = rows(len(t), 2222, "f32", seed=6)
    _, u = uniforms(len(t), 6)
    check_sample(pkg, x, host, u, t)


def test_sample_far_rows(pkg):
    """Offsets past 32 bits."""
    import torch
    store = torch.empty(3, 1 << 31, dtype=torch.bfloat16, device="cuda")
    x, host = rows(3, 900, "bf16", seed=1)
    store[:, :900] = x
    q = torch.empty(3, 1 << 30, device="cuda")
    _, u = uniforms(3, 2)
    got = pkg.sample_rows(store[:, :900], dev(u, np.float32), 1.0, probs_out=q[:, :900])
    want, p = ref.sample(host, u, [1.0] * 3)
    assert got.tolist() == want
    assert (np.abs(q[:, :900].cpu().numpy() - p) <= 2.0 ** -17 * p + 2.0 ** -120).all()
    del store, q
    torch.cuda.empty_cache()


# ---------------------------------------------------------------------------
# Chains
# ---------------------------------------------------------------------------
def chains(sizes, v, dtype, seed, noise=0.6, greedy=(), **kw):
    """Drafts of sequences of `sizes` rows, drawn from a draft that mostly agrees."""
    n = sum(sizes)
    rng = np.random.default_rng(seed)
    x, host = rows(n, v, dtype, seed, **kw)
    t = rng.uniform(0.5, 1.2, n).astype(np.float32)
    for r in greedy:
        t[r] = 0
    q = np.zeros((n, v), np.float32)
    drafts = np.zeros(n, np.int32)
    for r in range(n):
        q[r] = ref.probs(host[r] + noise * rng.standard_normal(v), t[r])
        drafts[r] = ref.token(q[r].astype(np.float64), rng.random())
    start = np.concatenate([[0], np.cumsum(sizes)]).astype(np.int32)
    return x, host, t, q, drafts, start


def check_chain(pkg, x, host, t, q, drafts, u, start, q_dev=None):
    n, token = pkg.verify_drafts(x, dev(drafts, np.int32), dev(q, np.float32) if q_dev is None else q_dev,
                                 dev(u, np.float32), dev(start, np.int32), dev(t, np.float32))
    want = [ref.chain(host, drafts, q, u, t, a, b, len(host)) for a, b in zip(start[:-1], start[1:])]
    assert list(zip(n.tolist(), token.tolist())) == want
    return want


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("v", [3, 513, 2048, 32003])
def test_chain(pkg, v, dtype):
    sizes = [5, 1, 2, 9, 5, 17, 3, 5, 12, 4]
    x, host, t, q, drafts, start = chains(sizes, v, dtype, seed=v, greedy=[0, 1, 12], pad=v % 3)
    kept = 0
    for seed in range(4):
        _, u = uniforms(len(host), seed)
        kept += sum(n for n, _ in check_chain(pkg, x, host, t, q, drafts, u, start))
    assert kept > 0


def test_chain_large_vocabulary_and_many_sequences(pkg):
    x, host, t, q, drafts, start = chains([5, 3], 128256, "f32", seed=2)
    for seed in range(3):
        check_chain(pkg, x, host, t, q, drafts, uniforms(8, seed)[1], start)
    sizes = [1 + i % 4 for i in range(400)]
    x, host, t, q, drafts, start = chains(sizes, 700, "bf16", seed=3)
    check_chain(pkg, x, host, t, q, drafts, uniforms(len(host), 1)[1], start)


def test_chain_at_the_border(pkg):
    """Uniforms as near to p / q as float32 gets: the comparison is that of 64 bits."""
    n = 64
    x, host, t, q, drafts, start = chains([2] * (n // 2), 1200, "f32", seed=5, spread=1.0)
    u = np.zeros(n, np.float32)
    for r in range(0, n, 2):
        d = drafts[r]
        near = np.float32(min(ref.probs(host[r], t[r])[d] / float(q[r, d]), 1.0))
        u[r] = [near, np.nextafter(near, np.float32(0)), np.nextafter(near, np.float32(2))][r // 2 % 3]
        u[r + 1] = 0.37
    check_chain(pkg, x, host, t, q, drafts, u, start)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("noise", [0.05, 1.5])
def test_chain_around_borders_of_the_rest(pkg, noise, dtype):
    """Rejected drafts; the next uniform 2^-24 to 2^-12 off a cumulative weight of max(p - q, 0)."""
    v, n = 20000, 128
    x, host, t, q, drafts, start = chains([2] * (n // 2), v, dtype, seed=13, noise=noise)
    u = np.ones(n, np.float32)
    for i, r in enumerate(range(0, n, 2)):
        p = ref.probs(host[r], t[r])
        drafts[r] = int(np.argmax(q[r] - p))
        rest = np.fmax(p - q[r].astype(np.float64), 0.0)
        c = np.cumsum(rest) / rest.sum()
        k = np.argsort(-rest)[i % 7] if i % 2 else np.searchsorted(c, (i + 0.5) / (n // 2))
        u[r + 1] = np.clip(c[k] + (-1) ** (i // 2) * 2.0 ** -(12 + i % 13), 0, 1)
    want = check_chain(pkg, x, host, t, q, drafts, u, start)
    assert all(k == 0 for k, _ in want)


def test_chain_draft_equal_to_the_target(pkg):
    """q is p rounded to f32: next to nothing is left of max(p - q, 0)."""
    sizes = [4] * 8
    x, host, t, q, drafts, start = chains(sizes, 5000, "f32", seed=7, noise=0.0)
    u = np.full(len(host), 1.0 - 2.0 ** -24, np.float32)
    check_chain(pkg, x, host, t, q, drafts, u, start)
    check_chain(pkg, x, host, t, q * np.float32(1.5), drafts, u, start)  # p is above q nowhere: p itself
    for seed in range(3):
        check_chain(pkg, x, host, t, q * np.float32(1.0 + 2.0 ** -20), drafts, uniforms(len(host), seed)[1], start)


def test_chain_odd_drafts_and_probabilities(pkg):
    sizes = [4] * 10
    v = 1500
    x, host, t, q, drafts, start = chains(sizes, v, "bf16", seed=9)
    drafts[0], drafts[5], drafts[10] = -1, v, 2 ** 31 - 1  # no tokens: the drafts end there
    q[12, drafts[12]] = 0.0     # kept
    q[16, drafts[16]] = -1.0    # kept
    q[20, drafts[20]] = np.nan  # not kept, nor drawn
    q[24, :] = np.nan           # likewise, and nothing is left: p itself
    q[28, drafts[28]] = np.inf
    x[33, 7] = float("nan")     # no distribution
    x[36] = -float("inf")
    host = x.double().cpu().numpy()
    for seed in range(3):
        check_chain(pkg, x, host, t, q, drafts, uniforms(len(host), seed)[1], start)
    check_chain(pkg, x, host, t, q, drafts, np.zeros(len(host), np.float32), start)


def test_chain_row_starts(pkg):
    x, host, t, q, drafts, _ = chains([12], 800, "f32", seed=10)
    _, u = uniforms(12, 3)
    for start in ([0, 5, 5, 12], [2, 4, 9], [0, 13], [-1, 4, 6], [7, 3, 6], [2 ** 31 - 1, 0], [12, 12], [0]):
        check_chain(pkg, x, host, t, q, drafts, u, np.array(start, np.int32))


def test_chain_strided_probabilities(pkg):
    import torch
    x, host, t, q, drafts, start = chains([5, 4, 6], 1001, "f16", seed=12, pad=3)
    _, u = uniforms(len(host), 4)
    for at, width in ((0, 1004), (1, 1003), (2, 2000)):
        store = torch.full((len(host), width + at), float("nan"), device="cuda")
        store[:, at:at + 1001] = dev(q, np.float32)
        check_chain(pkg, x, host, t, q, drafts, u, start, q_dev=store[:, at:at + 1001])


# ---------------------------------------------------------------------------
# Trees
# ---------------------------------------------------------------------------
def trees(sizes, v, dtype, seed, **kw):
    n = sum(sizes)
    rng = np.random.default_rng(seed)
    x, host = rows(n, v, dtype, seed, **kw)
    parents, tokens, at = [], [], 0
    for m in sizes:
        seen = [0] * m
        for i in range(m):
            p = 0 if i == 0 else int(rng.integers(max(0, i - 6), i))
            parents.append(p)
            best = np.argsort(-host[at + p], kind="stable")
            tokens.append(0 if i == 0 else int(best[min(seen[p], v - 1)]))
            seen[p] += i > 0
        at += m
    t = rng.uniform(0.3, 1.0, n).astype(np.float32)
    start = np.concatenate([[0], np.cumsum(sizes)]).astype(np.int32)
    return x, host, t, np.array(tokens, np.int32), np.array(parents, np.int32), start


def check_tree(pkg, x, host, t, tokens, parents, u, start):
    path, n, token = pkg.verify_trees(x, dev(tokens, np.int32), dev(parents, np.int32), dev(u, np.float32),
                                      dev(start, np.int32), dev(t, np.float32))
    want_path = np.full(len(host), -1)
    lens = []
    for b, (a, e) in enumerate(zip(start[:-1], start[1:])):
        way, nxt = ref.tree(host, tokens, parents, u, t, a, e, len(host))
        want_path[a:a + len(way)] = way
        assert int(n[b]) == len(way) and int(token[b]) == nxt
        lens.append(len(way))
    assert path.tolist() == want_path.tolist()
    return lens


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("v", [4, 600, 32003])
def test_tree(pkg, v, dtype):
    sizes = [1, 60, 7, 31, 2, 64, 13, 200]
    x, host, t, tokens, parents, start = trees(sizes, v, dtype, seed=v, pad=v % 2)
    t[::5] = 0
    deep = 0
    for seed in range(3):
        deep = max([deep] + check_tree(pkg, x, host, t, tokens, parents, uniforms(len(host), seed)[1], start))
    assert deep > 2


def test_tree_long_chain_and_flat_rows(pkg):
    """300 drafts in a row at temperature 0, and rows that f32 does not decide on the way."""
    m = 301
    x, host, t, tokens, parents, start = trees([m], 3001, "f32", seed=3, spread=0.02, hot=0)
    parents = np.arange(-1, m - 1)
    parents[0] = 0
    _, u = uniforms(m, 1)
    t[:] = np.where(np.arange(m) % 3 == 0, 1.0, 0.0)
    tokens[1:] = [ref.token(ref.probs(host[i], t[i]), u[i]) for i in range(m - 1)]
    assert check_tree(pkg, x, host, t, tokens, parents, u, start) == [m]


def test_tree_odd_trees(pkg):
    """Twins (the first one counts), parents that come later or are none, tokens outside the vocabulary, bad rows."""
    x, host, t, tokens, parents, start = trees([20, 20, 20, 20], 500, "bf16", seed=8)
    t[:] = 0
    best = host.argmax(1)
    tokens[1], parents[1], tokens[2], parents[2] = best[0], 0, best[0], 0
    tokens[3], parents[3] = best[1], 1
    tokens[23], parents[23] = best[20], 7  # its parent comes later
    parents[25:28] = [-1, 2 ** 31 - 1, 100]
    tokens[40:60] = -1
    x[60, 3] = float("nan")
    host = x.double().cpu().numpy()
    check_tree(pkg, x, host, t, tokens, parents, uniforms(80, 1)[1], start)
    for odd in ([0, 80, 80], [3, 1], [0, 81], [-4, 10, 20], [10, 30]):
        check_tree(pkg, x, host, t, tokens, parents, uniforms(80, 1)[1], np.array(odd, np.int32))


# ---------------------------------------------------------------------------
# Calls as a server makes them
# ---------------------------------------------------------------------------
def test_calls_are_captured_and_replayed(pkg):
    """A draft step and a verification in a graph, replayed on new contents, next to eager calls on another stream."""
    import torch
    sizes = [4] * 6
    x, host, t, q, drafts, start = chains(sizes, 2100, "bf16", seed=1)
    n = len(host)
    bx, bq, bd = x.clone(), dev(q, np.float32), dev(drafts, np.int32)
    bu, bt, bs = dev(np.zeros(n), np.float32), dev(t, np.float32), dev(start, np.int32)
    probs = torch.zeros_like(bq)

    def step():
        return (pkg.sample_rows(bx, bu, bt, probs_out=probs), *pkg.verify_drafts(bx, bd, bq, bu, bs, bt))

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        out = step()
    for seed in range(3):
        x2, host2, t2, q2, drafts2, _ = chains(sizes, 2100, "bf16", seed=seed + 20)
        _, u = uniforms(n, seed)
        bx.copy_(x2), bq.copy_(dev(q2, np.float32)), bd.copy_(dev(drafts2, np.int32))
        bu.copy_(dev(u, np.float32)), bt.copy_(dev(t2, np.float32))
        torch.cuda.synchronize()
        g.replay()
        with torch.cuda.stream(side):
            y = pkg.sample_rows(x, bu, 1.0)  # another call at the same time, with a workspace of its own
        torch.cuda.synchronize()
        assert out[0].tolist() == ref.sample(host2, u, t2)[0]
        want = [ref.chain(host2, drafts2, q2, u, t2, a, b, n) for a, b in zip(start[:-1], start[1:])]
        assert list(zip(out[1].tolist(), out[2].tolist())) == want
        assert y.tolist() == ref.sample(host, u, [1.0] * n)[0]


def test_results_do_not_depend_on_the_batch(pkg):
    """A row alone, in a batch and in another order gives the same token and the same bits."""
    import torch
    x, host = rows(40, 5003, "f32", seed=2)
    u, _ = uniforms(40, 2)
    q = torch.empty(40, 5003, device="cuda")
    both = pkg.sample_rows(x, u, 0.8, probs_out=q)
    for r in (0, 17, 39):
        one = torch.empty(1, 5003, device="cuda")
        assert pkg.sample_rows(x[r:r + 1], u[r:r + 1], 0.8, probs_out=one).tolist() == [int(both[r])]
        assert torch.equal(one[0], q[r])


def test_refusals(pkg):
    import torch
    x, _ = rows(4, 100, "f32", seed=0)
    u, i = torch.zeros(4, device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda")
    q, s = torch.zeros(4, 100, device="cuda"), torch.tensor([0, 4], dtype=torch.int32, device="cuda")
    bad = [lambda: pkg.sample_rows(x.double(), u), lambda: pkg.sample_rows(x[0], u), lambda: pkg.sample_rows(x, u[:3]),
           lambda: pkg.sample_rows(x, u.double()), lambda: pkg.sample_rows(x, u.cpu()), lambda: pkg.sample_rows(x.T, u),
           lambda: pkg.sample_rows(x, u, -1.0), lambda: pkg.sample_rows(x, u, float("nan")),
           lambda: pkg.sample_rows(x, u, u[:2]), lambda: pkg.sample_rows(x, u, probs_out=q[:3]),
           lambda: pkg.sample_rows(x, u, probs_out=q[:1].expand(4, 100)), lambda: pkg.sample_rows(x, u, probs_out=q.half()),
           lambda: pkg.sample_rows(x, u, tokens_out=i.long()), lambda: pkg.sample_rows(x, u, tokens_out=i[::2]),
           lambda: pkg.verify_drafts(x, i[:3], q, u, s), lambda: pkg.verify_drafts(x, i, q[:, :99], u, s),
           lambda: pkg.verify_drafts(x, i, q, u, s.long()), lambda: pkg.verify_drafts(x, i, q, u, s[:0]),
           lambda: pkg.verify_drafts(x, i, q, u, s[:, None]), lambda: pkg.verify_trees(x, i, i[:2], u, s),
           lambda: pkg.verify_trees(x, i.float(), i, u, s), lambda: pkg.verify_trees(x, i, i, u, 3)]
    for call in bad:
        with pytest.raises(pkg.SamplingError):
            call()
    empty = torch.empty(0, 100, device="cuda")
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    assert pkg.sample_rows(empty, u[:0]).numel() == 0
    n, token = pkg.verify_drafts(empty, none, empty, u[:0], torch.zeros(3, dtype=torch.int32, device="cuda"))
    assert n.tolist() == [0, 0] and token.tolist() == [-1, -1]
    path, n, token = pkg.verify_trees(empty, none, none, u[:0], torch.zeros(2, dtype=torch.int32, device="cuda"))
    assert path.numel() == 0 and n.tolist() == [0] and token.tolist() == [-1]


@pytest.mark.parametrize("dtype", TYPES)
def test_tree_without_sequences(pkg, dtype):
    """Rows that belong to no sequence: their path is -1, nothing else is written."""
    import torch
    n, v = 300, 700
    x, _ = rows(n, v, dtype, seed=3)
    zeros, u = torch.zeros(n, dtype=torch.int32, device="cuda"), torch.zeros(n, device="cuda")
    junk = [torch.full((n,), 5, dtype=torch.int32, device="cuda") for _ in range(4)]  # what a new tensor may hold
    del junk
    for start in ([0], [n], [-1]):
        path, count, token = pkg.verify_trees(x, zeros, zeros, u, dev(start, np.int32))
        assert path.tolist() == [-1] * n and count.numel() == token.numel() == 0
    # The same through the C entry, into the middle of other memory.
    lib = pkg.load()
    from importlib import import_module
    _lib = import_module("abyo-speculate_b200._lib")
    kind = TYPES.index(dtype)
    need = lib.spec_batch_workspace_bytes(n, v, kind)
    work = torch.empty(need, dtype=torch.uint8, device="cuda")
    a = _lib.BatchLogits(device=0, vocab=v, dtype=kind, temperature=1.0, logits=x.data_ptr(), row_stride=x.stride(0), n_rows=n,
                         temperatures=None, uniforms=u.data_ptr(), workspace=work.data_ptr(), workspace_bytes=need)
    wide = torch.full((n + 2,), 7, dtype=torch.int32, device="cuda")
    stream = torch.cuda.current_stream().cuda_stream
    assert lib.spec_batch_verify_tree(ctypes.byref(a), 0, None, None, None, wide[1:].data_ptr(), None, None, stream) == 0
    assert wide.tolist() == [7] + [-1] * n + [7]
    # And captured.
    g = torch.cuda.CUDAGraph()
    start = dev([0], np.int32)
    with torch.cuda.graph(g):
        path, _, _ = pkg.verify_trees(x, zeros, zeros, u, start)
    path.fill_(3)
    g.replay()
    assert path.tolist() == [-1] * n


def test_probabilities_beside_the_logits(pkg):
    """Columns of one tensor, and rows in turn; not the logits' own memory."""
    import torch
    n, v = 6, 300
    x, host = rows(n, v, "f32", seed=1)
    _, u = uniforms(n, 4)
    tokens, p = ref.sample(host, u, np.ones(n))
    one = torch.cat([x, torch.zeros(n, v, device="cuda")], 1)
    turns = torch.stack([x, torch.zeros(n, v, device="cuda")], 1).reshape(2 * n, v)
    for logits, q in ((one[:, :v], one[:, v:]), (turns[0::2], turns[1::2])):
        assert pkg.sample_rows(logits, dev(u, np.float32), probs_out=q).tolist() == tokens
        assert (np.abs(q.cpu().numpy().astype(np.float64) - p) <= 2.0 ** -17 * p + 2.0 ** -120).all()
        with pytest.raises(pkg.SamplingError):
            pkg.sample_rows(logits, dev(u, np.float32), probs_out=logits)


@pytest.mark.parametrize("m", [512, 513, 700])
def test_trees_of_very_many_nodes(pkg, m):
    """Nodes behind the first 512: a path through all of them, one that ends behind them, and a bush whose child is its last."""
    x, host, t, tokens, parents, start = trees([m, m, m], 900, "f16", seed=m, spread=0.3, hot=2)
    _, u = uniforms(3 * m, 2)
    t[:] = np.where(np.arange(3 * m) % 7 == 0, 1.0, 0.0)
    drawn = [ref.token(ref.probs(host[i], t[i]), u[i]) for i in range(3 * m)]
    for b, length in ((0, m), (1, m - 20)):
        parents[b * m + 1:(b + 1) * m] = np.arange(m - 1)
        tokens[b * m + 1:b * m + length] = drawn[b * m:b * m + length - 1]
        tokens[b * m + length:(b + 1) * m] = -1
    parents[2 * m:] = 0
    tokens[2 * m:] = (drawn[2 * m] + 1) % 900
    tokens[3 * m - 1] = drawn[2 * m]
    assert check_tree(pkg, x, host, t, tokens, parents, u, start) == [m, m - 20, 2]


@pytest.mark.parametrize("dtype", TYPES)
def test_the_largest_vocabulary(pkg, dtype):
    import torch
    v = 1 << 20
    x, host = rows(6, v, dtype, seed=7, spread=1.0)
    _, u = uniforms(6, 3)
    u[1], u[2] = 1.0, 0.0
    t = np.array([1.0, 1.0, 1.0, 0.0, 0.4, 2.0], np.float32)
    check_sample(pkg, x, host, u, t)
    with pytest.raises(pkg.SamplingError):
        pkg.sample_rows(torch.zeros(1, v + 1, device="cuda"), dev(u[:1], np.float32))
    q = np.stack([ref.probs(h, 1.0) for h in host * 0.9]).astype(np.float32)
    drafts = np.array([int(np.argmax(h)) for h in host], np.int32)
    check_chain(pkg, x, host, t, q, drafts, u, np.array([0, 3, 6], np.int32))
    check_tree(pkg, x, host, t, np.array([0, drafts[0], 5, 0, drafts[3], 1], np.int32), np.array([0, 0, 0, 0, 0, 1], np.int32), u,
               np.array([0, 3, 6], np.int32))


def test_the_most_rows(pkg):
    """2^20 rows, and as many sequences."""
    import torch
    n = 1 << 20
    gen = torch.Generator(device="cuda").manual_seed(1)
    best = torch.randint(0, 3, (n,), device="cuda", generator=gen)
    x = torch.zeros(n, 3, device="cuda").scatter_(1, best[:, None], 60.0)
    u = torch.rand(n, device="cuda", generator=gen)
    want = best.to(torch.int32)
    q = torch.empty(n, 3, device="cuda")
    assert torch.equal(pkg.sample_rows(x, u, probs_out=q), want) and (q.argmax(1) == best).all()
    start = torch.arange(n + 1, dtype=torch.int32, device="cuda")
    zeros = torch.zeros(n, dtype=torch.int32, device="cuda")
    count, token = pkg.verify_drafts(x, zeros, q, u, start)
    assert not count.any() and torch.equal(token, want)
    path, count, token = pkg.verify_trees(x, zeros, zeros, u, start)
    assert not path.any() and (count == 1).all() and torch.equal(token, want)
    with pytest.raises(pkg.SamplingError):
        pkg.sample_rows(torch.zeros(n + 1, 3, device="cuda"), torch.zeros(n + 1, device="cuda"))
