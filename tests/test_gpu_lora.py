"""Low-rank adapters of many requests on the GPU against float64.

Tolerances, with u = 2^-24, |.| sums of magnitudes: t = x A^T has f32 sums of k
terms, taken by the tensor core in blocks of 8 or 16, which may drop what lies
below 2^-23 of the running sum at every step: |dt| <= 2^-23 (k / 8 + 32) |x| |A|
(operands exact, or f32 rows as two tf32 numbers, 2^-24 more).  The second
product likewise over the rank, t split into parts that leave 2^-22 of the
row's largest (f16), 2^-16 (bf16 for a bf16 result) or 2^-24 (bf16 for f32).  The
result is rounded once to its type.  The bound is the worst case, so the norm
of the error is checked too, against a sixteenth of it."""

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

EPS = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11, "f32": 2.0 ** -24}


def kinds():
    import torch
    return {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def dev(x, dtype):
    import torch
    return torch.from_numpy(np.ascontiguousarray(x, np.float32)).cuda().to(kinds()[dtype])


class Case:
    """A bank, rows and their adapters; views into wider memory where `pad` says so."""

    def __init__(self, pkg, ids, n_adapters, k, n, rank, dtype="bf16", x="same", y="same", ranks=None, scaled=True, seed=0,
                 pad=(0, 0, 0, 0)):
        import torch
        rng = np.random.default_rng(seed)
        self.pkg, self.ids, self.dtype = pkg, np.asarray(ids), dtype
        self.xt, self.yt = (dtype if x == "same" else "f32"), (dtype if y == "same" else "f32")
        rows = len(ids)

        def view(a, kind, extra):
            t = torch.full((*a.shape[:-1], a.shape[-1] + extra), float("nan"), dtype=kinds()[kind], device="cuda")
            t[..., :a.shape[-1]] = dev(a, kind)
            return t[..., :a.shape[-1]]

        self.a = view(rng.standard_normal((n_adapters, rank, k)) / np.sqrt(k), dtype, pad[0])
        self.b = view(rng.standard_normal((n_adapters, n, rank)), dtype, pad[1])
        self.x = view(rng.standard_normal((rows, k)) * (1 + 6 * (rng.random((1, k)) < 0.02)), self.xt, pad[2])
        self.y = view(rng.standard_normal((rows, n)), self.yt, pad[3])
        self.ranks = ranks
        self.scales = rng.uniform(0.25, 2, n_adapters).astype(np.float32) if scaled else None
        if ranks is not None:  # what lies behind an adapter's rank is not read
            for i, r in enumerate(ranks):
                self.a[i, r:] = float("nan")
                self.b[i, :, r:] = float("nan")
        self.bank = pkg.LoraBank(self.a, self.b, ranks=ranks, scales=self.scales)
        self.plan = pkg.LoraPlan(self.ids.astype(np.int32), n_adapters)

    def exact(self):
        """The result and the bound of its error, in float64."""
        a, b, x, y = (t.double().cpu().numpy() for t in (self.a, self.b, self.x, self.y))
        want, bound = y.copy(), np.zeros_like(y)
        for i in np.unique(self.ids):
            if i < 0:
                continue
            at = np.flatnonzero(self.ids == i)
            r = a.shape[1] if self.ranks is None else self.ranks[i]
            s = 1.0 if self.scales is None else float(self.scales[i])
            A, B = a[i, :r], b[i, :, :r]
            t = s * (x[at] @ A.T)
            want[at] += t @ B.T
            if not r:
                continue
            dt = s * (np.abs(x[at]) @ np.abs(A).T) * (2.0 ** -23 * (a.shape[2] / 8 + 32) + 2.0 ** -23) + np.abs(t) * 2.0 ** -22
            split = 2.0 ** -22 if self.dtype == "f16" else 2.0 ** -16 if self.yt == "bf16" else 2.0 ** -23
            dt += split * (np.abs(t).max(1, keepdims=True) if self.dtype == "f16" else np.abs(t))
            bound[at] = dt @ np.abs(B).T + 2.0 ** -23 * (r / 8 + 16) * (np.abs(t) @ np.abs(B).T)
        return want, bound

    def check(self, out=None):
        import torch
        want, bound = self.exact()
        keep = self.y.clone()
        got = self.bank.apply(self.plan, self.x, self.y, out=out)
        assert got is (self.y if out is None else out)
        if out is not None:
            assert torch.equal(self.y, keep)
        g = got[:len(self.ids)].double().cpu().numpy()
        half = EPS[self.yt] * (np.abs(want) + bound) + (2.0 ** -25 if self.yt == "f16" else 0)
        assert (np.abs(g - want) <= bound + half).all()
        none = self.ids < 0
        assert torch.equal(got[:len(self.ids)][torch.from_numpy(none).cuda()], keep[torch.from_numpy(none).cuda()])
        assert np.linalg.norm(g - want) <= np.linalg.norm(bound) / 16 + np.linalg.norm(half)
        return g


TYPES = [("bf16", "same", "same"), ("bf16", "f32", "f32"), ("bf16", "same", "f32"), ("bf16", "f32", "same"),
         ("f16", "same", "same"), ("f16", "f32", "f32"), ("f16", "same", "f32"), ("f16", "f32", "same")]


def mixed(rows, adapters, seed=0, none=0.1):
    rng = np.random.default_rng(seed)
    ids = rng.integers(0, adapters, rows)
    ids[rng.random(rows) < none] = -1
    return ids


@pytest.mark.parametrize("dtype,x,y", TYPES)
@pytest.mark.parametrize("rows,adapters,k,n,rank", [(1, 1, 64, 48, 8), (1, 2, 4096, 4096, 16), (64, 64, 896, 1152, 16),
                                                    (37, 5, 1000, 333, 24), (130, 3, 257, 1025, 64), (300, 2, 512, 2048, 32),
                                                    (9, 1, 33, 17, 5), (70, 4, 128, 128, 128), (20, 2, 640, 96, 120)])
def test_sizes_and_types(pkg, rows, adapters, k, n, rank, dtype, x, y):
    import torch
    ids = mixed(rows, adapters, seed=rows) if rows > 1 else [adapters - 1]
    c = Case(pkg, ids, adapters, k, n, rank, dtype, x, y, seed=k)
    c.check(out=torch.empty_like(c.y))
    c.check()


@pytest.mark.parametrize("rank", [1, 2, 3, 7, 8, 9, 15, 16, 17, 31, 33, 48, 63, 65, 100, 121, 128])
def test_ranks(pkg, rank):
    Case(pkg, mixed(40, 3, seed=rank), 3, 320, 272, rank, seed=rank).check()


@pytest.mark.parametrize("dtype,x,y", TYPES)
def test_adapters_of_their_own_ranks(pkg, dtype, x, y):
    """Every rank from 0 to the bank's; NaN behind each adapter's own."""
    ranks = [0, 1, 5, 8, 13, 16, 24, 31, 32, 0, 3]
    c = Case(pkg, mixed(120, len(ranks), seed=2), len(ranks), 500, 700, 32, dtype, x, y, ranks=ranks)
    import torch
    c.check(out=torch.full_like(c.y, float("nan")))


@pytest.mark.parametrize("pad", [(1, 0, 0, 0), (0, 1, 0, 0), (0, 0, 1, 0), (0, 0, 0, 1), (8, 8, 8, 8), (4, 4, 4, 4), (3, 5, 7, 9)])
@pytest.mark.parametrize("dtype,x,y", [("bf16", "same", "same"), ("f16", "f32", "f32")])
def test_strides(pkg, pad, dtype, x, y):
    import torch
    for rows in (11, 150):
        c = Case(pkg, mixed(rows, 3, seed=4), 3, 264, 200, 24, dtype, x, y, pad=pad, seed=5)
        wide = torch.full((rows + 2, 200 + 6), -7.0, dtype=c.y.dtype, device="cuda")
        c.check(out=wide[:rows, 2:202])
        assert (wide[:, :2] == -7).all() and (wide[:, 202:] == -7).all() and (wide[rows:] == -7).all()


def test_expanded_inputs(pkg):
    """Rows and adapters that share memory, where they are only read."""
    import torch
    c = Case(pkg, mixed(30, 4, seed=1), 4, 256, 128, 16)
    c.x = c.x[:1].expand(30, 256)
    c.a = c.a[:1].expand(4, 16, 256)
    c.y = c.y[:1].expand(30, 128)
    c.bank = pkg.LoraBank(c.a, c.b, scales=c.scales)
    c.check(out=torch.empty(30, 128, dtype=torch.bfloat16, device="cuda"))
    with pytest.raises(pkg.SamplingError):
        c.bank.apply(c.plan, c.x, c.y)  # rows of the result on one another


@pytest.mark.parametrize("counts", [[1], [8], [9], [16], [17], [64], [65], [127], [128], [129], [500, 1, 40], [2000, 3]])
def test_rows_of_one_adapter(pkg, counts):
    ids = np.concatenate([np.full(c, i) for i, c in enumerate(counts)])
    np.random.default_rng(0).shuffle(ids)
    for dtype, x, y in TYPES[:2]:
        Case(pkg, ids, len(counts), 288, 352, 16, dtype, x, y, seed=len(ids)).check()


@pytest.mark.parametrize("dtype,x,y", TYPES)
@pytest.mark.parametrize("counts,k,n,rank", [([1100], 256, 320, 16), ([700, 65, 500, 9, 3], 1000, 333, 24), ([1500, 40], 129, 1025, 64),
                                             ([1024], 4096, 128, 128), ([900, 201], 64, 64, 1), ([1300], 640, 200, 90)])
def test_very_many_rows(pkg, counts, k, n, rank, dtype, x, y):
    import torch
    ids = np.concatenate([np.full(c, i) for i, c in enumerate(counts)] + [np.full(7, -1)])
    np.random.default_rng(1).shuffle(ids)
    c = Case(pkg, ids, len(counts), k, n, rank, dtype, x, y, seed=k)
    c.check(out=torch.full_like(c.y, float("nan")))
    c.check()
    c.plan.status()


@pytest.mark.parametrize("pad", [(1, 0, 0, 0), (0, 3, 0, 0), (0, 0, 5, 0), (0, 0, 0, 7), (8, 8, 8, 8)])
def test_very_many_rows_of_other_strides_and_ranks(pkg, pad):
    ids = np.random.default_rng(2).integers(0, 4, 1600)
    for dtype, y in (("bf16", "same"), ("f16", "f32")):
        Case(pkg, ids, 4, 264, 200, 32, dtype, "same", y, ranks=[0, 5, 16, 31], pad=pad, seed=5).check()


def test_long_sums(pkg):
    for rows in (3, 100):
        Case(pkg, [0] * rows, 1, 18944, 3584, 16, "bf16", seed=1).check()
        Case(pkg, [0] * rows, 1, 18944, 256, 64, "f16", "f32", "f32", seed=2).check()


def test_many_rows_of_many_adapters(pkg):
    Case(pkg, mixed(3000, 70, seed=3, none=0.3), 70, 128, 160, 8, seed=3).check()


def test_rows_behind_the_plan_are_left(pkg):
    import torch
    c = Case(pkg, mixed(20, 2, seed=6), 2, 96, 80, 8)
    x = torch.cat([c.x, torch.full((5, 96), float("nan"), device="cuda", dtype=c.x.dtype)])
    y = torch.cat([c.y, torch.full((5, 80), 3.0, device="cuda", dtype=c.y.dtype)])
    c.x, c.y = x, y
    c.bank.apply(c.plan, x, y)
    assert (y[20:] == 3).all()


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("scale", [1e-6, 1e-3, 1e4])
def test_small_and_large_values(pkg, dtype, scale):
    """f32 rows of any size: t is split relative to its row's largest value."""
    for rows in (4, 90):
        c = Case(pkg, [0] * rows, 1, 512, 256, 16, dtype, "f32", "f32", seed=7)
        c.x.mul_(scale)
        c.y.mul_(scale)
        c.check()


@pytest.mark.parametrize("rows", [5, 80])
@pytest.mark.parametrize("dtype,x,y", [("bf16", "same", "same"), ("f16", "same", "same"), ("bf16", "f32", "f32")])
def test_a_bad_row_stays_alone(pkg, rows, dtype, x, y):
    """NaN and infinities of one row reach that row only."""
    import torch
    c = Case(pkg, [0] * rows, 1, 256, 192, 16, dtype, x, y, seed=8)
    good = torch.empty_like(c.y)
    c.bank.apply(c.plan, c.x, c.y, out=good)
    c.x[2, 17] = float("nan")
    c.x[3, 5] = float("inf")
    got = torch.empty_like(c.y)
    c.bank.apply(c.plan, c.x, c.y, out=got)
    rest = [i for i in range(rows) if i not in (2, 3)]
    assert torch.equal(got[rest], good[rest])
    assert got[2].isnan().all() and not got[3].isfinite().any()


def test_far_strides(pkg):
    """Offsets past 32 bits in the bank and the rows."""
    import torch
    c = Case(pkg, [2, 0, 1, 2], 3, 64, 40, 8)
    far = torch.empty(3, (1 << 31) + 8, dtype=torch.bfloat16, device="cuda")
    a = far[:, :8 * 64].view(3, 8, 64)
    a.copy_(c.a)
    c.a, c.bank = a, pkg.LoraBank(a, c.b, scales=c.scales)
    c.check(out=torch.empty_like(c.y))
    far_x = torch.empty(4, 1 << 30, dtype=torch.bfloat16, device="cuda")
    far_x[:, :64] = c.x
    c.x = far_x[:, :64]
    c.check()
    del far, far_x, a
    c.a = c.x = c.bank = None
    torch.cuda.empty_cache()


def test_two_calls_give_the_same_bits(pkg):
    """Units of two sizes in one call, twice."""
    import torch
    c = Case(pkg, [0] * 5 + [1] * 40, 2, 512, 384, 16, seed=9)
    both = torch.empty_like(c.y)
    c.bank.apply(c.plan, c.x, c.y, out=both)
    again = torch.empty_like(c.y)
    c.bank.apply(c.plan, c.x, c.y, out=again)
    assert torch.equal(both, again)


def test_capture_and_other_streams(pkg):
    import torch
    c = Case(pkg, mixed(50, 4, seed=2), 4, 300, 400, 16, seed=10)
    out = torch.empty_like(c.y)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        c.bank.apply(c.plan, c.x, c.y, out=out)
    side.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        c.bank.apply(c.plan, c.x, c.y, out=out)
    for seed in range(2):
        c.x.copy_(torch.randn_like(c.x))
        c.y.copy_(torch.randn_like(c.y))
        eager = c.bank.apply(c.plan, c.x, c.y, out=torch.empty_like(c.y))
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(eager, out)


def test_refusals(pkg):
    import torch
    c = Case(pkg, [0, 1, -1], 2, 64, 32, 8)
    a, b, x, y, plan = c.a, c.b, c.x, c.y, c.plan
    bad = [lambda: pkg.LoraBank(a, b.half()), lambda: pkg.LoraBank(a.float(), b.float()), lambda: pkg.LoraBank(a[:1], b),
           lambda: pkg.LoraBank(a, b[..., :4]), lambda: pkg.LoraBank(a[0], b), lambda: pkg.LoraBank(a.transpose(1, 2), b),
           lambda: pkg.LoraBank(a, b, ranks=[1]), lambda: pkg.LoraBank(a, b, ranks=[1, 9]), lambda: pkg.LoraBank(a, b, ranks=[-1, 2]),
           lambda: pkg.LoraBank(a, b, ranks=[1.5, 2]), lambda: pkg.LoraBank(a, b, scales=[1.0]),
           lambda: pkg.LoraBank(a, b, scales=torch.ones(2)), lambda: pkg.LoraPlan([2], 2), lambda: pkg.LoraPlan([-2], 2),
           lambda: c.bank.apply(plan, x[:2], y), lambda: c.bank.apply(plan, x, y[:, :31]), lambda: c.bank.apply(plan, x.half(), y),
           lambda: c.bank.apply(plan, x, y, out=y.float()), lambda: c.bank.apply(plan, x.T, y),
           lambda: c.bank.apply(plan, x.cpu(), y), lambda: c.bank.apply(pkg.LoraPlan([0], 3), x, y),
           lambda: c.bank.apply(plan, x, y, out=torch.empty(3, 64, device="cuda", dtype=y.dtype)[:, ::2])]
    for call in bad:
        with pytest.raises(pkg.SpecError):
            call()
    with pytest.raises(pkg.UnsupportedMethodError):
        pkg.LoraBank(torch.zeros(1, 129, 8, device="cuda").half(), torch.zeros(1, 8, 129, device="cuda").half()).apply(
            pkg.LoraPlan([0], 1), torch.zeros(1, 8, device="cuda"), torch.zeros(1, 8, device="cuda"))
    keep = y.clone()
    c.bank.apply(pkg.LoraPlan([], 2), x[:0], y[:0])
    c.bank.apply(pkg.LoraPlan([-1] * 3, 2), x, y)
    assert torch.equal(y, keep)


# Runs of rows that units of 8 and larger ones can take: by the bank's and the rows' bytes.
@pytest.mark.parametrize("dtype,x,y", [("bf16", "same", "same"), ("bf16", "f32", "f32"), ("f16", "same", "f32")])
@pytest.mark.parametrize("k,n,rank", [(2048, 96, 64), (64, 1000, 16), (520, 264, 128)])
@pytest.mark.parametrize("runs,none", [((24, 40, 9, 64), 5), ((17, 300), 0), ((33,) * 40, 3), ((889,), 1), ((700, 100), 0)])
def test_runs_that_two_kernels_take(pkg, runs, none, k, n, rank, dtype, x, y):
    import torch
    ids = np.repeat(np.arange(len(runs) + 1) - 1, (none,) + runs)
    ids = np.random.default_rng(5).permutation(ids)
    c = Case(pkg, ids, len(runs), k, n, rank, dtype, x=x, y=y, seed=7, pad=(8, 8, 8, 8))
    out = torch.empty_like(c.y)
    g = c.check(out)
    assert (c.check() == g).all()  # in place, the rows without an adapter as they are


def test_one_plan_on_two_streams_at_once(pkg):
    """A plan and a bank used on two streams at a time, and dropped while their calls may still run."""
    import torch
    ids = mixed(200, 6, seed=11)
    c = Case(pkg, ids, 6, 1024, 2048, 16, seed=12)
    xs = [torch.randn_like(c.x) for _ in range(8)]
    want = [c.bank.apply(c.plan, x, c.y, out=torch.empty_like(c.y)) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    outs = [torch.empty_like(c.y) for _ in xs]
    plan, bank = c.plan, c.bank
    del c.plan, c.bank
    for i, (x, out) in enumerate(zip(xs, outs)):
        with torch.cuda.stream(streams[i % 2]):
            bank.apply(plan, x, c.y, out=out)
    del plan, bank
    junk = [torch.full((1 << 16,), 255, dtype=torch.uint8, device="cuda") for _ in range(8)]
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, want)) and junk


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("rows,adapters,rank,x", [(8100, 3, 64, "same"), (2400, 40, 128, "f32"), (2400, 40, 128, "same"),
                                                  (3000, 60, 16, "f32"), (300, 300, 128, "f32"), (300, 300, 128, "same"),
                                                  (5, 5, 16, "f32")])
def test_long_sums_are_no_less_than_f32(pkg, rows, adapters, rank, dtype, x):
    """x A^T of 14336 positive terms: a sum that drops its last bits at every step ends too small.

    B = 1 hands x A^T out in f32.  The tensor core adds up at most 16 instructions in a row, each of which may drop
    2^-23 of the running sum on either side of it: (16 + 1) 2^-23 of positive terms.  Those sums meet in rounded
    additions, at most 448 of them, random to first order: sqrt(448) 2^-24 in the norm.  Splits of x and of
    x A^T: 2^-23 and 2^-22.  Together below 3.7e-6; 448 to 3584 instructions in a row end 1e-5 to 1e-4 too small."""
    import torch
    k, kind = 14336, kinds()[dtype]
    gen = torch.Generator(device="cuda").manual_seed(rank)
    xs = 0.5 + 0.5 * torch.rand(rows, k, device="cuda", generator=gen)
    xs = xs if x == "f32" else xs.to(kind)
    a = ((0.5 + 0.5 * torch.rand(rank, k, device="cuda", generator=gen)) / 128).to(kind)
    b = torch.eye(rank, device="cuda").to(kind)
    bank = pkg.LoraBank(a.expand(adapters, rank, k), b.expand(adapters, rank, rank))
    got = bank.apply(pkg.LoraPlan(np.arange(rows) % adapters, adapters), xs, torch.zeros(rows, rank, device="cuda"))
    want = xs.double() @ a.double().T
    assert float((got.double() - want).norm() / want.norm()) <= 17 * 2.0 ** -23 + 448 ** 0.5 * 2.0 ** -24 + 2.0 ** -23 + 2.0 ** -22



@pytest.mark.parametrize("dtype,x,y", TYPES)
@pytest.mark.parametrize("rows", [3, 40, 1000])
@pytest.mark.parametrize("rank", [2, 24, 72])
def test_all_bits_of_the_first_product_count(pkg, rows, rank, dtype, x, y):
    """x A^T holds 21-bit whole numbers t and -t + d: their sum d + y is small, so that it is exact in every type.

    Every number that enters has at most 7 bits, every sum at most 21: f32 sums are exact, and t is, in parts of
    21 bits in all or more."""
    import torch
    rng = np.random.default_rng(rows + rank)
    k, n = 200, 96
    digits = rng.integers(0, 128, (rows, 3))
    at, pair = rng.permutation(k)[:3], rng.permutation(rank)[:2]
    xs, a = np.zeros((rows, k)), np.zeros((1, rank, k))
    xs[:, at] = digits
    a[0, pair[0], at] = [1 << 14, 1 << 7, 1]
    a[0, pair[1], at] = [-(1 << 14), -(1 << 7), 0]
    ys = rng.integers(-64, 65, (rows, n))
    bank = pkg.LoraBank(dev(a, dtype), dev(np.ones((1, n, rank)), dtype))
    got = bank.apply(pkg.LoraPlan([0] * rows, 1), dev(xs, dtype if x == "same" else x), dev(ys, dtype if y == "same" else y))
    assert np.array_equal(got.double().cpu().numpy(), (digits[:, 2:] + ys).astype(np.float64))


def test_weights_of_another_stream_outlive_the_bank(pkg):
    """Weights of one stream, bank and call on another, all dropped while the call waits: their memory is not handed out."""
    import torch
    main, side = torch.cuda.current_stream(), torch.cuda.Stream()
    shapes = ((3, 16, 1 << 17), (3, 1 << 17, 16))  # blocks of their own
    kept = [torch.zeros(s, dtype=torch.bfloat16, device="cuda") for s in shapes]
    ranks, scales = torch.full((3,), 16, dtype=torch.int32, device="cuda"), torch.ones(3, device="cuda")
    x, y = (torch.zeros(3, 1 << 17, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    at = [t.data_ptr() for t in kept]
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        bank = pkg.LoraBank(*kept, ranks=ranks, scales=scales)
        plan = pkg.LoraPlan([0, 2, -1], 3)
        torch.cuda._sleep(200_000_000)  # about 0.1 s
        bank.apply(plan, x, y)
    del kept, bank, plan
    assert torch.cuda.current_stream() == main
    again = [torch.empty(s, dtype=torch.bfloat16, device="cuda") for s in shapes * 2]
    assert not side.query()  # the call has still to run
    assert not {t.data_ptr() for t in again} & set(at)
    side.synchronize()


CALLERS = r"""
#include <atomic>
#include <thread>
#include "spec_b200.h"
using Apply = int (*)(const spec_lora_bank*, const spec_lora_plan*, const spec_lora_rows*, const spec_lora_rows*, const spec_lora_rows*, void*);
struct Call { void *bank, *plan, *rows, *stream; };
extern "C" int run_callers(Apply apply, const Call* calls, int n, int turns) {
  std::atomic<int> failed{0}, ready{0};
  auto loop = [&](const Call& c) {
    const spec_lora_rows* r = static_cast<const spec_lora_rows*>(c.rows);
    for (++ready; ready < n;) {}
    for (int i = 0; i < turns; ++i)
      if (apply(static_cast<spec_lora_bank*>(c.bank), static_cast<spec_lora_plan*>(c.plan), r, r + 1, r + 2, c.stream)) ++failed;
  };
  std::thread other(loop, calls[1]);
  loop(calls[0]);
  other.join();
  return failed;
}
"""


def test_calls_of_two_host_threads(pkg, tmp_path):
    """Few units, which take an SM's whole shared memory, beside many, which share it, from two native threads at once
    (python's wait for each other's lock)."""
    import ctypes
    import os
    import shutil
    import subprocess
    import torch
    if not shutil.which("g++"):
        pytest.skip("no C++ compiler")
    src, lib = tmp_path / "callers.cpp", tmp_path / "libcallers.so"
    src.write_text(CALLERS)
    include = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include")
    subprocess.run(["g++", "-std=c++17", "-O2", "-shared", "-fPIC", "-pthread", f"-I{include}", str(src), "-o", str(lib)], check=True)
    cases = [Case(pkg, np.repeat(np.arange(n), 40), n, 128, 128, 64, seed=n) for n in (2, 40)]
    outs, streams = [torch.zeros_like(c.y) for c in cases], [torch.cuda.Stream() for _ in cases]
    want = [c.bank.apply(c.plan, c.x, c.y, out=torch.empty_like(c.y)) for c in cases]
    torch.cuda.synchronize()
    from importlib import import_module
    rows = [import_module("abyo-speculate_b200.lora")._THREE_ROWS.pack(
        *c.bank._rows(c.x, c.bank.k, "x"), *c.bank._rows(c.y, c.bank.n, "y"), *c.bank._rows(o, c.bank.n, "out")) for c, o in zip(cases, outs)]
    calls = (ctypes.c_void_p * 8)(*[at for c, r, s in zip(cases, rows, streams) for at in (
        c.bank._at, c.plan._at, ctypes.cast(ctypes.c_char_p(r), ctypes.c_void_p).value, s.cuda_stream)])
    apply = ctypes.cast(pkg.load().spec_lora_apply, ctypes.c_void_p)
    assert ctypes.CDLL(str(lib)).run_callers(apply, calls, 2, 5000) == 0
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, want))


@pytest.mark.parametrize("dtype,x,y", [t for t in TYPES if t[1] == "same"])
@pytest.mark.parametrize("counts,k,n,rank", [([1290, 9], 264, 200, 128), ([2500, 70, 40], 520, 333, 72), ([1900, 900], 4096, 64, 16),
                                             ([4900], 136, 1025, 100), ([9600, 65], 72, 130, 24)])
def test_units_of_128_rows_in_clusters_of_every_size(pkg, counts, k, n, rank, dtype, x, y):
    """11, 21, 23, 39 and 76 units of 128 rows: clusters of 8, 4, 4, 2 blocks and single ones."""
    import torch
    ids = np.random.default_rng(3).permutation(np.repeat(np.arange(len(counts)), counts))
    c = Case(pkg, ids, len(counts), k, n, rank, dtype, x, y, seed=rank)
    c.check(out=torch.full_like(c.y, float("nan")))
    c.check()
    c.plan.status()


@pytest.mark.parametrize("dtype,y", [("bf16", "same"), ("f16", "f32")])
def test_very_many_rows_with_bad_rows_and_other_ranks(pkg, dtype, y):
    """NaN and infinities reach their rows alone, and what lies behind an adapter's rank none."""
    import torch
    c = Case(pkg, np.arange(2700) % 3, 3, 264, 200, 80, dtype, "same", y, ranks=[80, 17, 0], seed=4)
    good = c.bank.apply(c.plan, c.x, c.y, out=torch.empty_like(c.y))
    c.x[300, 7], c.x[1501, 200] = float("nan"), float("inf")
    got = c.bank.apply(c.plan, c.x, c.y, out=torch.empty_like(c.y))
    same = torch.ones(2700, dtype=torch.bool, device="cuda")
    same[300] = same[1501] = False
    assert torch.equal(got[same], good[same]) and got[300].isnan().all()
    c.x[300] = c.x[1501] = 0
    c.check()


@pytest.mark.parametrize("rows", [1, 3, 200])
def test_a_wait_that_gave_up_is_reported_once(pkg, rows):
    """The plan's word of the device's waits, set as a wait that gives up sets it; calls leave it as it is."""
    import torch
    c = Case(pkg, [0] * rows, 1, 64, 48, 8)
    c.check()
    c.plan.status()
    word = c.plan._copy[rows * 52:rows * 52 + 4]
    assert c.plan._copy.numel() == rows * 52 + 16 and not word.any()
    word[0] = 1
    c.check()
    with pytest.raises(pkg.DeviceError, match="gave up") as e:
        c.plan.status()
    assert e.value.code == 7
    c.plan.status()
    assert not word.any()
    c.check()


@pytest.mark.parametrize("rows", [1, 6, 300])
def test_rows_beside_each_other(pkg, rows):
    """x, y and the result as columns of one tensor, rows in turn, a row before or behind the others: none shares memory."""
    import torch
    c = Case(pkg, mixed(rows, 3, seed=rows, none=0) if rows > 1 else [0], 3, 64, 64, 16, seed=1)
    want = c.bank.apply(c.plan, c.x, c.y, out=torch.empty_like(c.y))
    one = torch.cat([c.x, c.y, torch.zeros_like(c.y)], 1)
    got = c.bank.apply(c.plan, one[:, :64], one[:, 64:128], out=one[:, 128:])
    assert torch.equal(got, want) and torch.equal(one[:, :64], c.x) and torch.equal(one[:, 64:128], c.y)
    turns = torch.stack([c.x, c.y, torch.zeros_like(c.y)], 1).reshape(3 * rows, 64)
    assert torch.equal(c.bank.apply(c.plan, turns[0::3], turns[1::3], out=turns[2::3]), want)
    behind = torch.cat([c.x, c.y, torch.zeros_like(c.y)])
    assert torch.equal(c.bank.apply(c.plan, behind[:rows], behind[rows:2 * rows], out=behind[2 * rows:]), want)
    for bad in (lambda: c.bank.apply(c.plan, c.x, c.x), lambda: c.bank.apply(c.plan, c.x, c.y, out=c.x),
                lambda: c.bank.apply(c.plan, one[:, :64], one[:, 64:128], out=one[:, 65:129])):
        with pytest.raises(pkg.SamplingError):
            bad()


@pytest.mark.parametrize("x", ["same", "f32"])
def test_the_most_rows(pkg, x):
    """2^20 rows: of one adapter, and most without one."""
    n = 1 << 20
    Case(pkg, np.zeros(n, np.int32), 1, 24, 16, 5, "bf16", x, x, seed=1).check()
    ids = np.full(n, -1)
    ids[::4001], ids[-1] = 1, 0
    Case(pkg, ids, 2, 24, 16, 5, "bf16", x, x, seed=2).check()
    with pytest.raises(pkg.SamplingError):
        pkg.LoraPlan(np.zeros(n + 1, np.int32), 1)


def test_very_many_adapters(pkg):
    Case(pkg, np.random.default_rng(0).permutation(20000), 20000, 40, 32, 8, seed=3).check()
