"""4-bit paged KV cache on the GPU: stored bytes against the f32 restatement
(equal), attention against float64 within the bound kv4_ref.attend derives
plus the rounding of the output's type."""

import numpy as np
import pytest

import kv4_ref as ref

pytestmark = pytest.mark.gpu

ROUND = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11, "f32": 0.0}


def dtype_of(name):
    import torch
    return {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}[name]


class Setup:
    """A pool of NaN bytes, page tables of shuffled pages, rotation tables, and
    the same pool on the host."""

    def __init__(self, pkg, heads, kv_heads, d, page, lens, half=True, layers=1, layer=0, seed=0, rope=True):
        import torch
        self.rng = np.random.default_rng(seed)
        self.heads, self.kv, self.d, self.p, self.layer, self.half = heads, kv_heads, d, page, layer, half
        need = [-(-n // page) for n in lens]
        self.n_pages = sum(need) + 2
        order = self.rng.permutation(self.n_pages)
        self.table, at = [], 0
        for n in need:
            self.table.append([int(x) for x in order[at:at + n]])
            at += n
        size = pkg.KV4Cache.pool_bytes(n_layers=layers, n_kv_heads=kv_heads, head_dim=d, page_tokens=page,
                                       n_pages=self.n_pages)
        assert size == layers * self.n_pages * kv_heads * ref.block_bytes(page, d)
        self.pool = torch.full((size,), 255, dtype=torch.uint8, device="cuda")
        self.host = np.full((layers, self.n_pages, kv_heads, ref.block_bytes(page, d)), 255, np.uint8)
        tables = pkg.rope_tables(d, max(lens) + 80, 1e4) if rope else None
        self.cos, self.sin = [t.cpu().numpy() for t in tables] if rope else (None, None)
        self.cache = pkg.KV4Cache(self.pool, n_layers=layers, n_heads=heads, n_kv_heads=kv_heads, head_dim=d,
                                  page_tokens=page, n_pages=self.n_pages, rope=tables, rope_half=half)
        self.batch = pkg.KV4Batch(self.cache)

    def rows(self, n, heads, dtype, spread=1.0, pad=0):
        """Tensor [n, heads, d] (a view with `pad` extra channels between heads) and its f32 values."""
        import torch
        x = self.rng.standard_normal((n, heads, self.d + pad)).astype(np.float32) * np.float32(spread)
        x += (self.rng.random((1, heads, self.d + pad)) < 0.05) * np.float32(4 * spread)
        t = torch.from_numpy(x).cuda().to(dtype_of(dtype))[:, :, :self.d]
        return t, t.float().cpu().numpy()

    def store(self, b, slot, k, v):
        """The restatement's append of rotated k [kv heads, d] and v at a slot of sequence b; returns the values."""
        out = np.empty((2, self.kv, self.d), np.float32)
        page, j = self.table[b][slot // self.p], slot % self.p
        for which, x in ((0, k), (1, v)):
            for h in range(self.kv):
                codes, so, val = ref.quantize(x[h])
                ref.store(self.host[self.layer, page, h], self.p, self.d, j, codes, so, which == 1)
                out[which, h] = val
        return out

    def turned(self, x, pos):
        return x if self.cos is None else ref.rotate(x, self.cos[pos], self.sin[pos], self.half)

    def fill(self, lens):
        """Appends lens[b] random rows to every sequence, through the library in one step, and to the host pool."""
        import torch
        total = sum(lens)
        if total == 0:
            return
        k, kn = self.rows(total, self.kv, "f16", 1.5)
        v, vn = self.rows(total, self.kv, "f16")
        self.batch.plan([0] * len(lens), lens, self.table)
        self.batch.append(self.layer, None, k, v)
        r = 0
        for b, n in enumerate(lens):
            for i in range(n):
                self.store(b, i, self.turned(kn[r], i), vn[r])
                r += 1
        torch.cuda.synchronize()

    def device_pool(self):
        return self.pool.cpu().numpy().reshape(self.host.shape)

    def values(self, b, n):
        """Stored K and V of sequence b's first n tokens [n, kv heads, d] in float64."""
        out = np.empty((2, n, self.kv, self.d))
        for t in range(n):
            page = self.table[b][t // self.p]
            for h in range(self.kv):
                for which in (0, 1):
                    out[which, t, h] = ref.load(self.host[self.layer, page, h], self.p, self.d, t % self.p, which == 1)
        return out


def check_attend(s, kv, rows, q, out, masks, out_type, scale=None):
    scale = s.d ** -0.5 if scale is None else scale
    got = out.float().cpu().numpy().astype(np.float64)
    qn = q.float().cpu().numpy().astype(np.float64)
    r = 0
    for b, (n, m) in enumerate(zip(kv, rows)):
        k, v = s.values(b, n + m)
        want, bound = ref.attend(qn[r:r + m], k, v, n, None if masks is None else masks[r:r + m], scale)
        bound = bound + ROUND[out_type] * np.abs(want)
        bad = ~(np.abs(got[r:r + m] - want) <= bound) & ~(np.isnan(want) & np.isnan(got[r:r + m]))
        assert not bad.any(), (b, n, m, np.argwhere(bad)[:4], got[r:r + m][bad][:4], want[bad][:4], bound[bad][:4])
        r += m


@pytest.mark.parametrize("d,page,heads,kv_heads", [(128, 64, 4, 2), (64, 16, 6, 2), (128, 16, 7, 1), (64, 128, 3, 3),
                                                   (128, 32, 8, 8)])
@pytest.mark.parametrize("dtype,half,pad", [("bf16", True, 0), ("f16", False, 0), ("f32", True, 3), ("f32", False, 8),
                                            ("bf16", False, 1)])
def test_append_stores_the_restated_bytes(pkg, d, page, heads, kv_heads, dtype, half, pad):
    import torch
    lens, rows = [0, 5, page - 1, 0], [1, 3, page + 2, 0]
    s = Setup(pkg, heads, kv_heads, d, page, [a + b for a, b in zip(lens, rows)], half, layers=2, layer=1, seed=d + page)
    total = sum(rows)
    q, qn = s.rows(total, heads, dtype, pad=pad)
    k, kn = s.rows(total, kv_heads, dtype, 2.0, pad)
    v, vn = s.rows(total, kv_heads, dtype, 1.0, pad)
    pos = [int(x) for x in s.rng.integers(0, max(lens) + 80, total)]
    q_out = torch.empty(total, heads, d, dtype=dtype_of("f16" if dtype == "f16" else "bf16"), device="cuda")
    k_out = torch.empty(total, kv_heads, d, dtype=torch.float16, device="cuda")
    v_out = torch.empty_like(k_out)
    s.batch.plan(lens, rows, s.table, positions=pos)
    assert s.batch.append(1, q, k, v, q_out=q_out, k_out=k_out, v_out=v_out) is q_out
    torch.cuda.synchronize()
    r = 0
    for b, (n, m) in enumerate(zip(lens, rows)):
        for i in range(m):
            val = s.store(b, n + i, s.turned(kn[r], pos[r]), vn[r])
            assert np.array_equal(k_out[r].cpu().numpy(), val[0].astype(np.float16)), (b, i)
            assert np.array_equal(v_out[r].cpu().numpy(), val[1].astype(np.float16)), (b, i)
            want = torch.from_numpy(s.turned(qn[r], pos[r])).to(q_out.dtype)
            assert torch.equal(q_out[r].cpu(), want), (b, i)
            r += 1
    assert np.array_equal(s.device_pool(), s.host)  # rows elsewhere, other layers and pages untouched


def test_append_in_place_selected_rows_and_no_rotation(pkg):
    """q in place; rows taken by src_rows (an accepted path written at its final
    slots); a cache without rotation tables stores rows as they are."""
    import torch
    s = Setup(pkg, 4, 2, 128, 16, [40], seed=3)
    q, qn = s.rows(6, 4, "bf16")
    k, kn = s.rows(6, 2, "bf16", 2.0)
    v, vn = s.rows(6, 2, "bf16")
    s.batch.plan([20], [6], s.table, positions=[20, 21, 21, 22, 22, 23], masks=[1, 3, 5, 11, 21, 43])
    s.batch.append(0, q, k, v, q_out=q)
    for i, p in enumerate([20, 21, 21, 22, 22, 23]):
        want = torch.from_numpy(s.turned(qn[i], p)).to(q.dtype)
        assert torch.equal(q[i].cpu(), want)
        s.store(0, 20 + i, s.turned(kn[i], p), vn[i])
    assert np.array_equal(s.device_pool(), s.host)
    # The path 0 -> 2 -> 4 is accepted.
    s.batch.plan([20], [3], s.table, src_rows=[0, 2, 4])
    s.batch.append(0, None, k, v)
    for i, r in enumerate([0, 2, 4]):
        s.store(0, 20 + i, s.turned(kn[r], 20 + i), vn[r])
    assert np.array_equal(s.device_pool(), s.host)
    t = Setup(pkg, 2, 2, 64, 32, [9], rope=False, seed=4)
    k, kn = t.rows(9, 2, "f32", 2.0)
    v, vn = t.rows(9, 2, "f32")
    t.batch.plan([0], [9], t.table)
    t.batch.append(0, None, k, v)
    for i in range(9):
        t.store(0, i, kn[i], vn[i])
    assert np.array_equal(t.device_pool(), t.host)


def test_append_extreme_rows(pkg):
    """Constant groups, values past the clamp, infinities, tiny values, and a
    NaN (which makes the row of its head NaN and no other)."""
    import torch
    s = Setup(pkg, 2, 2, 128, 16, [8], rope=False, seed=5)
    k = torch.zeros(8, 2, 128)
    k[1] = 3.7
    k[2, 0, :32] = torch.linspace(-1e9, 1e9, 32)
    k[3, 1, 40] = float("inf")
    k[3, 0, 41] = -float("inf")
    k[4] = torch.linspace(-1e-7, 1e-7, 128)
    k[5, 0, 100] = float("nan")
    k[6] = torch.linspace(1000.0, 1000.5, 128)
    k[7] = torch.randn(2, 128) * 1e-30
    v = k.flip(0).contiguous()
    s.batch.plan([0], [8], s.table)
    s.batch.append(0, None, k.cuda(), v.cuda())
    for i in range(8):
        s.store(0, i, k[i].numpy(), v[i].numpy())
    got = s.device_pool()
    nan = np.frombuffer(got.tobytes(), np.float16)
    want = np.frombuffer(s.host.tobytes(), np.float16)
    same = (got == s.host)
    # NaN payloads may differ; everything else is equal.
    pair = same.reshape(-1, 2).all(1) | (np.isnan(nan) & np.isnan(want))
    assert pair.all()
    x = np.clip(k.numpy().astype(np.float64), -20000, 20000)
    val = s.values(0, 8)[0]
    for i in range(8):
        for h in range(2):
            if np.isnan(x[i, h]).any():
                assert np.isnan(val[i, h]).all()
                continue
            for g in range(4):
                xs, vs = x[i, h, 32 * g:32 * g + 32], val[i, h, 32 * g:32 * g + 32]
                span, low = xs.max() - xs.min(), np.abs(xs.min())
                s16 = span * 16 / 15
                # half a step, the rounding of s and o to f16 (a subnormal s or o: 2^-25), f32 noise
                bound = s16 / 32 + (low + 2 * s16) * 2.0 ** -11 + 2.0 ** -24 + np.abs(xs).max() * 2.0 ** -20
                assert (np.abs(xs - vs) <= bound).all(), (i, h, g)


def wide_from(monkeypatch, columns):
    """Sends sequences of more columns to the kernel for many (None: the plan's estimate decides)."""
    if columns is None:
        monkeypatch.delenv("SPEC_B200_KV4_WIDE_FROM", raising=False)
    else:
        monkeypatch.setenv("SPEC_B200_KV4_WIDE_FROM", str(columns))


CASES = [
    # heads, kv heads, d, page, kv lengths, rows
    (4, 2, 128, 64, [0, 1, 63, 64, 129], [1, 1, 1, 1, 1]),
    (8, 2, 128, 16, [300, 0, 17], [5, 5, 5]),
    (7, 1, 128, 32, [45, 130], [9, 2]),
    (14, 2, 64, 32, [200, 31, 0], [1, 4, 7]),
    (3, 3, 64, 128, [257, 5], [2, 33]),
    (2, 2, 128, 128, [128, 1], [1, 0]),
    (32, 1, 64, 16, [77], [3]),
    (5, 1, 128, 64, [190], [20]),
]


@pytest.mark.parametrize("case", range(len(CASES)))
@pytest.mark.parametrize("q_type,out_type,columns", [("bf16", "bf16", None), ("f16", "f16", None), ("bf16", "f32", None),
                                                     ("bf16", "bf16", 0)])
def test_attend_causal(pkg, monkeypatch, case, q_type, out_type, columns):
    import torch
    wide_from(monkeypatch, columns)
    heads, kv_heads, d, page, kv, rows = CASES[case]
    s = Setup(pkg, heads, kv_heads, d, page, [a + b for a, b in zip(kv, rows)], layers=2, layer=1, seed=10 + case)
    s.fill([a + b for a, b in zip(kv, rows)])
    q, _ = s.rows(sum(rows), heads, q_type, 1.5)
    s.batch.plan(kv, rows, s.table)
    out = torch.full((sum(rows), heads, d), float("nan"), dtype=dtype_of(out_type), device="cuda")
    assert s.batch.attend(1, q, out=out) is out
    s.batch.status()
    check_attend(s, kv, rows, q, out, None, out_type)
    again = s.batch.attend(1, q, out=torch.empty_like(out))
    assert torch.equal(again, out)


@pytest.mark.parametrize("rows", [65, 150, 300])
@pytest.mark.parametrize("d,heads,kv_heads", [(128, 4, 1), (64, 2, 2)])
def test_attend_prompt_chunk(pkg, rows, d, heads, kv_heads):
    """Row counts past one tile, over a prefix that ends inside a page; the
    sequence beside it decodes one token."""
    kv, m = [37, 70], [rows, 1]
    s = Setup(pkg, heads, kv_heads, d, 32, [a + b for a, b in zip(kv, m)], seed=rows)
    s.fill([a + b for a, b in zip(kv, m)])
    q, _ = s.rows(sum(m), heads, "bf16", 1.5)
    s.batch.plan(kv, m, s.table)
    out = s.batch.attend(0, q)
    s.batch.status()
    check_attend(s, kv, m, q, out, None, "bf16")


def random_masks(rng, n):
    anc = []
    for i in range(n):
        anc.append((1 << i) | (anc[int(rng.integers(max(0, i - 6), i))] if i else 0))
    return anc


@pytest.mark.parametrize("d,heads,kv_heads,page", [(128, 8, 2, 64), (64, 14, 2, 16), (128, 4, 4, 32)])
def test_attend_trees(pkg, d, heads, kv_heads, page):
    kv, rows = [100, 0, 63, 8], [31, 64, 1, 60]
    s = Setup(pkg, heads, kv_heads, d, page, [a + b for a, b in zip(kv, rows)], seed=d)
    s.fill([a + b for a, b in zip(kv, rows)])
    masks = [m for n in rows for m in random_masks(s.rng, n)]
    q, _ = s.rows(sum(rows), heads, "f16", 1.5)
    s.batch.plan(kv, rows, s.table, masks=masks)
    out = s.batch.attend(0, q)
    s.batch.status()
    check_attend(s, kv, rows, q, out, masks, "f16")


@pytest.mark.parametrize("heads,columns", [(4, None), (64, None), (4, 0), (64, 0)])
def test_attend_rows_that_see_nothing_give_zeros(pkg, monkeypatch, heads, columns):
    wide_from(monkeypatch, columns)
    kv, rows = [0, 12], [5, 3]
    s = Setup(pkg, heads, 2, 128, 16, [5, 15], seed=8)
    s.fill([5, 15])
    masks = [0, 1, 0, 8, 0b11111, 0, 0, 1]
    q, _ = s.rows(8, heads, "bf16")
    s.batch.plan(kv, rows, s.table, masks=masks)
    out = s.batch.attend(0, q)
    check_attend(s, kv, rows, q, out, masks, "bf16")
    assert (out[0] == 0).all() and (out[2] == 0).all() and not (out[5] == 0).all()


@pytest.mark.parametrize("heads,columns", [(4, None), (32, None), (4, 0), (32, 0)])
def test_attend_nan_stays_where_it_is_seen(pkg, monkeypatch, heads, columns):
    """A NaN key row, and a NaN value row, of a draft node reach the rows that
    see the node and no other; the unwritten bytes of a page read as NaN and
    reach none.  12 and 96 columns."""
    import torch
    wide_from(monkeypatch, columns)
    kv, rows = [9], [6]
    s = Setup(pkg, heads, 2, 128, 16, [15], rope=False, seed=9)
    s.fill([9])
    k, kn = s.rows(6, 2, "f32")
    v, vn = s.rows(6, 2, "f32")
    k[2, 0, 5] = float("nan")
    v[3, 1, 77] = float("nan")
    kn[2, 0, 5] = vn[3, 1, 77] = np.nan
    masks = [1, 3, 5, 9, 17, 33]
    s.batch.plan(kv, rows, s.table, masks=masks)
    s.batch.append(0, None, k, v)
    for i in range(6):
        s.store(0, 9 + i, kn[i], vn[i])
    q, _ = s.rows(6, heads, "bf16")
    out = s.batch.attend(0, q)
    check_attend(s, kv, rows, q, out, masks, "bf16")
    bad = torch.isnan(out).flatten(2).any(2).cpu().numpy()
    want = np.zeros((6, heads), bool)
    want[2, :heads // 2] = want[3, heads // 2:] = True
    assert (bad == want).all()


@pytest.mark.parametrize("heads,columns", [(4, None), (32, None), (4, 0), (32, 0)])
def test_attend_peaked_and_large_scores(pkg, monkeypatch, heads, columns):
    """Scores far apart (the running maximum moves late in the row), q beyond
    f16's range, a scale of zero and a negative one; 16 and 128 columns."""
    import torch
    wide_from(monkeypatch, columns)
    kv, rows = [700], [4]
    s = Setup(pkg, heads, 1, 128, 64, [704], rope=False, seed=12)
    k, kn = s.rows(704, 1, "f32")
    v, vn = s.rows(704, 1, "f32")
    grow = torch.linspace(0.1, 6.0, 704)[:, None, None]
    k, kn = k * grow.cuda(), kn * grow.numpy()
    s.batch.plan([0], [704], s.table)
    s.batch.append(0, None, k, v)
    k32 = k.cpu().numpy()
    for i in range(704):
        s.store(0, i, k32[i], vn[i])
    s.batch.plan(kv, rows, s.table)
    q, _ = s.rows(4, heads, "bf16", 3.0)
    for scale in (None, 0.0, -0.05):
        check_attend(s, kv, rows, q, s.batch.attend(0, q, scale=scale), None, "bf16", scale)
    big = q * 1e6
    out = s.batch.attend(0, big, scale=1e-7)
    check_attend(s, kv, rows, big, out, None, "bf16", 1e-7)


def test_attend_strides_and_streams(pkg):
    """q and out as views of wider tensors with odd strides; plan, append and
    attention on different streams, in the batch's order."""
    import torch
    kv, rows = [50, 3], [2, 2]
    s = Setup(pkg, 4, 2, 64, 16, [52, 5], seed=21)
    s.fill([50, 3])
    k, kn = s.rows(4, 2, "bf16", 2.0, pad=5)
    v, vn = s.rows(4, 2, "bf16", 1.0, pad=5)
    q, qn = s.rows(4, 4, "bf16", 1.0, pad=3)
    wide = torch.zeros(4, 4, 71, dtype=torch.bfloat16, device="cuda")
    turned = torch.empty(4, 4, 64, dtype=torch.bfloat16, device="cuda")
    torch.cuda.synchronize()
    a, b, c = (torch.cuda.Stream() for _ in range(3))
    with torch.cuda.stream(a):
        s.batch.plan(kv, rows, s.table)
    with torch.cuda.stream(b):
        s.batch.append(0, q, k, v, q_out=turned)
    with torch.cuda.stream(c):
        s.batch.attend(0, turned, out=wide[:, :, 3:67])
        s.batch.plan([1], [1], [s.table[0]])  # the old plan is read before it is overwritten
    s.batch.status()
    r = 0
    for i, (n, m) in enumerate(zip(kv, rows)):
        for j in range(m):
            s.store(i, n + j, s.turned(kn[r], n + j), vn[r])
            r += 1
    assert np.array_equal(s.device_pool(), s.host)
    check_attend(s, kv, rows, turned, wide[:, :, 3:67], None, "bf16")
    assert (wide[:, :, :3] == 0).all() and (wide[:, :, 67:] == 0).all()


# Sequences of many columns (rows x query heads of a KV head), on the kernel the
# plan estimates to be faster and on the one for many columns.
WIDE = [
    # heads, kv heads, d, page, kv lengths, rows, trees
    (8, 1, 128, 64, [0], [65], False),
    (8, 1, 64, 16, [131], [70], False),
    (14, 2, 64, 32, [50], [33], False),
    (32, 1, 128, 128, [1000], [9], False),
    (4, 1, 128, 16, [5], [300], False),
    (8, 2, 128, 32, [700, 3], [20, 64], False),
    (7, 1, 64, 128, [126, 0, 300], [19, 8, 40], False),
    (8, 1, 128, 64, [200], [60], True),
    (28, 4, 128, 16, [90], [31], True),
    (16, 2, 64, 32, [0, 63], [64, 50], True),
    (8, 1, 128, 64, [3000], [20], False),  # one tile split over many blocks and joined
    (8, 1, 64, 64, [2500], [33], True),
]


@pytest.mark.parametrize("case", range(len(WIDE)))
@pytest.mark.parametrize("q_type,out_type,pad,columns", [("bf16", "bf16", 0, 0), ("f16", "f32", 0, 0),
                                                         ("bf16", "f16", 3, 0), ("bf16", "bf16", 0, None)])
def test_attend_many_columns(pkg, monkeypatch, case, q_type, out_type, pad, columns):
    import torch
    wide_from(monkeypatch, columns)
    heads, kv_heads, d, page, kv, rows, trees = WIDE[case]
    s = Setup(pkg, heads, kv_heads, d, page, [a + b for a, b in zip(kv, rows)], seed=100 + case)
    s.fill([a + b for a, b in zip(kv, rows)])
    masks = [m for n in rows for m in random_masks(s.rng, n)] if trees else None
    q, _ = s.rows(sum(rows), heads, q_type, 1.5, pad=pad)
    s.batch.plan(kv, rows, s.table, masks=masks)
    out = torch.full((sum(rows), heads, d + pad), float("nan"), dtype=dtype_of(out_type), device="cuda")[:, :, :d]
    s.batch.attend(0, q, out=out)
    s.batch.status()
    check_attend(s, kv, rows, q, out, masks, out_type)
    again = torch.empty(sum(rows), heads, d, dtype=dtype_of(out_type), device="cuda")
    assert torch.equal(s.batch.attend(0, q, out=again), out)


@pytest.mark.parametrize("case", range(len(CASES)))
@pytest.mark.parametrize("most", [8, 16, 32])
def test_attend_causal_in_tiles_of_few_columns(pkg, monkeypatch, case, most):
    """The kernel for few columns in each of its tile sizes."""
    monkeypatch.setenv("SPEC_B200_KV4_NARROW_COLS", str(most))
    test_attend_causal(pkg, monkeypatch, case, "bf16", "f32", 1 << 20)


@pytest.mark.parametrize("most", [8, 16, 32])
def test_attend_odd_rows_in_tiles_of_few_columns(pkg, monkeypatch, most):
    """Rows that see nothing, NaN and large scores, and trees."""
    monkeypatch.setenv("SPEC_B200_KV4_NARROW_COLS", str(most))
    test_attend_rows_that_see_nothing_give_zeros(pkg, monkeypatch, 32, 1 << 20)
    test_attend_nan_stays_where_it_is_seen(pkg, monkeypatch, 32, 1 << 20)
    test_attend_peaked_and_large_scores(pkg, monkeypatch, 32, 1 << 20)
    test_attend_trees(pkg, 128, 8, 2, 64)


def one_tile(monkeypatch, on):
    """The kernel for many columns: one tile of 128 with its stages in pairs, or two tiles."""
    monkeypatch.setenv("SPEC_B200_KV4_WIDE_PAIR", str(int(on)))


@pytest.mark.parametrize("case", range(len(WIDE)))
@pytest.mark.parametrize("q_type,out_type,pad", [("bf16", "bf16", 0), ("f16", "f32", 3)])
def test_attend_many_columns_stages_in_pairs(pkg, monkeypatch, case, q_type, out_type, pad):
    one_tile(monkeypatch, True)
    test_attend_many_columns(pkg, monkeypatch, case, q_type, out_type, pad, 0)


@pytest.mark.parametrize("heads", [4, 32])
def test_attend_odd_rows_stages_in_pairs(pkg, monkeypatch, heads):
    """Rows that see nothing, NaN and large scores, through two accumulators."""
    one_tile(monkeypatch, True)
    test_attend_rows_that_see_nothing_give_zeros(pkg, monkeypatch, heads, 0)
    test_attend_nan_stays_where_it_is_seen(pkg, monkeypatch, heads, 0)
    test_attend_peaked_and_large_scores(pkg, monkeypatch, heads, 0)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("pair", [False, True])
def test_attend_many_columns_many_sequences(pkg, monkeypatch, d, pair):
    """More tiles than blocks: a block takes several, of 1 to 3 stages."""
    one_tile(monkeypatch, pair)
    wide_from(monkeypatch, 0)
    kv = [(97 * i) % 280 for i in range(44)]
    rows = [40 if i == 9 else 1 + i % 4 for i in range(44)]
    ends = [a + b for a, b in zip(kv, rows)]
    s = Setup(pkg, 16, 4, d, 64, ends, seed=91)
    s.fill(ends)
    q, _ = s.rows(sum(rows), 16, "bf16", 1.5)
    s.batch.plan(kv, rows, s.table)
    for _ in range(2):
        out = s.batch.attend(0, q)
        s.batch.status()
        check_attend(s, kv, rows, q, out, None, "bf16")


def test_attend_few_and_many_columns_in_one_batch(pkg, monkeypatch):
    """A prompt chunk beside decoding sequences: both kernels in one call, the
    partial states of the one after those of the other."""
    wide_from(monkeypatch, 64)
    kv, rows = [1500, 900, 40, 2200], [1, 200, 1, 2]
    s = Setup(pkg, 16, 2, 128, 64, [a + b for a, b in zip(kv, rows)], seed=77)
    s.fill([a + b for a, b in zip(kv, rows)])
    q, _ = s.rows(sum(rows), 16, "bf16", 1.5)
    s.batch.plan(kv, rows, s.table)
    for _ in range(2):
        out = s.batch.attend(0, q)
        s.batch.status()
        check_attend(s, kv, rows, q, out, None, "bf16")


def test_append_many_rows_and_heads_off_the_block_size(pkg):
    """300 rows (a block a row) of head counts that leave threads idle."""
    import torch
    s = Setup(pkg, 9, 3, 64, 32, [310], half=False, seed=50)
    q, qn = s.rows(300, 9, "f16")
    k, kn = s.rows(300, 3, "f16", 2.0)
    v, vn = s.rows(300, 3, "f16")
    s.batch.plan([10], [300], s.table)
    q_out = s.batch.append(0, q, k, v)
    for i in range(300):
        s.store(0, 10 + i, s.turned(kn[i], 10 + i), vn[i])
        assert torch.equal(q_out[i].cpu(), torch.from_numpy(s.turned(qn[i], 10 + i)).half()), i
    assert np.array_equal(s.device_pool(), s.host)


def test_calls_under_graph_capture(pkg):
    """append and attend captured after a plan, and replayed on new rows."""
    import torch
    s = Setup(pkg, 4, 2, 128, 32, [40], seed=60)
    s.fill([33])
    q, _ = s.rows(2, 4, "bf16")
    k, _ = s.rows(2, 2, "bf16", 2.0)
    v, _ = s.rows(2, 2, "bf16")
    q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    turned, out = torch.empty_like(q), torch.empty_like(q)
    s.batch.plan([33], [2], s.table)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        s.batch.append(0, q, k, v, q_out=turned)
        s.batch.attend(0, turned, out=out)
    with pytest.raises(pkg.UnsupportedMethodError, match="capture"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            s.batch.plan([33], [2], s.table)
    for _ in range(2):
        for t in (q, k, v):
            t.copy_(torch.randn_like(t))
        g.replay()
        torch.cuda.synchronize()
        for i in range(2):
            s.store(0, 33 + i, s.turned(k[i].float().cpu().numpy(), 33 + i), v[i].float().cpu().numpy())
        assert np.array_equal(s.device_pool(), s.host)
        check_attend(s, [33], [2], turned, out, None, "bf16")


def test_long_context_split_over_many_blocks(pkg):
    """5000 tokens of one sequence beside short ones: the long axis is split and joined."""
    kv, rows = [5000, 2, 700], [2, 2, 2]
    s = Setup(pkg, 4, 1, 64, 128, [5002, 4, 702], seed=30)
    s.fill([5002, 4, 702])
    q, _ = s.rows(6, 4, "bf16", 2.0)
    s.batch.plan(kv, rows, s.table)
    out = s.batch.attend(0, q)
    s.batch.status()
    check_attend(s, kv, rows, q, out, None, "bf16")


def test_pool_past_32_bits(pkg):
    """Pages whose byte offset passes 2^32: the last pages of a 5 GB pool."""
    import torch
    d, p, kvh, layers = 128, 128, 8, 2
    n_pages = 16000  # 2 layers x 16000 x 8 x 20480 B = 5.2 GB
    size = pkg.KV4Cache.pool_bytes(n_layers=layers, n_kv_heads=kvh, head_dim=d, page_tokens=p, n_pages=n_pages)
    assert size > 1 << 32
    pool = torch.zeros(size, dtype=torch.uint8, device="cuda")
    cache = pkg.KV4Cache(pool, n_layers=layers, n_heads=8, n_kv_heads=kvh, head_dim=d, page_tokens=p, n_pages=n_pages)
    b = pkg.KV4Batch(cache)
    rows = 130
    gen = torch.Generator(device="cuda").manual_seed(1)
    k = torch.randn(rows, kvh, d, device="cuda", generator=gen)
    v = torch.randn(rows, kvh, d, device="cuda", generator=gen)
    q = torch.randn(rows, 8, d, device="cuda", generator=gen).bfloat16()
    outs = []
    for table in ([n_pages - 1, n_pages - 7], [3, 0]):
        b.plan([0], [rows], [table])
        b.append(layers - 1, None, k, v)
        outs.append(b.attend(layers - 1, q))
    b.status()
    assert torch.equal(outs[0], outs[1])
    block = ref.block_bytes(p, d) * kvh
    view = pool.view(layers, n_pages, block)
    assert torch.equal(view[1, n_pages - 1], view[1, 3]) and torch.equal(view[1, n_pages - 7, :1], view[1, 0, :1])
    assert not view[0].any()


def test_refusals(pkg):
    import torch
    s = Setup(pkg, 4, 2, 64, 16, [40, 40], seed=40)
    b, t = s.batch, s.table
    q, k = (torch.zeros(4, n, 64, dtype=torch.bfloat16, device="cuda") for n in (4, 2))
    with pytest.raises(pkg.SamplingError, match="no plan"):
        b.append(0, None, k, k)
    for bad in ([-1], [41]):  # negative, past the table's 3 pages with 8 rows
        with pytest.raises(pkg.SamplingError):
            b.plan(bad, [8], [t[0]])
    with pytest.raises(pkg.SamplingError):
        b.plan([0], [-1], [t[0]])
    with pytest.raises(pkg.SamplingError, match="page"):
        b.plan([0], [1], [[s.n_pages]])
    with pytest.raises(pkg.SamplingError, match="listed again"):
        b.plan([0, 16], [1, 1], [t[0], [t[0][0], t[1][0]]])  # a written page that another sequence reads
    with pytest.raises(pkg.SamplingError, match="listed again"):
        b.plan([0], [20], [[t[0][0], t[0][0]]])
    b.plan([16, 16], [1, 1], [[t[0][0], t[0][1]], [t[0][0], t[1][1]]])  # a shared prefix page is fine
    with pytest.raises(pkg.UnsupportedMethodError, match="64"):
        b.plan([0], [65], [list(range(5))], masks=[1] * 65)
    with pytest.raises(pkg.SamplingError, match="entries"):
        b.plan([0], [2], [t[0]], masks=[1])
    with pytest.raises(pkg.SamplingError):
        b.plan([0], [1], [t[0]], src_rows=[-2])
    b.plan([0], [4], [t[0]], src_rows=[0, 1, 2, 9])
    with pytest.raises(pkg.SamplingError, match="rows"):
        b.append(0, None, k, k)
    b.plan([0], [4], [t[0]], positions=[0, 1, 2, 10 ** 6])
    with pytest.raises(pkg.SamplingError, match="positions"):
        b.append(0, q, k, k)
    b.plan([0], [4], [t[0]])
    for args in ((2, q, k, k), (-1, q, k, k), (0, q, k, k[:3]), (0, q, q, k), (0, q.cpu(), k, k),
                 (0, q.double(), k, k), (0, q[:, :, ::2], k, k)):
        with pytest.raises(pkg.SamplingError):
            b.append(*args)
    with pytest.raises(pkg.SamplingError, match="f16"):
        b.append(0, q, k, k, k_out=torch.empty_like(k))
    with pytest.raises(pkg.SamplingError, match="overlap"):
        b.attend(0, q, out=torch.empty(4, 1, 64, dtype=torch.bfloat16, device="cuda").expand(4, 4, 64))
    with pytest.raises(pkg.UnsupportedMethodError):
        b.attend(0, q.float())
    with pytest.raises(pkg.SamplingError, match="finite"):
        b.attend(0, q, scale=float("nan"))
    before = s.device_pool().copy()
    assert (before == 255).all()  # nothing was launched
    b.plan([], [], [])
    assert b.attend(0, q[:0]).shape == (0, 4, 64)
    b.close()
    with pytest.raises(pkg.SamplingError):
        b.attend(0, q)


def test_batch_outlives_its_cache_handle(pkg):
    s = Setup(pkg, 4, 2, 64, 16, [20], seed=41)
    s.fill([20])
    s.cache.close()
    q, _ = s.rows(1, 4, "bf16")
    s.batch.plan([19], [1], s.table)
    check_attend(s, [19], [1], q, s.batch.attend(0, q), None, "bf16")


def test_tree_decoding_example(pkg):
    """Draft trees over the paged cache commit the tokens of a token a step, in fewer steps."""
    import importlib.util
    import os
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "kv4_tree_decoding.py")
    spec = importlib.util.spec_from_file_location("kv4_tree_decoding", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    same, steps, tokens = mod.run()
    assert same and tokens > 1.3 * steps
