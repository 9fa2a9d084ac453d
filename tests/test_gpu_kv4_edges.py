"""4-bit paged KV cache on the GPU, edges: scores of any finite size, rows
around the clamp, a context of half a billion tokens, outputs that overlap
themselves, errors left behind, the size of the error, and joins of more than
one round."""

import numpy as np
import pytest

from kv4_error import exact_and_deviation, in_deviations
from test_gpu_kv4 import Setup, one_tile, wide_from

pytestmark = pytest.mark.gpu

# Which kernel takes the columns: the one for few, the one for many in two tiles, and in one with stages in pairs.
KERNELS = ["few", "many", "pairs"]


def on(monkeypatch, kernel):
    wide_from(monkeypatch, 1 << 20 if kernel == "few" else 0)
    if kernel != "few":
        one_tile(monkeypatch, kernel == "pairs")


def stored_rows(s, n, k, v):
    """Appends f32 rows k, v [n, kv heads, d] to the one sequence; their stored values in float64."""
    import torch
    s.batch.plan([0], [n], s.table)
    s.batch.append(0, None, torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda())
    for i in range(n):
        s.store(0, i, k[i], v[i])
    return s.values(0, n)


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("logit", [1e4, 1e7, 1e9, 1e12, 1e20])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("d,heads,rows", [(128, 8, 4), (64, 6, 30)])
def test_attend_far_scores_take_the_largest(pkg, monkeypatch, kernel, logit, sign, d, heads, rows):
    """One score of every column stands far above the others: the output is its
    token's value, at any size of the scores.  The largest score grows from
    stage to stage, so the reference moves late as well as early."""
    import torch
    on(monkeypatch, kernel)
    n = 700
    s = Setup(pkg, heads, 1, d, 64, [n], rope=False, seed=int(np.log10(logit)))
    # Keys along one pattern of signs, lengths of both signs, every stage's
    # extremes 10 % past the others and 30 % past the stage before.
    pattern = np.sign(s.rng.standard_normal(d)).astype(np.float32)
    size = s.rng.uniform(-1, 1, n).astype(np.float32)
    for st in range(0, n, 128):
        top, low = s.rng.permutation(min(128, n - rows - st))[:2] + st
        size[top], size[low] = 1.1, -1.1
        size[st:st + 128] *= np.float32(1.3 ** (st // 128))
    k = size[:, None, None] * pattern[None, None]
    v = s.rng.standard_normal((n, 1, d)).astype(np.float32)
    kk, vv = stored_rows(s, n, k, v)
    q = (pattern * s.rng.uniform(0.5, 1, (rows, heads, 1)) * logit / np.sqrt(d)).astype(np.float32)
    q = torch.from_numpy(q).cuda().bfloat16()
    s.batch.plan([n - rows], [rows], s.table)
    scale = sign * d ** -0.5
    out = s.batch.attend(0, q, out=torch.empty(rows, heads, d, device="cuda"), scale=scale)
    s.batch.status()
    got, qn = out.cpu().numpy(), q.float().cpu().numpy().astype(np.float64)
    for i in range(rows):
        seen = n - rows + i + 1
        scores = np.einsum("td,hd->ht", kk[:seen, 0], qn[i]) * scale
        order = np.sort(scores, 1)
        # Far enough apart for f16 keys (2^-11) and their exponentials.
        assert (order[:, -1] - order[:, -2] > 0.02 * np.abs(order[:, -1]) + 30).all()
        want = vv[scores.argmax(1), 0]
        # One weight and one value, each rounded to f16: kv4_ref.attend's term of 2.5 roundings.
        assert (np.abs(got[i] - want) <= 2.5 * 2.0 ** -11 * np.abs(want) + 1e-6).all(), i


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("logit", [1e3, 1e6, 1e8, 1e9, 3e9, 1e12, 1e20])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("d,heads", [(128, 32), (64, 5)])
def test_attend_equal_scores_share_alike(pkg, monkeypatch, kernel, logit, sign, d, heads):
    """All keys are one row: every output is the mean of the values seen, at any size of the scores."""
    import torch
    on(monkeypatch, kernel)
    n, rows = 300, 5
    s = Setup(pkg, heads, 1, d, 32, [n], rope=False, seed=77)
    k = np.repeat(s.rng.standard_normal((1, 1, d)).astype(np.float32), n, 0)
    v = s.rng.standard_normal((n, 1, d)).astype(np.float32)
    kk, vv = stored_rows(s, n, k, v)
    # q along the key, so that the score is the sum of |.| and columns differ in size.
    q = np.sign(kk[0, 0]) * s.rng.uniform(0.5, 1, (rows, heads, 1)) * logit / np.abs(kk[0, 0]).sum() * np.sqrt(d)
    q = torch.from_numpy(q.astype(np.float32)).cuda().bfloat16()
    s.batch.plan([n - rows], [rows], s.table)
    out = s.batch.attend(0, q, out=torch.empty(rows, heads, d, device="cuda"), scale=sign * d ** -0.5)
    s.batch.status()
    got = out.cpu().numpy()
    for i in range(rows):
        seen = vv[:n - rows + i + 1, 0]
        want = seen.mean(0)
        # Values as f16 (2^-11), weights all alike (as f16 2^-11 once more where
        # the largest exponent is not 0), sums in f32.
        bound = (2.0 ** -11 + 2.0 ** -11 + 2.0 ** -18) * np.abs(seen).mean(0) + 1e-6
        assert (np.abs(got[i] - want) <= bound).all(), i


def same_bytes_or_nan(got, want):
    """Equal pools, but for the payloads of NaN scales."""
    a, b = (np.frombuffer(x.tobytes(), np.float16) for x in (got, want))
    pair = (got == want).reshape(-1, 2).all(1) | (np.isnan(a) & np.isnan(b))
    return pair.all()


@pytest.mark.parametrize("d,wide", [(128, True), (64, True), (128, False)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_append_rows_around_the_clamp(pkg, d, wide, dtype):
    """Groups that lie across +-20000 are clamped before they are coded: their
    clamped range is small and o is rounded to 16 there, so that a value past
    the clamp need not have the least or the largest code."""
    import torch
    n, kv = 40, 2
    s = Setup(pkg, 2, kv, d, 16, [n], rope=False, seed=d)
    x = np.empty((n, kv, d), np.float32)
    for i in range(n):
        half_width = [10, 40, 100, 1000, 9000][i % 5]
        x[i] = (20000 + s.rng.uniform(-1, 1, (kv, d)) * half_width) * (1 if i % 2 else -1)
    x[0, 0], x[1, 0] = np.linspace(19990, 20010, d), np.linspace(-20010, -19990, d)
    x[2, 1, 3], x[3, 1, d - 1], x[4, 0, 7] = np.inf, -np.inf, -30000
    x[5] = 25000  # a group all past the clamp
    k = torch.from_numpy(x).cuda().to(torch.float32 if dtype == "f32" else torch.bfloat16)
    v = k.flip(0).contiguous()
    if not wide:  # rows that are not 16-byte pieces
        k, v = (torch.cat([t, t[:, :, :1]], 2)[:, :, :d] for t in (k, v))
    k_out, v_out = (torch.empty(n, kv, d, dtype=torch.float16, device="cuda") for _ in range(2))
    s.batch.plan([0], [n], s.table)
    s.batch.append(0, None, k, v, k_out=k_out, v_out=v_out)
    kn, vn = k.float().cpu().numpy(), v.float().cpu().numpy()
    for i in range(n):
        val = s.store(0, i, kn[i], vn[i])
        assert np.array_equal(k_out[i].cpu().numpy(), val[0].astype(np.float16)), i
        assert np.array_equal(v_out[i].cpu().numpy(), val[1].astype(np.float16)), i
    assert same_bytes_or_nan(s.device_pool(), s.host)


def test_attend_length_times_parts_past_32_bits(pkg, monkeypatch):
    """A context of 4.2 million stages in some hundred parts.  Its table lists
    one page over and over, so the attention is that over the page's tokens."""
    import torch
    on(monkeypatch, "few")
    d, p = 64, 128
    stages = 4_200_000
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    assert stages * sms * 4 > 1 << 31
    s = Setup(pkg, 1, 1, d, p, [p + 1], rope=False, seed=6)
    s.fill([p + 1])
    table = np.full((1, stages + 1), s.table[0][0], np.int32)
    table[0, -1] = s.table[0][1]
    q, _ = s.rows(1, 1, "bf16", 1.5)
    s.batch.plan([p], [1], s.table)
    want = s.batch.attend(0, q, out=torch.empty(1, 1, d, device="cuda")).cpu().numpy()[0, 0]
    s.batch.plan([stages * p], [1], table)
    got = s.batch.attend(0, q, out=torch.empty(1, 1, d, device="cuda")).cpu().numpy()[0, 0]
    s.batch.status()
    # The token after the pages weighs 1 / 4.2e6 of them here and is an
    # 129th of what is seen there: it is taken out of the first.
    k, v = s.values(0, p + 1)
    score = np.exp(k[:, 0] @ q[0, 0].float().cpu().numpy().astype(np.float64) * d ** -0.5)
    mean = score[:p] @ v[:p, 0] / score[:p].sum()
    one = score @ v[:, 0] / score.sum()
    near = np.abs(v[:p + 1, 0]).max()
    assert np.abs(want - one).max() <= 2.5 * 2.0 ** -11 * near + 1e-6
    # f32 running sums of a warp: 4.2e6 * 4 / (4 sms * 4 warps) tiles of 32
    # tokens, 8 additions a lane and tile, half an ulp (2^-24) each and the
    # matrix products' truncation (2^-23) as much again, all one way.
    tiles = stages * 4 / (sms * 4 * 4)
    assert np.abs(got - mean).max() <= (2.5 * 2.0 ** -11 + tiles * 8 * 2.0 ** -23) * near + 1e-6


def test_outputs_that_overlap_themselves_are_refused(pkg):
    """Rows and heads whose strides make them meet, and layouts that look alike but do not."""
    import torch
    s = Setup(pkg, 4, 2, 64, 16, [40], seed=42)
    s.fill([36])
    b, d = s.batch, 64
    q = torch.randn(4, 4, d, device="cuda").bfloat16()
    k = torch.randn(4, 2, d, device="cuda").bfloat16()
    b.plan([32], [4], s.table)
    room = torch.zeros(40 * d, dtype=torch.bfloat16, device="cuda")

    def out(heads, row, head, dtype=None):
        t = room if dtype is None else room.to(dtype)
        return t.as_strided((4, heads, d), (row, head, 1))

    want = b.attend(0, q)
    for row, head in ((d, d), (2 * d, d), (3 * d, 2 * d), (d + 8, d), (d, d + 8), (4 * d - 8, d), (d, 4 * d - 8),
                      (5 * d, 5 * d)):
        with pytest.raises(pkg.SamplingError, match="overlap"):
            b.attend(0, q, out=out(4, row, head))
    for row, head in ((4 * d, d), (d, 4 * d), (d + 8, 4 * (d + 8)), (2 * d, 8 * d), (5 * d, d + 8), (3 * d, 4 * d)):
        got = b.attend(0, q, out=out(4, row, head))
        assert torch.equal(got, want), (row, head)
    got = b.append(0, q, k, k, q_out=torch.empty_like(q))
    with pytest.raises(pkg.SamplingError, match="overlap"):
        b.append(0, q, k, k, q_out=out(4, d, d))
    with pytest.raises(pkg.SamplingError, match="overlap"):
        b.append(0, q, k, k, q_out=got, k_out=out(2, d, d, torch.float16))
    with pytest.raises(pkg.SamplingError, match="overlap"):
        b.append(0, q, k, k, q_out=got, v_out=out(2, d, d, torch.float16))
    b.append(0, q, k, k, q_out=got, k_out=out(2, 3 * d, 2 * d, torch.float16))  # interleaved, nothing shared
    b.plan([32], [1], s.table)  # one row: its stride is not used
    assert torch.equal(b.attend(0, q[:1], out=out(4, d, d)[:1]), b.attend(0, q[:1]))


def test_a_failed_call_leaves_no_error_behind(pkg):
    """A CUDA error that a call returned is not the next call's: an upload and a
    matmul, whose launches are checked, go through after it."""
    import ctypes
    from importlib import import_module
    import torch
    raw = import_module("abyo-speculate_b200._lib")
    synth = import_module("abyo-speculate_b200.gguf_synth")
    lib = raw.load()
    pool = torch.zeros(1 << 20, dtype=torch.uint8, device="cuda")
    desc = raw.KV4Desc(9999, 1, 2, 2, 64, 16, 4, 1)  # no such device
    cache, batch = ctypes.c_void_p(), ctypes.c_void_p()
    assert lib.spec_kv4_create(ctypes.byref(desc), pool.data_ptr(), pool.numel(), None, None, 0, ctypes.byref(cache)) == 0
    x, y = torch.ones(1, 256, device="cuda"), torch.zeros(1, 128, device="cuda")
    for _ in range(2):
        assert lib.spec_kv4_batch_create(cache, ctypes.byref(batch)) == raw.SPEC_ERR_CUDA
        w = pkg.QWeight(8, synth.quantize(np.ones((128, 256), np.float32), 8), 128, 256)
        assert lib.spec_kv4_batch_create(cache, ctypes.byref(batch)) == raw.SPEC_ERR_CUDA
        w.matmul(x.data_ptr(), 1, y.zero_().data_ptr(), torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        assert torch.allclose(y, torch.full_like(y, 256.0), rtol=1e-2)
    lib.spec_kv4_free(cache)


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("logit", [-1e31, -1e34, -2e37, 2e37])
@pytest.mark.parametrize("n", [40, 300, 3000])
def test_attend_scores_past_1e30(pkg, monkeypatch, kernel, logit, n):
    """Equal scores of any finite size: a row that sees tokens gives their mean,
    in one part, two accumulators and many parts alike."""
    import torch
    on(monkeypatch, kernel)
    d, heads, rows = 64, 4, 2
    s = Setup(pkg, heads, 1, d, 64, [n], rope=False, seed=5)
    k = np.repeat(s.rng.standard_normal((1, 1, d)).astype(np.float32), n, 0)
    v = s.rng.standard_normal((n, 1, d)).astype(np.float32)
    kk, vv = stored_rows(s, n, k, v)
    q = np.sign(kk[0, 0]) * s.rng.uniform(0.5, 1, (rows, heads, 1)) * logit / np.abs(kk[0, 0]).sum() * np.sqrt(d)
    q = torch.from_numpy(q.astype(np.float32)).cuda().bfloat16()
    s.batch.plan([n - rows], [rows], s.table)
    got = s.batch.attend(0, q, out=torch.empty(rows, heads, d, device="cuda")).cpu().numpy()
    s.batch.status()
    for i in range(rows):
        seen = vv[:n - rows + i + 1, 0]
        bound = (2.0 ** -11 + 2.0 ** -11 + 2.0 ** -16) * np.abs(seen).mean(0) + 1e-6
        assert (np.abs(got[i] - seen.mean(0)) <= bound).all(), i


def narrow_tiles(monkeypatch, most):
    monkeypatch.setenv("SPEC_B200_KV4_NARROW_COLS", str(most))


@pytest.mark.parametrize("kernel,most", [("few", 8), ("few", 16), ("few", 32), ("many", 32), ("pairs", 32)])
@pytest.mark.parametrize("d,page,q_type", [(128, 64, "bf16"), (128, 16, "f16"), (64, 32, "bf16"), (64, 128, "f16")])
def test_attend_error_is_that_of_its_roundings(pkg, monkeypatch, kernel, most, d, page, q_type):
    """Values and weights rounded to f16 once each; keys too in the kernel for
    many columns, and not in the one for few."""
    import torch
    on(monkeypatch, kernel)
    narrow_tiles(monkeypatch, most)
    n, rows, heads, kv_heads = 600, 7, 8, 2
    s = Setup(pkg, heads, kv_heads, d, page, [n], seed=d + most)
    s.fill([n])
    q, qn = s.rows(rows, heads, q_type, 2.0)
    s.batch.plan([n - rows], [rows], s.table)
    got = s.batch.attend(0, q, out=torch.empty(rows, heads, d, device="cuda")).cpu().numpy()
    s.batch.status()
    k, v = s.values(0, n)
    want, dev = exact_and_deviation(qn.astype(np.float64), k, v, np.tri(rows, n, n - rows), d ** -0.5, kernel != "few")
    assert in_deviations(got, want, dev) < 1


@pytest.mark.parametrize("kernel,most", [("few", 8), ("few", 16), ("few", 32), ("many", 32), ("pairs", 32)])
@pytest.mark.parametrize("tokens", [2200, 12000, 40000])
@pytest.mark.parametrize("d", [64, 128])
def test_attend_contexts_in_many_parts(pkg, monkeypatch, kernel, most, tokens, d):
    """Long contexts of one KV head: 18, 94 and 313 stages, up to one a block, so
    that partial states are joined in two and three rounds.  The table lists 20
    pages over and over."""
    import torch
    on(monkeypatch, kernel)
    narrow_tiles(monkeypatch, most)
    p, rows, heads = 32, 3, 4
    s = Setup(pkg, heads, 1, d, p, [20 * p + rows], rope=False, seed=tokens + d)
    s.fill([20 * p])
    listed = s.rng.integers(0, 20, tokens // p)
    kv_len = len(listed) * p
    table = [s.table[0][i] for i in listed] + [s.table[0][20]]
    k, kn = s.rows(rows, 1, "f32", 1.5)
    v, vn = s.rows(rows, 1, "f32")
    s.batch.plan([kv_len], [rows], [table])
    s.batch.append(0, None, k, v)
    for i in range(rows):
        s.store(0, 20 * p + i, kn[i], vn[i])
    q, qn = s.rows(rows, heads, "bf16", 2.0)
    got = s.batch.attend(0, q, out=torch.empty(rows, heads, d, device="cuda"))
    again = s.batch.attend(0, q, out=torch.empty_like(got))
    s.batch.status()
    assert torch.equal(got, again)
    kk, vv = s.values(0, 20 * p + rows)
    times = np.concatenate([np.repeat(np.bincount(listed, minlength=20), p), np.zeros(rows)])
    see = np.repeat(times[None], rows, 0)
    see[:, 20 * p:] = np.tri(rows)
    want, dev = exact_and_deviation(qn.astype(np.float64), kk, vv, see, d ** -0.5, kernel != "few")
    assert in_deviations(got.cpu().numpy(), want, dev) < 1
