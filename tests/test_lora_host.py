"""Low-rank adapters, what needs no GPU: plans and refusals, which come before any CUDA call."""

import ctypes

import numpy as np
import pytest

P = 1 << 20  # a pointer that nothing follows


@pytest.fixture(scope="module")
def mod():
    from importlib import import_module
    return import_module("abyo-speculate_b200._lib")


def make(mod, ids, n_adapters):
    lib = mod.load()
    ids = np.asarray(ids, np.int32)
    buf = np.zeros(max(1, lib.spec_lora_plan_bytes(ids.size)), np.uint8)
    plan = mod.LoraPlanDesc()
    rc = lib.spec_lora_plan_make(ids.ctypes.data, ids.size, n_adapters, buf.ctypes.data, buf.size, ctypes.byref(plan))
    return rc, plan, buf


@pytest.mark.parametrize("n,adapters,seed", [(1, 1, 0), (7, 3, 1), (64, 64, 2), (300, 2, 3), (2000, 5, 4), (40, 1, 5), (9000, 2, 6)])
def test_every_row_is_in_one_unit_of_its_adapter(mod, n, adapters, seed):
    rng = np.random.default_rng(seed)
    ids = rng.integers(-1, adapters, n)
    rc, plan, buf = make(mod, ids, adapters)
    assert rc == 0 and plan.n_rows == n and plan.n_adapters == adapters
    counts = [plan.n_tall, plan.n_big, plan.n_wide, plan.n_narrow, plan.n_bare]
    units = buf[:48 * sum(counts)].view(np.int32).reshape(-1, 12)
    order = buf[48 * n:52 * n].view(np.int32)
    kind = np.repeat(np.arange(5), counts)
    seen = [[], [], [], [], []]
    for k, (a, first, count, _, *near) in zip(kind, units):
        assert 0 < count <= (128, 64, 64, 8, 1)[k] and (a >= 0) == (k < 4)
        assert near[:count] == order[first:first + min(count, 8)].tolist()
        rows = order[first:first + count]
        assert (ids[rows] == a).all()
        seen[k] += rows.tolist()
    assert sorted(sum(seen[1:], [])) == list(range(n))
    assert sorted(seen[0]) == sorted(seen[1])  # the same rows, for another kernel
    assert (buf[52 * n:] == 0).all()


@pytest.mark.parametrize("runs", [(24, 20, 30), (256,), (64, 17, 3), (880,), (900,), (24,) * 60, (200,) + (40,) * 40, (17,) * 37,
                                  (16,) * 30, (5, 70)])
def test_rows_that_units_of_eight_can_take_too(mod, runs):
    ids = np.random.default_rng(0).permutation(np.repeat(np.arange(len(runs)), runs))
    rc, plan, buf = make(mod, ids, len(runs))
    n = ids.size
    order = buf[48 * n:52 * n].view(np.int32)
    main = plan.n_tall + plan.n_big + plan.n_wide + plan.n_narrow + plan.n_bare
    assert rc == 0 and main + plan.n_mid <= n and 0 <= plan.n_mid_wide <= plan.n_wide
    units = buf[:48 * n].view(np.int32).reshape(-1, 12)

    def rows_of(part, most):
        out = []
        for a, first, count, _, *near in part:
            rows = order[first:first + count]
            assert 0 < count <= most and a >= 0 and (ids[rows] == a).all() and near[:min(count, 8)] == rows[:8].tolist()
            out += rows.tolist()
        return sorted(out)

    mid = rows_of(units[main:main + plan.n_mid], 8)
    wide_end = plan.n_tall + plan.n_big + plan.n_wide
    replaced = units[plan.n_tall:wide_end] if plan.mid_all else units[wide_end - plan.n_mid_wide:wide_end]
    assert mid == rows_of(replaced, 64)
    few = sum((r + 7) // 8 for r in runs) <= 111
    assert bool(plan.mid_all) == few and (not few or len(mid) == sum(r for r in runs if r > 16))


def test_empty_plans(mod):
    rc, plan, _ = make(mod, [], 3)
    assert rc == 0 and plan.n_wide == plan.n_narrow == plan.n_bare == 0
    rc, plan, _ = make(mod, [-1, -1], 0)
    assert rc == 0 and plan.n_narrow == 0 and plan.n_bare == 2


def test_bad_plans_are_refused(mod):
    lib = mod.load()
    assert make(mod, [0, 3], 3)[0] == 1 and make(mod, [-2], 3)[0] == 1 and make(mod, [0], -1)[0] == 1
    assert lib.spec_lora_plan_bytes(-1) == -1 and lib.spec_lora_plan_bytes(1 << 21) == -1
    ids, buf, plan = np.zeros(4, np.int32), np.zeros(224, np.uint8), mod.LoraPlanDesc()
    args = [ids.ctypes.data, 4, 1, buf.ctypes.data, 224, ctypes.byref(plan)]
    assert lib.spec_lora_plan_make(*args) == 0
    for at, bad in ((0, None), (1, -1), (3, None), (4, 223), (5, None)):
        assert lib.spec_lora_plan_make(*args[:at], bad, *args[at + 1:]) == 1


def test_bad_calls_are_refused(mod):
    lib = mod.load()

    def call(bank=(), plan=(), x=(), y=(), out=()):
        b = dict(device=0, n_adapters=2, k=64, n=32, rank=8, dtype=0, a=P, b=P, a_adapter_stride=512, a_row_stride=64,
                 b_adapter_stride=256, b_row_stride=8, ranks=None, scales=None)
        p = dict(n_rows=3, n_adapters=2, n_wide=0, n_narrow=1, n_bare=1, n_tall=0, n_big=0, reserved=0, device_copy=P)
        r = [dict(ptr=P, row_stride=64, n_rows=3, dtype=0, reserved=0), dict(ptr=P, row_stride=32, n_rows=3, dtype=0, reserved=0),
             dict(ptr=P + 4096, row_stride=32, n_rows=3, dtype=0, reserved=0)]
        b.update(bank), p.update(plan)
        for d, change in zip(r, (x, y, out)):
            d.update(change)
        rows = [ctypes.byref(mod.LoraRows(**d)) for d in r]
        return lib.spec_lora_apply(ctypes.byref(mod.LoraBankDesc(**b)), ctypes.byref(mod.LoraPlanDesc(**p)), *rows, None)

    for change in (dict(k=0), dict(n=0), dict(k=1 << 25), dict(device=-1), dict(n_adapters=-1), dict(n_adapters=1), dict(a=None),
                   dict(b=None), dict(a=P + 1), dict(ranks=P + 2), dict(scales=P + 1), dict(a_row_stride=-1),
                   dict(b_adapter_stride=1 << 41)):
        assert call(bank=change) == 1, change
    for change in (dict(dtype=2), dict(dtype=-1), dict(rank=129), dict(rank=-1)):
        assert call(bank=change) == 3, change
    for change in (dict(n_rows=-1), dict(n_narrow=-1), dict(n_wide=-1), dict(n_bare=-1), dict(n_narrow=3), dict(n_wide=2), dict(n_tall=-1), dict(n_tall=2), dict(n_big=-1), dict(device_copy=None), dict(device_copy=P + 8),
                   dict(n_rows=(1 << 20) + 1), dict(n_mid=-1), dict(n_mid=2), dict(n_mid_wide=-1), dict(n_mid_wide=1)):
        assert call(plan=change) == 1, change
    for which in ("x", "y", "out"):
        for change in (dict(ptr=None), dict(ptr=P + 1), dict(n_rows=2), dict(row_stride=-1), dict(row_stride=1 << 41)):
            assert call(**{which: change}) == 1, (which, change)
        assert call(**{which: dict(dtype=1)}) == 3
    assert call(y=dict(dtype=2)) == 1                                # y and out of two types
    assert call(out=dict(row_stride=31)) == 1                        # rows that overlap
    assert call(out=dict(ptr=P, row_stride=40)) == 1                 # in place, two strides
    assert lib.spec_lora_apply(None, None, None, None, None, None) == 1
    assert lib.spec_lora_status(None, 0, None) == 1
    assert call(plan=dict(n_rows=0, n_narrow=0, n_bare=0)) == 0       # nothing to do


def test_python_refuses_host_tensors(pkg):
    import torch
    a, b = torch.zeros(2, 4, 8, dtype=torch.bfloat16), torch.zeros(2, 6, 4, dtype=torch.bfloat16)
    with pytest.raises(pkg.SamplingError):
        pkg.LoraBank(a, b)
    with pytest.raises(pkg.SamplingError):
        pkg.LoraPlan([0, 1], 2, device="cpu")
    with pytest.raises(pkg.SamplingError):
        pkg.LoraPlan([0, 2], 2, device="cpu")
    with pytest.raises(pkg.SamplingError):
        pkg.LoraPlan([0.5], 2, device="cpu")


@pytest.mark.parametrize("seed", range(12))
def test_units_fit_their_kernels(mod, seed):
    """At most 128 rows for the kernel of very many, 32 for that of many, 8 for that of few, one without an adapter."""
    rng = np.random.default_rng(seed)
    runs = rng.integers(1, [10, 40, 70, 300, 3000][seed % 5], rng.integers(1, 60))
    ids = rng.permutation(np.concatenate([np.repeat(np.arange(runs.size), runs), np.full(seed, -1)]))
    rc, plan, buf = make(mod, ids, runs.size)
    assert rc == 0
    counts = [plan.n_tall, plan.n_big, plan.n_wide, plan.n_narrow, plan.n_bare, plan.n_mid]
    units = buf[:48 * sum(counts)].view(np.int32).reshape(-1, 12)
    most = np.repeat([128, 32, 32, 8, 1, 8], counts)
    assert (units[:, 2] >= 1).all() and (units[:, 2] <= most).all()
    assert ((units[:, 0] < 0) == (np.repeat(np.arange(6), counts) == 4)).all()
    rows = units[:, 2].astype(np.int64)
    assert sum(rows[sum(counts[:1]):sum(counts[:5])]) == ids.size


@pytest.mark.parametrize("x,y,out", [
    ((P, 48), (P + 8192, 48), (P, 48)),                 # the result in x's place
    ((P, 48), (P, 48), (P, 48)),                        # x, y and the result one
    ((P, 48), (P + 8192, 48), (P + 8192 + 96, 48)),     # y a row further on
    ((P, 48), (P + 8192, 48), (P + 8192 - 2, 48)),      # or an element
    ((P, 0), (P + 8192, 0), (P + 8192 - 94, 48)),       # rows on one another, the result's first one meets them
    ((P, 100), (P + 106, 100), (P + 106 - 10, 100)),    # columns of one wider row that meet
    ((P + 4 * 96 + 40, 0), (P + 8192, 48), (P, 48)),    # x's only row under the result's fifth
    ((P, 96), (P + 8192, 48), (P + 7 * 192 + 95, 50)),  # strides that differ: x's eighth row
])
def test_results_on_their_inputs_are_refused(mod, x, y, out):
    lib = mod.load()
    out = (out[0] & ~1, out[1])
    bank = mod.LoraBankDesc(device=0, n_adapters=1, k=48, n=48, rank=8, dtype=0, a=P, b=P, a_adapter_stride=0, a_row_stride=48,
                            b_adapter_stride=0, b_row_stride=8, ranks=None, scales=None)
    plan = mod.LoraPlanDesc(n_rows=8, n_adapters=1, n_narrow=1, device_copy=P)
    rows = [ctypes.byref(mod.LoraRows(ptr=p, row_stride=s, n_rows=8, dtype=0, reserved=0)) for p, s in (x, y, out)]
    assert lib.spec_lora_apply(ctypes.byref(bank), ctypes.byref(plan), *rows, None) == 1
    assert b"shares memory" in lib.spec_last_error(None)
