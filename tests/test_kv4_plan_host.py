"""What KV4Batch.plan hands to the library, on the CPU: the library's plan is replaced by one that copies its arguments."""

import ctypes
import gc
import types
import weakref
from importlib import import_module

import numpy as np
import pytest

kv4 = import_module("abyo-speculate_b200.kv4")


class Recorder:
    """Stands for the library: keeps a copy of the step it is given."""

    def spec_kv4_plan(self, handle, step, stream):
        s = ctypes.cast(step, ctypes.POINTER(kv4._lib.KV4Step)).contents

        def read(p, n, kind):
            return None if not p else list(ctypes.cast(p, ctypes.POINTER(kind))[:n])

        n = s.n_seqs
        self.kv, self.rows = read(s.kv_len, n, ctypes.c_int32), read(s.n_rows, n, ctypes.c_int32)
        total = sum(self.rows or [])
        self.stride = s.table_stride
        self.table = read(s.page_table, n * s.table_stride, ctypes.c_int32)
        self.pos, self.src = read(s.positions, total, ctypes.c_int32), read(s.src_rows, total, ctypes.c_int32)
        self.masks = read(s.masks, total, ctypes.c_uint64)
        return 0


@pytest.fixture
def batch():
    b = kv4.KV4Batch.__new__(kv4.KV4Batch)
    b._lib, b._h, b._stream = Recorder(), None, lambda: 0
    return b


FORMS = [list, tuple, np.array, lambda x: np.array(x, np.int32), lambda x: np.array(x, np.uint64),
         lambda x: [np.int64(v) for v in x]]


@pytest.mark.parametrize("form", FORMS)
def test_whole_numbers_arrive_as_they_are(batch, form):
    batch.plan(form([7, 0]), form([2, 1]), [form([4, 5]), form([9])], positions=form([3, 3, 0]), masks=form([1, 3, 1]),
               src_rows=form([2, 1, 0]))
    r = batch._lib
    assert (r.kv, r.rows, r.stride, r.table) == ([7, 0], [2, 1], 2, [4, 5, 9, -1])
    assert (r.pos, r.masks, r.src) == ([3, 3, 0], [1, 3, 1], [2, 1, 0])
    assert batch.n_rows == 3


@pytest.mark.parametrize("kind", [np.int32, np.int64, np.uint16, np.uint64])
def test_tables_as_one_array(batch, kind):
    batch.plan([5, 6], [1, 1], np.array([[3, 4, 0], [8, 9, 1]], kind))
    assert (batch._lib.stride, batch._lib.table) == (3, [3, 4, 0, 8, 9, 1])


def test_masks_of_all_64_bits(batch):
    top = (1 << 63) | 5
    for masks in ([top, 3], np.array([top, 3], np.uint64), np.array([top - (1 << 64), 3], np.int64)):
        batch.plan([0], [2], [[0]], masks=masks)
        assert batch._lib.masks == [top, 3]


LOST = [np.array([2 ** 32 + 5]), np.array([-2 ** 33]), np.array([2 ** 31], np.uint32), np.array([2 ** 64 - 1], np.uint64),
        np.array([3.7]), np.array([3.0], np.float32), [3.7], [2 ** 31], [-2 ** 40], (2 ** 64,), np.array(["1"]), [None]]


@pytest.mark.parametrize("bad", LOST)
def test_numbers_that_would_change_are_refused(pkg, batch, bad):
    ok = dict(kv_len=[0], n_rows=[1], page_table=[[2]], positions=[0], src_rows=[0])
    batch.plan(**ok)
    for name in ("kv_len", "n_rows", "positions", "src_rows"):
        with pytest.raises(pkg.SamplingError, match=name):
            batch.plan(**{**ok, name: bad})
    for table in ([bad], np.array([bad]) if isinstance(bad, np.ndarray) else [list(bad)]):
        with pytest.raises(pkg.SamplingError, match="page_table"):
            batch.plan(**{**ok, "page_table": table})


@pytest.mark.parametrize("bad", [[-1], [1 << 64], [0.5], np.array([-1], np.int32), np.array([1.0])])
def test_masks_that_would_change_are_refused(pkg, batch, bad):
    with pytest.raises(pkg.SamplingError, match="masks"):
        batch.plan([0], [1], [[0]], masks=bad)


@pytest.mark.parametrize("table", [[[], []], np.zeros((2, 0), np.int32), np.zeros((2, 0)), [np.zeros(0, np.int32)] * 2])
def test_tables_without_pages_list_none(batch, table):
    """A table of no columns still has one entry a sequence, which is no page."""
    batch.plan([0, 0], [1, 1], table)
    assert (batch._lib.stride, batch._lib.table) == (1, [-1, -1])


def test_a_dropped_batch_is_freed_at_once(monkeypatch):
    """Its workspace goes with the last reference, not when the collector finds
    a cycle (which may be inside somebody's stream capture)."""
    import torch  # noqa: F401  (a first import inside the constructor would keep its frame)
    freed = []

    class Lib:
        def spec_kv4_batch_create(self, cache, out):
            ctypes.cast(out, ctypes.POINTER(ctypes.c_void_p))[0] = 16
            return 0

        def spec_kv4_batch_free(self, handle):
            freed.append(handle.value)

    monkeypatch.setattr(kv4._lib, "load", Lib)
    cache = types.SimpleNamespace(_h=ctypes.c_void_p(8), head_dim=64, device=types.SimpleNamespace(index=0))
    on = gc.isenabled()
    gc.disable()
    try:
        batch = kv4.KV4Batch(cache)
        seen = weakref.ref(batch)
        del batch
        assert seen() is None and freed == [16]
    finally:
        if on:
            gc.enable()
