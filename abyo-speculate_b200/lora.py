"""Low-rank adapters of many requests over torch tensors: the host side of spec_lora_* (include/spec_b200.h).

    bank = LoraBank(a, b, ranks=..., scales=...)     # of one projection: a [adapters, rank, k], b [adapters, n, rank]
    plan = LoraPlan(adapter_of_each_row, n_adapters)  # once per step, for all projections and layers
    w.matmul(x.data_ptr(), rows, y.data_ptr(), stream)  # the shared projection
    bank.apply(plan, x, y)                            # y += scale (x A^T) B^T

Calls are queued on torch's current stream of the bank's device and return
without waiting for it.  No gradients are recorded.
"""

from __future__ import annotations

import ctypes
import struct
from typing import Optional

import numpy as np

from . import _lib
from .sampling import _setup
from .kv4 import _host


_THREE_ROWS = struct.Struct("=" + "Qqqii" * 3)  # spec_lora_rows


def _invalid(msg: str) -> _lib.SamplingError:
    return _lib.SamplingError(_lib.SPEC_ERR_INVALID, msg)


class LoraPlan:
    """Which adapter each row of a step has (spec_lora_plan_make).

    adapters: one whole number a row, -1 for a row without an adapter; rows of
    one adapter need not be neighbours.  The plan does not change: a captured
    call replays with it as long as it lives."""

    def __init__(self, adapters, n_adapters: int, device="cuda"):
        import torch
        lib = _lib.load()
        ids = _host(adapters, np.int32, "adapters")
        self.n_rows, self.n_adapters = int(ids.size), int(n_adapters)
        size = lib.spec_lora_plan_bytes(self.n_rows)
        if size < 0:
            _lib.check(-size)
        buf = np.empty(max(size, 1), np.uint8)
        self._desc = _lib.LoraPlanDesc()
        _lib.check(lib.spec_lora_plan_make(ids.ctypes.data, self.n_rows, self.n_adapters, buf.ctypes.data, size,
                                           ctypes.byref(self._desc)))
        self._copy = torch.from_numpy(buf).to(device)
        self.device = self._copy.device
        if not self._copy.is_cuda:
            raise _invalid(f"a plan on {self.device}: a CUDA device is needed")
        self._desc.device_copy = self._copy.data_ptr()
        self._at = ctypes.addressof(self._desc)
        self._seen = set()  # streams that calls ran on

    def status(self) -> None:
        """Waits for the current stream's calls; raises if a device wait in a call with this plan gave up."""
        _, lib, _, current = _setup()
        _lib.check(lib.spec_lora_status(self._at, self.device.index, current(self.device.index)))


class LoraBank:
    """The adapters of one projection (spec_lora_bank).

    a [adapters, rank, k] and b [adapters, n, rank]: bfloat16 or float16 CUDA
    tensors with contiguous rows, kept as they are.  ranks: adapters' own ranks
    (what lies behind them in a and b does not count), whole numbers or an int32 tensor
    on the device; scales: numbers or a float32 tensor on the device."""

    def __init__(self, a, b, ranks=None, scales=None):
        import torch
        self._lib = _lib.load()
        types = {torch.bfloat16: 0, torch.float16: 1}
        if not all(isinstance(t, torch.Tensor) and t.is_cuda and t.dim() == 3 for t in (a, b)):
            raise _invalid("a and b are not CUDA tensors of three dimensions")
        if a.dtype not in types or b.dtype != a.dtype or a.device != b.device:
            raise _invalid(f"a is {a.dtype} on {a.device}, b {b.dtype} on {b.device}: both bfloat16 or float16 on one device")
        n, r, k = a.shape
        if b.shape[0] != n or b.shape[2] != r:
            raise _invalid(f"a has shape {tuple(a.shape)}, b {tuple(b.shape)}: [adapters, rank, k] and [adapters, n, rank]")
        for t, what in ((a, "a"), (b, "b")):
            if t.shape[2] > 1 and t.stride(2) != 1:
                raise _invalid(f"the rows of {what} are not contiguous")
        self.device, self.n_adapters, self.rank, self.k, self.n = a.device, n, r, k, b.shape[1]
        if ranks is not None and not isinstance(ranks, torch.Tensor):
            host = _host(ranks, np.int32, "ranks", n)
            if host.size and (host.min() < 0 or host.max() > r):
                raise _invalid(f"ranks from {host.min()} to {host.max()}, 0 to {r} are taken")
            ranks = torch.from_numpy(host.copy()).to(self.device)
        if scales is not None and not isinstance(scales, torch.Tensor):
            scales = torch.tensor([float(s) for s in scales], dtype=torch.float32, device=self.device)
        for t, dtype, what in ((ranks, torch.int32, "ranks"), (scales, torch.float32, "scales")):
            if t is not None and not (t.dtype == dtype and t.device == self.device and tuple(t.shape) == (n,) and
                                      t.is_contiguous()):
                raise _invalid(f"{what} is not a contiguous {dtype} tensor [{n}] on {self.device}")
        self._keep = (a, b, ranks, scales)
        self._seen = set()
        self._types = {a.dtype: types[a.dtype], torch.float32: 2}
        self._desc = _lib.LoraBankDesc(
            a.device.index, n, k, self.n, r, types[a.dtype], a.data_ptr(), b.data_ptr(), a.stride(0), a.stride(1),
            b.stride(0), b.stride(1), ranks.data_ptr() if ranks is not None else None,
            scales.data_ptr() if scales is not None else None)
        self._at, self._index = ctypes.addressof(self._desc), a.device.index

    def _rows(self, t, width: int, what: str):
        """The fields of spec_lora_rows for tensor t [rows, width]."""
        torch = _setup()[0]
        if not isinstance(t, torch.Tensor) or t.get_device() != self._index:
            raise _invalid(f"{what} is not a tensor on {self.device}")
        kind = self._types.get(t.dtype)
        if kind is None:
            raise _invalid(f"{what} is {t.dtype}: float32 and the adapters' type are taken")
        if t.dim() != 2 or t.shape[1] != width:
            raise _invalid(f"{what} has shape {tuple(t.shape)}, [rows, {width}] is needed")
        row, column = t.stride()
        if column != 1 and width > 1:
            raise _invalid(f"the rows of {what} are not contiguous")
        return t.data_ptr(), row, t.shape[0], kind, 0

    def apply(self, plan: LoraPlan, x, y, out=None):
        """out = y + scale (x A^T) B^T, each row with its own adapter; x [rows, k],
        y and out [rows, n] (out None: y itself; otherwise memory of neither x nor y).  Returns out."""
        torch, lib, _, current = _setup()
        if plan.device != self.device:
            raise _invalid(f"the plan is on {plan.device}, the bank on {self.device}")
        if out is None:
            out = y
        rows = _THREE_ROWS.pack(*self._rows(x, self.k, "x"), *self._rows(y, self.n, "y"), *self._rows(out, self.n, "out"))
        stream = current(self._index)
        # The three structures lie behind one another.
        at = ctypes.cast(ctypes.c_char_p(rows), ctypes.c_void_p).value
        rc = lib.spec_lora_apply(self._at, plan._at, at, at + 32, at + 64, stream)
        if rc:
            _lib.check(rc)
        # Memory of a plan or bank that is dropped is not handed out before this stream is done with it.  Each stream
        # counts, whichever was current when the bank was made: the caller's tensors may be of another one.
        if stream not in plan._seen:
            plan._seen.add(stream)
            plan._copy.record_stream(torch.cuda.current_stream(self.device))
        if stream not in self._seen:
            self._seen.add(stream)
            for t in self._keep:
                if t is not None:
                    t.record_stream(torch.cuda.current_stream(self.device))
        return out
