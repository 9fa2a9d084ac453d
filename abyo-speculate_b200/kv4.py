"""4-bit paged KV cache over torch tensors: the host side of spec_kv4_* (include/spec_b200.h).

    pool = torch.empty(KV4Cache.pool_bytes(...), dtype=torch.uint8, device="cuda")
    cache = KV4Cache(pool, n_layers=..., n_heads=..., n_kv_heads=..., head_dim=..., page_tokens=..., n_pages=...,
                     rope=rope_tables(head_dim, n_positions, theta))
    step = KV4Batch(cache)
    step.plan(kv_len, n_rows, page_table, masks=...)      # once per step, shared by all layers
    step.append(layer, q, k, v, q_out=q)                  # rotate, quantize, store
    o = step.attend(layer, q)                             # [rows, n_heads, head_dim]

Calls are queued on torch's current stream of the pool's device and return
without waiting for it.
"""

from __future__ import annotations

import array
import ctypes
import math
import struct
from typing import Optional, Sequence, Tuple

import numpy as np

from . import _lib


_TWO_ROWS, _SIX_ROWS = struct.Struct("=" + "Qqqqii" * 2), struct.Struct("=" + "Qqqqii" * 6)  # spec_kv4_rows
_NONE = (0,) * 6


def _invalid(msg: str) -> _lib.SamplingError:
    return _lib.SamplingError(_lib.SPEC_ERR_INVALID, msg)


_CODES = {np.int32: "i", np.uint64: "Q"}


def _host(a, dtype, what: str, n: Optional[int] = None) -> np.ndarray:
    """Whole numbers `a` as a flat contiguous array of `dtype`, every one of them
    as it is: what is not whole or does not fit is refused.  (Signed 64-bit
    arrays stand for 64-bit masks bit by bit.)"""
    x = None
    try:
        if isinstance(a, (list, tuple)):
            try:
                x = np.asarray(array.array(_CODES[dtype], a))
            except TypeError:  # not flat, or not whole
                pass
        if x is None:
            x = np.asarray(a)
            if x.size and x.dtype.kind not in "iub":
                raise _invalid(f"{what}: {x.dtype} entries, whole numbers are needed")
            if x.dtype == np.int64 and dtype == np.uint64 and not isinstance(a, (list, tuple)):
                x = x.view(np.uint64)
            if x.size and not np.can_cast(x.dtype, dtype):
                lo, hi, ends = x.min(), x.max(), np.iinfo(dtype)
                if lo < ends.min or hi > ends.max:
                    raise _invalid(f"{what}: entries {lo} to {hi} do not fit {np.dtype(dtype)}")
        out = np.ascontiguousarray(x.reshape(-1), dtype=dtype)
    except (OverflowError, ValueError, TypeError) as e:
        raise _invalid(f"{what}: {e}") from None
    if n is not None and out.size != n:
        raise _invalid(f"{what} has {out.size} entries, {n} are needed")
    return out


def rope_tables(head_dim: int, n_positions: int, theta: float, device="cuda", llama3: Optional[dict] = None) -> Tuple:
    """(cos, sin) tables [n_positions, head_dim / 2] f32 on `device`, as the
    model forwards build theirs (model/quantized_llama_local.rs:189-205, the
    Llama-3.1 frequency scaling of model/llama_local.rs:47-75): angles are f32
    products.  llama3: {"factor", "low_freq_factor", "high_freq_factor",
    "original_max_position_embeddings"}."""
    import torch
    i = np.arange(0, head_dim, 2, dtype=np.float32)
    inv = (np.float32(1.0) / np.power(np.float32(theta), i / np.float32(head_dim))).astype(np.float32)
    if llama3:
        factor, low, high = (float(llama3[k]) for k in ("factor", "low_freq_factor", "high_freq_factor"))
        orig = float(llama3["original_max_position_embeddings"])
        wave = 2.0 * math.pi / inv
        smooth = (orig / wave - low) / (high - low)
        mixed = (1.0 - smooth) * inv / factor + smooth * inv
        inv = np.where(wave < orig / high, inv, np.where(wave > orig / low, inv / factor, mixed)).astype(np.float32)
    angle = np.arange(n_positions, dtype=np.float32)[:, None] * inv[None]
    return (torch.from_numpy(np.cos(angle)).to(device), torch.from_numpy(np.sin(angle)).to(device))


class KV4Cache:
    """A pool of 4-bit pages for all layers (spec_kv4_create).

    pool: contiguous uint8 CUDA tensor of at least pool_bytes(...) bytes, kept
    as it is.  rope: (cos, sin) f32 tensors [n_positions, head_dim / 2], or
    None for rows that need no rotation."""

    def __init__(self, pool, *, n_layers: int, n_heads: int, n_kv_heads: int, head_dim: int, page_tokens: int,
                 n_pages: int, rope: Optional[Tuple] = None, rope_half: bool = True):
        import torch
        self._lib = _lib.load()
        self._h = None
        if not (isinstance(pool, torch.Tensor) and pool.is_cuda and pool.is_contiguous()):
            raise _invalid("pool is not a contiguous CUDA tensor")
        self.device = pool.device
        self.n_layers, self.n_heads, self.n_kv_heads = int(n_layers), int(n_heads), int(n_kv_heads)
        self.head_dim, self.page_tokens, self.n_pages = int(head_dim), int(page_tokens), int(n_pages)
        d = self._desc(pool.device.index, n_layers, n_heads, n_kv_heads, head_dim, page_tokens, n_pages, rope_half)
        cos = sin = None
        if rope is not None:
            cos, sin = rope
            for t in (cos, sin):
                if not (t.device == pool.device and t.dtype == torch.float32 and t.is_contiguous() and t.dim() == 2 and
                        t.shape[1] * 2 == head_dim and t.shape == cos.shape):
                    raise _invalid("rope is not a pair of contiguous f32 tensors [n_positions, head_dim / 2] on the "
                                   "pool's device")
        h = ctypes.c_void_p()
        _lib.check(self._lib.spec_kv4_create(ctypes.byref(d), pool.data_ptr(), pool.numel() * pool.element_size(),
                                             cos.data_ptr() if cos is not None else None,
                                             sin.data_ptr() if sin is not None else None,
                                             cos.shape[0] if cos is not None else 0, ctypes.byref(h)))
        self._h = h
        self._keep = (pool, cos, sin)

    @staticmethod
    def _desc(device, n_layers, n_heads, n_kv_heads, head_dim, page_tokens, n_pages, rope_half) -> _lib.KV4Desc:
        return _lib.KV4Desc(int(device), int(n_layers), int(n_heads), int(n_kv_heads), int(head_dim),
                            int(page_tokens), int(n_pages), 1 if rope_half else 0)

    @staticmethod
    def pool_bytes(*, n_layers: int, n_kv_heads: int, head_dim: int, page_tokens: int, n_pages: int) -> int:
        d = KV4Cache._desc(0, n_layers, n_kv_heads, n_kv_heads, head_dim, page_tokens, n_pages, True)
        n = int(_lib.load().spec_kv4_pool_bytes(ctypes.byref(d)))
        if n < 0:
            _lib.check(-n)
        return n

    def close(self) -> None:
        if self._h:
            self._lib.spec_kv4_free(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class KV4Batch:
    """One step's plan over a KV4Cache, and its appends and attentions (spec_kv4_batch)."""

    def __init__(self, cache: KV4Cache):
        import torch
        self._torch = torch
        self._lib = _lib.load()
        self._h = None
        self.cache = cache
        if not cache._h:
            raise _invalid("the cache is closed")
        h = ctypes.c_void_p()
        _lib.check(self._lib.spec_kv4_batch_create(cache._h, ctypes.byref(h)))
        self._h = h
        self.n_rows = 0
        self._types = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
        # One buffer of spec_kv4_rows structures, packed at once (the host's part
        # of a call takes longer than a small one's kernel).
        size = ctypes.sizeof(_lib.KV4Rows)
        self._buf = ctypes.create_string_buffer(6 * size)
        self._at = [ctypes.addressof(self._buf) + i * size for i in range(6)]
        self._dim = cache.head_dim
        self._index = cache.device.index
        self._scale = cache.head_dim ** -0.5
        # The raw handle of torch's current stream, without a Stream object around it.
        raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)
        if raw is not None:
            index = self._index  # not self: the batch would hold itself
            self._stream = lambda: raw(index)

    def plan(self, kv_len: Sequence[int], n_rows: Sequence[int], page_table, positions=None, masks=None,
             src_rows=None) -> None:
        """One step: sequence b holds kv_len[b] tokens and brings n_rows[b]
        rows; page_table[b] lists its pages (rows may differ in length).
        positions, masks (ancestor bits, see DraftTree.ancestor_bits) and
        src_rows are per row, sequence by sequence."""
        kv = _host(kv_len, np.int32, "kv_len")
        m = _host(n_rows, np.int32, "n_rows", kv.size)
        if len(page_table) != kv.size:
            raise _invalid(f"page_table has {len(page_table)} rows, {kv.size} are needed")
        if isinstance(page_table, np.ndarray) and page_table.ndim == 2 and page_table.shape[1]:
            stride, flat = page_table.shape[1], _host(page_table, np.int32, "page_table")
        else:
            sizes = [len(t) for t in page_table]
            stride = max(sizes, default=1)
            flat = np.full((kv.size, max(stride, 1)), -1, dtype=np.int32)
            try:  # lists, the usual form, in one go
                pages = array.array("i")
                for t in page_table:
                    pages.fromlist(t)
            except (OverflowError, TypeError):
                pages = np.concatenate([_host(t, np.int32, "page_table", len(t)) for t in page_table])
            flat[np.arange(flat.shape[1]) < np.array(sizes, np.int64)[:, None]] = pages
        total = int(m.sum()) if (m >= 0).all() else None
        pos = None if positions is None else _host(positions, np.int32, "positions", total)
        msk = None if masks is None else _host(masks, np.uint64, "masks", total)
        src = None if src_rows is None else _host(src_rows, np.int32, "src_rows", total)
        step = _lib.KV4Step(kv.size, max(int(stride), 1), kv.ctypes.data, m.ctypes.data, flat.ctypes.data,
                            pos.ctypes.data if pos is not None else None, msk.ctypes.data if msk is not None else None,
                            src.ctypes.data if src is not None else None)
        _lib.check(self._lib.spec_kv4_plan(self._h, ctypes.byref(step), self._stream()))
        self.n_rows = total

    def _stream(self) -> int:
        return self._torch.cuda.current_stream(self._index).cuda_stream

    def _rows(self, t, heads: int, what: str):
        """The fields of spec_kv4_rows for tensor t [rows, heads, head_dim]."""
        if t is None:
            return _NONE
        try:
            n, h, d = t.shape
            row, head, ch = t.stride()
            kind = self._types[t.dtype]
        except ValueError:
            h = d = ch = None
        except KeyError:
            raise _invalid(f"{what} is {t.dtype}: bfloat16, float16 and float32 are taken") from None
        if h != heads or d != self._dim:
            raise _invalid(f"{what} has shape {tuple(t.shape)}, [rows, {heads}, {self._dim}] is needed")
        if ch != 1:
            raise _invalid(f"the channels of {what} are not contiguous")
        if t.get_device() != self._index:
            raise _invalid(f"{what} is on {t.device}, the pool on {self.cache.device}")
        return t.data_ptr(), row, head, n, kind, 0

    def append(self, layer: int, q, k, v, q_out=None, k_out=None, v_out=None):
        """Stores the plan's rows of k and v in `layer`'s pages, k rotated, and
        rotates q (None: no queries) into q_out (None: a new tensor of q's
        type).  k_out / v_out: optional float16 tensors for the stored values.
        Returns q_out."""
        c = self.cache
        if q is not None and q_out is None:
            q_out = self._torch.empty((self.n_rows, c.n_heads, c.head_dim), dtype=q.dtype, device=c.device)
        rows, nq, nk, at = self._rows, c.n_heads, c.n_kv_heads, self._at
        _SIX_ROWS.pack_into(self._buf, 0, *rows(q, nq, "q"), *rows(q_out, nq, "q_out"), *rows(k, nk, "k"),
                            *rows(v, nk, "v"), *rows(k_out, nk, "k_out"), *rows(v_out, nk, "v_out"))
        rc = self._lib.spec_kv4_append(self._h, layer, at[0] if q is not None else None,
                                       at[1] if q_out is not None else None, at[2] if k is not None else None,
                                       at[3] if v is not None else None, at[4] if k_out is not None else None,
                                       at[5] if v_out is not None else None, self._stream())
        if rc:
            _lib.check(rc)
        return q_out

    def attend(self, layer: int, q, out=None, scale: Optional[float] = None):
        """Attention of the plan's rows over `layer`: q [rows, n_heads,
        head_dim] rotated queries; returns out (None: a new tensor of q's
        type).  scale: 1 / sqrt(head_dim) when None."""
        c = self.cache
        if out is None:
            out = self._torch.empty((self.n_rows, c.n_heads, c.head_dim), dtype=q.dtype, device=c.device)
        _TWO_ROWS.pack_into(self._buf, 0, *self._rows(q, c.n_heads, "q"), *self._rows(out, c.n_heads, "out"))
        rc = self._lib.spec_kv4_attend(self._h, layer, self._at[0], self._at[1],
                                       self._scale if scale is None else scale, self._stream())
        if rc:
            _lib.check(rc)
        return out

    def status(self) -> None:
        """Waits for this batch's calls; raises if a device wait in one of them gave up."""
        _lib.check(self._lib.spec_kv4_status(self._h))

    def close(self) -> None:
        if self._h:
            self._lib.spec_kv4_batch_free(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass
