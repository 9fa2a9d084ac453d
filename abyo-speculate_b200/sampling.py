"""Sampling and verification of a batch over torch tensors: the host side of spec_batch_* (include/spec_b200.h).

    token = sample_rows(draft_logits, u, temperature, probs_out=q[:, i])      # a draft step
    n, token = verify_drafts(logits, drafts, q, u, row_start, temperature)    # chains
    path, n, token = verify_trees(logits, tokens, parents, u, row_start, temperature)

Calls are queued on torch's current stream of the logits' device and return
without waiting for it; results are new int32 tensors on that device.  Decisions
are those of 64-bit arithmetic on the given logits, probabilities and uniforms.
No gradients are recorded.
"""

from __future__ import annotations

import functools
import struct
from typing import Tuple

from . import _lib

_LOGITS = struct.Struct("=iiifQqqQQQq")  # spec_batch_logits (packing takes less time than a ctypes structure)


def _invalid(msg: str) -> _lib.SamplingError:
    return _lib.SamplingError(_lib.SPEC_ERR_INVALID, msg)


@functools.lru_cache(maxsize=None)
def _setup():
    """torch, the library, the element types, and torch's current stream of a device as a raw handle."""
    import torch
    raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)
    return (torch, _lib.load(), {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2},
            raw or (lambda index: torch.cuda.current_stream(index).cuda_stream))


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(n: int, v: int, kind: int) -> int:
    size = _lib.load().spec_batch_workspace_bytes(n, v, kind)
    if size < 0:
        _lib.check(-size)
    return size


def _on(t, what: str, index: int, dtype, n=None) -> int:
    """Data pointer of a contiguous one-dimensional tensor of `dtype` on device `index`, of n elements."""
    torch = _setup()[0]
    if not isinstance(t, torch.Tensor):
        raise _invalid(f"{what} is not a tensor")
    if t.get_device() != index:
        raise _invalid(f"{what} is on {t.device}, the logits on cuda:{index}")
    if t.dtype != dtype:
        raise _invalid(f"{what} is {t.dtype}, {dtype} is needed")
    if t.dim() != 1 or (n is not None and t.numel() != n):
        raise _invalid(f"{what} has shape {tuple(t.shape)}, {'[sequences + 1]' if n is None else (n,)} is needed")
    if not t.is_contiguous():
        raise _invalid(f"{what} is not contiguous")
    return t.data_ptr()


def _rows_of(t, what: str, index: int, dtype, n: int, v: int):
    """Data pointer and row stride of a tensor [n, v] whose columns are contiguous."""
    torch = _setup()[0]
    if not isinstance(t, torch.Tensor) or t.get_device() != index or t.dtype != dtype:
        raise _invalid(f"{what} is not a {dtype} tensor on cuda:{index}")
    if t.shape != (n, v):
        raise _invalid(f"{what} has shape {tuple(t.shape)}, {(n, v)} is needed")
    row, column = t.stride()
    if column != 1 and v > 1:
        raise _invalid(f"the columns of {what} are not contiguous")
    return t.data_ptr(), row


def _logits(logits, uniforms, temperature):
    """spec_batch_logits of a call, its workspace (which lives until the call is queued), and the device's index."""
    torch, _, types, _ = _setup()
    if not (isinstance(logits, torch.Tensor) and logits.is_cuda):
        raise _invalid("logits are not a CUDA tensor")
    if logits.dim() != 2:
        raise _invalid(f"logits have shape {tuple(logits.shape)}, [rows, vocabulary] is needed")
    dtype = logits.dtype
    if dtype not in types:
        raise _invalid(f"logits are {dtype}: bfloat16, float16 and float32 are taken")
    n, v = logits.shape
    index = logits.get_device()
    row, column = logits.stride()
    if column != 1 and v > 1:
        raise _invalid("the columns of logits are not contiguous")
    u = _on(uniforms, "uniforms", index, torch.float32, n)
    temps, temp = 0, 0.0
    if isinstance(temperature, torch.Tensor):
        temps = _on(temperature, "temperature", index, torch.float32, n)
    else:
        try:
            temp = float(temperature)
        except (TypeError, ValueError) as e:
            raise _invalid(f"temperature: {e}") from None
        if not 0.0 <= temp <= 3.4e38:
            raise _invalid(f"temperature {temp}")
    kind = types[dtype]
    size = _workspace_bytes(n, v, kind)
    work = logits.new_empty(size, dtype=torch.uint8)
    return _LOGITS.pack(index, v, kind, temp, logits.data_ptr(), row, n, temps, u, work.data_ptr(), size), work, index


def sample_rows(logits, uniforms, temperature=1.0, probs_out=None, tokens_out=None):
    """A token per row of logits [rows, vocabulary] (spec_batch_sample), int32.

    uniforms: float32 [rows]; temperature: a number, or float32 [rows] (0: the
    first largest logit).  probs_out: float32 [rows, vocabulary] for the rows'
    probabilities, not in the logits' memory; tokens_out: contiguous int32 [rows]."""
    torch, lib, _, stream = _setup()
    a, work, index = _logits(logits, uniforms, temperature)
    n, v = logits.shape
    if tokens_out is None:
        tokens_out = logits.new_empty(n, dtype=torch.int32)
        tokens = tokens_out.data_ptr()
    else:
        tokens = _on(tokens_out, "tokens_out", index, torch.int32, n)
    probs, row = (None, 0) if probs_out is None else _rows_of(probs_out, "probs_out", index, torch.float32, n, v)
    rc = lib.spec_batch_sample(a, probs, row, tokens, stream(index))
    if rc:
        _lib.check(rc)
    return tokens_out


def verify_drafts(logits, drafts, draft_probs, uniforms, row_start, temperature=1.0) -> Tuple:
    """Accepts drafted chains (spec_batch_verify): (n_accepted, next_token), int32 [sequences].

    Sequence b has rows row_start[b] .. row_start[b + 1] - 1 (int32, on the
    device), one more than its drafts.  drafts: int32 [rows], drafts[r] is the
    token that row r judges, drawn from row r of draft_probs (float32 [rows,
    vocabulary]); what they hold in a sequence's last row does not matter.
    uniforms: float32 [rows]; temperature: a number, or float32 [rows]."""
    torch, lib, _, stream = _setup()
    a, work, index = _logits(logits, uniforms, temperature)
    n, v = logits.shape
    start, seqs = _on(row_start, "row_start", index, torch.int32), row_start.numel() - 1
    if seqs < 0:
        raise _invalid("row_start is empty, [sequences + 1] is needed")
    d = _on(drafts, "drafts", index, torch.int32, n)
    q, row = _rows_of(draft_probs, "draft_probs", index, torch.float32, n, v)
    count, token = logits.new_empty(seqs, dtype=torch.int32), logits.new_empty(seqs, dtype=torch.int32)
    rc = lib.spec_batch_verify(a, seqs, start, d, q, row, count.data_ptr(), token.data_ptr(), stream(index))
    if rc:
        _lib.check(rc)
    return count, token


def verify_trees(logits, tokens, parents, uniforms, row_start, temperature=1.0) -> Tuple:
    """Walks draft trees whose candidates were picked, not drawn (spec_batch_verify_tree): (path, path_len, next_token).

    Node i of sequence b is row row_start[b] + i; tokens and parents: int32
    [rows] (parents within the sequence, node 0 the root).  path: int32 [rows],
    a sequence's accepted nodes from its first row on, root first, -1 in all
    other rows; path_len and next_token: int32 [sequences]."""
    torch, lib, _, stream = _setup()
    a, work, index = _logits(logits, uniforms, temperature)
    n = logits.shape[0]
    start, seqs = _on(row_start, "row_start", index, torch.int32), row_start.numel() - 1
    if seqs < 0:
        raise _invalid("row_start is empty, [sequences + 1] is needed")
    t = _on(tokens, "tokens", index, torch.int32, n)
    up = _on(parents, "parents", index, torch.int32, n)
    path, count, token = (logits.new_empty(size, dtype=torch.int32) for size in (n, seqs, seqs))
    rc = lib.spec_batch_verify_tree(a, seqs, start, t, up, path.data_ptr(), count.data_ptr(), token.data_ptr(),
                                    stream(index))
    if rc:
        _lib.check(rc)
    return path, count, token
