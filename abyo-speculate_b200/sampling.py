"""Sampling and verification of a batch over torch tensors: the host side of spec_batch_* (include/spec_b200.h).

    token = sample_rows(draft_logits, u, temperature, probs_out=q[:, i])      # a draft step
    n, token = verify_drafts(logits, drafts, q, u, row_start, temperature)    # chains
    path, n, token = verify_trees(logits, tokens, parents, u, row_start, temperature)

Calls are queued on torch's current stream of the logits' device and return
without waiting for it; results are new int32 tensors on that device.  Decisions
are those of 64-bit arithmetic on the given logits, probabilities and uniforms.
"""

from __future__ import annotations

import ctypes
from typing import Tuple

from . import _lib


def _invalid(msg: str) -> _lib.SamplingError:
    return _lib.SamplingError(_lib.SPEC_ERR_INVALID, msg)


def _on(t, what: str, device, dtype, shape=None):
    """Data pointer of a contiguous tensor of `dtype` on `device`."""
    import torch
    if not isinstance(t, torch.Tensor):
        raise _invalid(f"{what} is not a tensor")
    if t.device != device:
        raise _invalid(f"{what} is on {t.device}, the logits on {device}")
    if t.dtype != dtype:
        raise _invalid(f"{what} is {t.dtype}, {dtype} is needed")
    if shape is not None and tuple(t.shape) != shape:
        raise _invalid(f"{what} has shape {tuple(t.shape)}, {shape} is needed")
    if not t.is_contiguous():
        raise _invalid(f"{what} is not contiguous")
    return t.data_ptr()


def _rows_of(t, what: str, device, dtype, n: int, v: int):
    """Data pointer and row stride of a tensor [n, v] whose columns are contiguous."""
    import torch
    if not isinstance(t, torch.Tensor) or t.device != device or t.dtype != dtype:
        raise _invalid(f"{what} is not a {dtype} tensor on {device}")
    if tuple(t.shape) != (n, v):
        raise _invalid(f"{what} has shape {tuple(t.shape)}, {(n, v)} is needed")
    if v > 1 and t.stride(1) != 1:
        raise _invalid(f"the columns of {what} are not contiguous")
    return t.data_ptr(), t.stride(0)


def _logits(logits, uniforms, temperature):
    """spec_batch_logits of a call, and what has to live until it is queued."""
    import torch
    types = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
    if not (isinstance(logits, torch.Tensor) and logits.is_cuda):
        raise _invalid("logits are not a CUDA tensor")
    if logits.dim() != 2:
        raise _invalid(f"logits have shape {tuple(logits.shape)}, [rows, vocabulary] is needed")
    if logits.dtype not in types:
        raise _invalid(f"logits are {logits.dtype}: bfloat16, float16 and float32 are taken")
    n, v = logits.shape
    device = logits.device
    ptr, stride = _rows_of(logits, "logits", device, logits.dtype, n, v)
    u = _on(uniforms, "uniforms", device, torch.float32, (n,))
    temps, temp = None, 0.0
    if isinstance(temperature, torch.Tensor):
        temps = _on(temperature, "temperature", device, torch.float32, (n,))
    else:
        temp = float(temperature)
    kind = types[logits.dtype]
    size = _lib.load().spec_batch_workspace_bytes(n, v, kind)
    if size < 0:
        _lib.check(-size)
    work = torch.empty(size, dtype=torch.uint8, device=device)
    return _lib.BatchLogits(device.index, v, kind, temp, ptr, stride, n, temps, u, work.data_ptr(), size), work


def _stream(device) -> int:
    import torch
    return torch.cuda.current_stream(device).cuda_stream


def sample_rows(logits, uniforms, temperature=1.0, probs_out=None, tokens_out=None):
    """A token per row of logits [rows, vocabulary] (spec_batch_sample), int32.

    uniforms: float32 [rows]; temperature: a number, or float32 [rows] (0: the
    first largest logit).  probs_out: float32 [rows, vocabulary] for the rows'
    probabilities; tokens_out: contiguous int32 [rows]."""
    import torch
    a, work = _logits(logits, uniforms, temperature)
    n, v = logits.shape
    if tokens_out is None:
        tokens_out = torch.empty(n, dtype=torch.int32, device=logits.device)
    else:
        _on(tokens_out, "tokens_out", logits.device, torch.int32, (n,))
    probs, stride = (None, 0) if probs_out is None else _rows_of(probs_out, "probs_out", logits.device, torch.float32, n, v)
    _lib.check(_lib.load().spec_batch_sample(ctypes.byref(a), probs, stride, tokens_out.data_ptr(), _stream(logits.device)))
    return tokens_out


def verify_drafts(logits, drafts, draft_probs, uniforms, row_start, temperature=1.0) -> Tuple:
    """Accepts drafted chains (spec_batch_verify): (n_accepted, next_token), int32 [sequences].

    Sequence b has rows row_start[b] .. row_start[b + 1] - 1 (int32, on the
    device), one more than its drafts.  drafts: int32 [rows], drafts[r] is the
    token that row r judges, drawn from row r of draft_probs (float32 [rows,
    vocabulary]); those of a sequence's last row are not read.  uniforms: float32
    [rows]; temperature: a number, or float32 [rows]."""
    import torch
    a, work = _logits(logits, uniforms, temperature)
    n, v = logits.shape
    start = _on(row_start, "row_start", logits.device, torch.int32)
    if row_start.dim() != 1 or row_start.numel() < 1:
        raise _invalid(f"row_start has shape {tuple(row_start.shape)}, [sequences + 1] is needed")
    d = _on(drafts, "drafts", logits.device, torch.int32, (n,))
    q, stride = _rows_of(draft_probs, "draft_probs", logits.device, torch.float32, n, v)
    out = torch.empty(2, row_start.numel() - 1, dtype=torch.int32, device=logits.device)
    count, token = out[0], out[1]
    _lib.check(_lib.load().spec_batch_verify(ctypes.byref(a), row_start.numel() - 1, start, d, q, stride, count.data_ptr(),
                                             token.data_ptr(), _stream(logits.device)))
    return count, token


def verify_trees(logits, tokens, parents, uniforms, row_start, temperature=1.0) -> Tuple:
    """Walks draft trees whose candidates were picked, not drawn (spec_batch_verify_tree): (path, path_len, next_token).

    Node i of sequence b is row row_start[b] + i; tokens and parents: int32
    [rows] (parents within the sequence, node 0 the root).  path: int32 [rows],
    a sequence's accepted nodes from its first row on, root first, -1 in all
    other rows; path_len and next_token: int32 [sequences]."""
    import torch
    a, work = _logits(logits, uniforms, temperature)
    n = logits.shape[0]
    start = _on(row_start, "row_start", logits.device, torch.int32)
    if row_start.dim() != 1 or row_start.numel() < 1:
        raise _invalid(f"row_start has shape {tuple(row_start.shape)}, [sequences + 1] is needed")
    t = _on(tokens, "tokens", logits.device, torch.int32, (n,))
    up = _on(parents, "parents", logits.device, torch.int32, (n,))
    path = torch.empty(n, dtype=torch.int32, device=logits.device)
    out = torch.empty(2, row_start.numel() - 1, dtype=torch.int32, device=logits.device)
    count, token = out[0], out[1]
    _lib.check(_lib.load().spec_batch_verify_tree(ctypes.byref(a), row_start.numel() - 1, start, t, up, path.data_ptr(),
                                                  count.data_ptr(), token.data_ptr(), _stream(logits.device)))
    return path, count, token
