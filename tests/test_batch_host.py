"""Sampling and verification of a batch, what needs no GPU: workspace sizes and refusals, which come before any CUDA call."""

import ctypes

import pytest


@pytest.fixture(scope="module")
def lib():
    from importlib import import_module
    return import_module("abyo-speculate_b200._lib").load()


def logits(**change):
    from importlib import import_module
    _lib = import_module("abyo-speculate_b200._lib")
    need = _lib.load().spec_batch_workspace_bytes(4, 1000, 0)
    d = dict(device=0, vocab=1000, dtype=0, temperature=1.0, logits=1 << 20, row_stride=1000, n_rows=4, temperatures=None,
             uniforms=1 << 20, workspace=1 << 20, workspace_bytes=need)
    d.update(change)
    return _lib.BatchLogits(**d)


def test_workspace_bytes(lib):
    assert lib.spec_batch_workspace_bytes(0, 1000, 2) == 0
    # 16 bytes a chunk of 512 columns (of which up to 7 lie before the row), a multiple of 8 chunks, and 8 a row.
    for n, v, dtype, chunks in ((1, 1, 0, 8), (3, 4090, 0, 16), (3, 4089, 0, 8), (3, 4094, 2, 16), (64, 128256, 2, 256)):
        size = lib.spec_batch_workspace_bytes(n, v, dtype)
        assert n * (16 * chunks + 8) <= size < n * (16 * chunks + 8) + 3 * 256
    for bad in ((-1, 10, 0), (1 << 21, 10, 0), (1, 0, 0), (1, (1 << 20) + 1, 0), (1, 10, 3), (1, 10, -1)):
        assert lib.spec_batch_workspace_bytes(*bad) == -1


BAD = [dict(vocab=0), dict(dtype=3), dict(n_rows=-1), dict(logits=None), dict(uniforms=None), dict(workspace=None),
       dict(logits=(1 << 20) + 1), dict(uniforms=(1 << 20) + 2), dict(temperatures=(1 << 20) + 1), dict(row_stride=-1),
       dict(row_stride=1 << 41), dict(temperature=-1.0), dict(temperature=float("nan")), dict(temperature=float("inf")),
       dict(workspace=(1 << 20) + 8), dict(workspace_bytes=16), dict(device=-1)]


@pytest.mark.parametrize("change", BAD, ids=lambda c: "%s=%s" % next(iter(c.items())))
def test_bad_logits_are_refused(lib, change):
    a = logits(**change)
    p = 1 << 20
    assert lib.spec_batch_sample(ctypes.byref(a), None, 0, p, None) == 1
    assert lib.spec_batch_verify(ctypes.byref(a), 1, p, p, p, 1000, p, p, None) == 1
    assert lib.spec_batch_verify_tree(ctypes.byref(a), 1, p, p, p, p, p, p, None) == 1
    assert b"spec_batch" in lib.spec_last_error(None)


def test_other_bad_arguments_are_refused(lib):
    a, p = logits(), 1 << 20
    assert lib.spec_batch_sample(None, None, 0, p, None) == 1
    assert lib.spec_batch_sample(ctypes.byref(a), None, 0, None, None) == 1
    assert lib.spec_batch_sample(ctypes.byref(a), None, 0, p + 2, None) == 1
    assert lib.spec_batch_sample(ctypes.byref(a), p, 999, p, None) == 1  # rows of probabilities overlap
    assert lib.spec_batch_sample(ctypes.byref(a), p, 1 << 41, p, None) == 1
    assert lib.spec_batch_sample(ctypes.byref(a), p + 1, 1000, p, None) == 1
    for at in range(1, 5):
        args = [p, p, p, 1000, p, p]
        args[at if at < 3 else at + 1] = None
        assert lib.spec_batch_verify(ctypes.byref(a), 1, *args, None) == 1
        args[at if at < 3 else at + 1] = p + 1
        assert lib.spec_batch_verify(ctypes.byref(a), 1, *args, None) == 1
    assert lib.spec_batch_verify(ctypes.byref(a), 1, p, p, p, -1, p, p, None) == 1
    assert lib.spec_batch_verify(ctypes.byref(a), -1, p, p, p, 1000, p, p, None) == 1
    assert lib.spec_batch_verify(ctypes.byref(a), 1 << 21, p, p, p, 1000, p, p, None) == 1
    for at in range(6):
        args = [p] * 6
        args[at] = None
        assert lib.spec_batch_verify_tree(ctypes.byref(a), 1, *args, None) == 1
        args[at] = p + 1
        assert lib.spec_batch_verify_tree(ctypes.byref(a), 1, *args, None) == 1


def test_nothing_to_do_needs_no_device(lib):
    a = logits(n_rows=0, logits=None, uniforms=None, workspace=None, workspace_bytes=0)
    assert lib.spec_batch_sample(ctypes.byref(a), None, 0, None, None) == 0
    assert lib.spec_batch_verify(ctypes.byref(a), 0, None, None, None, 0, None, None, None) == 0
    assert lib.spec_batch_verify_tree(ctypes.byref(a), 0, None, None, None, None, None, None, None) == 0


def test_python_refuses_host_tensors(pkg):
    import torch
    x, u = torch.zeros(2, 8), torch.zeros(2)
    with pytest.raises(pkg.SamplingError):
        pkg.sample_rows(x, u)
    with pytest.raises(pkg.SamplingError):
        pkg.verify_drafts(x, u, x, u, u)
    with pytest.raises(pkg.SamplingError):
        pkg.verify_trees(x, u, u, u, u)


def test_a_tree_call_without_sequences_needs_its_path(lib):
    """Rows but no sequence: every row's path is to be -1, so that there has to be one."""
    a, p = logits(), 1 << 20
    assert lib.spec_batch_verify_tree(ctypes.byref(a), 0, None, None, None, None, None, None, None) == 1
    assert lib.spec_batch_verify_tree(ctypes.byref(a), 0, None, None, None, p + 2, None, None, None) == 1


@pytest.mark.parametrize("probs,stride", [(1 << 20, 1000), ((1 << 20) + 4 * 1000 * 3, 1000), ((1 << 20) - 4, 1000), ((1 << 20) - 4000 * 3, 1001)])
def test_probabilities_on_the_logits_are_refused(lib, probs, stride):
    a = logits(dtype=2, workspace_bytes=1 << 20)
    assert lib.spec_batch_sample(ctypes.byref(a), probs, stride, 1 << 26, None) == 1
    assert b"share memory" in lib.spec_last_error(None)


def test_one_row_of_probabilities_on_its_logits(lib):
    """A single row's stride does not count, whatever it is."""
    for stride in (-7, 0, 5):
        a = logits(dtype=2, n_rows=1, workspace_bytes=1 << 20)
        assert lib.spec_batch_sample(ctypes.byref(a), (1 << 20) + 3996, stride, 1 << 26, None) == 1
        assert b"share memory" in lib.spec_last_error(None)
