"""4-bit paged KV cache, what needs no GPU: sizes, refusals of descriptions, the layout's restatement."""

import ctypes

import numpy as np
import pytest

import kv4_ref as ref


@pytest.mark.parametrize("p", [16, 32, 64, 128])
@pytest.mark.parametrize("d", [64, 128])
def test_every_byte_of_a_block_has_one_owner(p, d):
    """Codes of all tokens and channels and all scales fill the block without overlap."""
    owner = np.zeros(ref.block_bytes(p, d), int)
    for value in (False, True):
        for j in range(p):
            for ch in range(0, d, 2):
                owner[ref.code_address(p, d, j, ch, value)] += 1
            for g in range(d // 32):
                at = ref.scale_address(p, d, j, g, value)
                owner[at:at + 4] += 1
    assert (owner == 1).all()


def test_quantize_bounds_the_error():
    rng = np.random.default_rng(0)
    x = rng.standard_normal(128).astype(np.float32) * 3
    codes, so, val = ref.quantize(x)
    s = so[:, 0].astype(np.float64).repeat(32)
    o = np.abs(so[:, 1].astype(np.float64)).repeat(32)
    assert (np.abs(val - x) <= s / 32 + (s + o) * 2.0 ** -11 + 1e-5).all()
    assert codes.max() <= 15


def test_pool_bytes_and_refused_descriptions(pkg):
    ok = dict(n_layers=3, n_kv_heads=8, head_dim=128, page_tokens=64, n_pages=10)
    assert pkg.KV4Cache.pool_bytes(**ok) == 3 * 10 * 8 * 64 * 160
    for change, error in ((dict(head_dim=96), pkg.UnsupportedMethodError), (dict(page_tokens=48), pkg.UnsupportedMethodError),
                          (dict(n_pages=0), pkg.SamplingError), (dict(n_kv_heads=0), pkg.SamplingError),
                          (dict(n_layers=2 ** 30, n_pages=2 ** 30, n_kv_heads=1024), pkg.SamplingError)):
        with pytest.raises(error):
            pkg.KV4Cache.pool_bytes(**{**ok, **change})


def test_null_arguments_are_refused(pkg):
    from importlib import import_module
    lib = import_module("abyo-speculate_b200._lib").load()
    out = ctypes.c_void_p()
    assert lib.spec_kv4_create(None, None, 0, None, None, 0, ctypes.byref(out)) == 1
    assert lib.spec_kv4_batch_create(None, ctypes.byref(out)) == 1
    assert lib.spec_kv4_plan(None, None, None) == 1
    assert lib.spec_kv4_append(None, 0, None, None, None, None, None, None, None) == 1
    assert lib.spec_kv4_attend(None, 0, None, None, 1.0, None) == 1
    assert lib.spec_kv4_status(None) == 1
    assert b"null" in lib.spec_last_error(None)
    lib.spec_kv4_free(None)
    lib.spec_kv4_batch_free(None)


def test_rope_tables(pkg):
    cos, sin = pkg.rope_tables(64, 50, 1e4, device="cpu")
    i = np.arange(0, 64, 2)
    angle = np.arange(50)[:, None] / 1e4 ** (i / 64)
    assert np.abs(cos.numpy() - np.cos(angle)).max() < 1e-5 and np.abs(sin.numpy() - np.sin(angle)).max() < 1e-5
    scaled, _ = pkg.rope_tables(64, 9000, 5e5, device="cpu", llama3={
        "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0, "original_max_position_embeddings": 8192})
    slow = 8999 / 5e5 ** (62 / 64)  # a wavelength past 8192: its frequency is divided by 8
    assert abs(float(scaled[8999, 31]) - np.cos(slow / 8)) < 1e-4
