"""Host side of the key/value cache and rotary positions: configuration checks
and frequencies (no GPU), and the 64-bit restatement's own properties."""
from __future__ import annotations

import ctypes as C
import math

import numpy as np
import pytest

from oracle import kv_cache as ref
from vicinity_b200 import KVCache, Rotary, _lib


@pytest.mark.parametrize("kw,match", [
    (dict(dim=3), "even"), (dict(dim=258), "even"), (dict(dim=0), "even"), (dict(dim=8, base=1.0), "base"),
    (dict(dim=8, base=math.inf), "base"), (dict(dim=8, layout="x"), "layout"), (dict(dim=8, scaling="x"), "scaling"),
    (dict(dim=8, scaling="linear", factor=0.5), "factor"), (dict(dim=8, scaling="linear", factor=math.nan), "factor"),
    (dict(dim=8, scaling="by_parts", factor=2.0), "original_length"),
    (dict(dim=8, scaling="by_parts", factor=2.0, original_length=100.0, low_turns=4.0, high_turns=4.0), "low_turns"),
    (dict(dim=8, magnitude=0.0), "magnitude"), (dict(dim=-2), "greater than 0"),
])
def test_rotary_refuses(kw, match):
    with pytest.raises(ValueError, match=match):
        Rotary(**kw)


@pytest.mark.parametrize("dim,kw", [
    (2, {}), (64, {}), (256, dict(base=500.0)), (128, dict(scaling="linear", factor=4.0)),
    (128, dict(scaling="by_parts", factor=8.0, original_length=4096.0)),
    (96, dict(scaling="by_parts", factor=2.0, original_length=100.0, low_turns=0.0, high_turns=3.0)),
])
def test_rotary_frequencies(dim, kw):
    assert np.allclose(Rotary(dim, **kw).frequencies(), ref.rotary_frequencies(dim, **kw), rtol=1e-14, atol=0)


@pytest.mark.parametrize("change", [
    dict(num_seqs=0), dict(capacity=0), dict(capacity=(1 << 30) + 1), dict(num_kv_heads=0), dict(num_kv_heads=65536),
    dict(head_dim=0), dict(head_dim=48), dict(head_dim=256), dict(block_tokens=8), dict(block_tokens=48),
    dict(num_seqs=1 << 40),
])
def test_create_refuses_before_touching_a_device(change):
    p = dict(num_seqs=2, capacity=64, num_kv_heads=2, head_dim=64, block_tokens=64)
    p.update(change)
    h = C.c_void_p()
    assert _lib.load().vg_kv_create(C.byref(_lib.VgKvParams(**p)), 0, C.byref(h)) == _lib.VG_ERR_INVALID_CONFIG
    assert not h.value and _lib.last_error()


def test_null_arguments_are_refused():
    lib = _lib.load()
    bad = _lib.VG_ERR_INVALID_PARAMETER
    h = C.c_void_p()
    assert lib.vg_kv_create(None, 0, C.byref(h)) == bad and lib.vg_rotary_create(None, C.byref(h)) == bad
    assert lib.vg_kv_append(None, None, 0, None, None, None) == bad
    assert lib.vg_kv_attend(None, None, 1, None, None, None, 1.0, 0, None) == bad
    assert lib.vg_kv_evict(None, 0, None, None, 1, 0, None, None) == bad
    assert lib.vg_kv_read(None, None, None, 0, None, None, None) == bad
    assert lib.vg_kv_load(None, 0, 0, None, None, None, None, None, None) == bad
    assert lib.vg_kv_export(None, 0, None, None, None, None, None, None) == bad
    assert lib.vg_kv_truncate(None, None) == bad and lib.vg_kv_lengths(None, None) == bad
    assert lib.vg_kv_destroy(None) == _lib.VG_OK and lib.vg_rotary_destroy(None) == _lib.VG_OK


def test_create_without_a_device_fails_loudly():
    if _lib.device_count() > 0:
        pytest.skip("a device is present")
    with pytest.raises(_lib.VicinityError, match="no CPU path"):
        KVCache(2, 64, 2, 64)


def test_reference_scale_is_the_smallest_power_of_two():
    g = np.random.default_rng(1)
    for x in list(np.exp(g.uniform(-60, 60, 500))) + [127.0, 127.0 * (1 + 2.0 ** -30), 128.0, 1.0, 2.0 ** -90]:
        s = ref.block_scale(np.array([x]))
        assert 127 * s >= x and 127 * s / 2 < x
    assert ref.block_scale(np.zeros(3)) == 2.0 ** -100


def test_reference_attention_of_equal_scores_is_the_mean():
    v = np.arange(12.0).reshape(6, 2)
    out, lse, w, _, _ = ref.attention(np.zeros((2, 1, 2)), np.ones((6, 2)), v, 2, 1.0)
    assert np.allclose(out[0, 0], v[:5].mean(0)) and np.allclose(out[1, 0], v.mean(0))
    assert np.allclose(lse[:, 0], np.log([5, 6])) and np.allclose(w.sum(), 2.0)
