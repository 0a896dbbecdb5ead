"""What the operators' entry points refuse before they need a device."""
import ctypes as C

import numpy as np
import pytest

import cortexsdr_b200 as cs
from cortexsdr_b200 import _lib
from tests import operator_refs as ref


def test_null_handles_are_refused(lib):
    b = cs.KVBatch(1, 1, 0, 0, 0, 1)
    out = C.c_void_p()
    assert lib.csdr_kv_cache_create(None, 1, 1, 16, 1, 64, 1e4, C.byref(out)) == _lib.ERR_INVALID_ARG
    assert lib.csdr_kv_cache_append_device_async(None, 0, b._ref, None, None, 0, 0, 0, None, 0, 0, None, 0) == _lib.ERR_INVALID_ARG
    assert lib.csdr_kv_cache_read_device_async(None, 0, b._ref, None, None) == _lib.ERR_INVALID_ARG
    assert lib.csdr_kv_cache_attention_device_async(None, 0, b._ref, None, 0, 0, 1, 0.0, None, 0) == _lib.ERR_INVALID_ARG
    assert lib.csdr_kv_cache_bytes(None, None) == _lib.ERR_INVALID_ARG
    assert lib.csdr_q4_create(None, b"q4_0", None, 18, 1, 32, C.byref(out)) == _lib.ERR_INVALID_ARG
    assert lib.csdr_q4_matmul_device_async(None, None, None, 0, 1, 1, None, 1, None) == _lib.ERR_INVALID_ARG
    assert lib.csdr_token_logprobs_device_async(None, None, 0, 0, 1, 1, None, None, None, 0, None, None) == _lib.ERR_INVALID_ARG
    assert lib.csdr_decoder_score(None, 0, None, 0, None, None, None, 0, None, None) == _lib.ERR_INVALID_ARG
    assert lib.csdr_kv_cache_destroy(None) == _lib.OK and lib.csdr_q4_destroy(None) == _lib.OK
    assert out.value is None


def test_the_cache_holds_values_within_half_a_step():
    """The definition that the device is tested against: off by half a step, by the rounding of minimum and step (15 of them) and
    by nothing else; groups by themselves; what is not finite spoils its group only."""
    rng = np.random.default_rng(0)
    x = rng.normal(0, 1, (9, 2, 128)) * (1 + 20 * (rng.random((9, 2, 128)) < 0.02))
    held = ref.held(x)
    g, h = x.reshape(-1, 64), held.reshape(-1, 64)
    width = g.max(1) - g.min(1)
    # half a step; fp16 steps are off by 2^-11, minima by 2^-11, the top code saturates by at most both
    bound = width / 15 * (0.5 + 2.0 ** -11) + width * 2.0 ** -11 + np.abs(g.min(1)) * 2.0 ** -11
    assert (np.abs(g - h).max(1) <= bound).all()
    x[3, 1, 70] = np.inf
    again = ref.held(x)
    assert np.isnan(again[3, 1, 64:]).all()
    again[3, 1, 64:] = held[3, 1, 64:]
    np.testing.assert_array_equal(again, held)


@pytest.mark.parametrize("fmt", ["q4_0", "q4_k"])
def test_weights_of_the_tests_are_what_the_format_says(fmt):
    rng = np.random.default_rng(1)
    payload, dense = ref.q4_weight(rng, 3, 512, fmt)
    assert payload.reshape(-1).size == 3 * 512 // (32 if fmt == "q4_0" else 256) * (18 if fmt == "q4_0" else 144)
    assert dense.shape == (3, 512) and np.isfinite(dense).all()
