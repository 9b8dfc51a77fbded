"""The 8-bit K/V pool without a GPU: its record, the plain form the GPU tests compare
with, and the arguments its entry points refuse before they touch a device."""
import ctypes

import numpy as np
import pytest

from nitrorag_amd import _native as N
from nitrorag_amd import kv_record_bytes
from oracle import kv_q8


@pytest.mark.parametrize("hd", [4, 16, 20, 64, 96, 128, 252, 256])
def test_record_bytes(hd):
    assert kv_record_bytes(hd) == kv_q8.record_bytes(hd)


@pytest.mark.parametrize("hd", [0, 2, 66, 260, -4])
def test_record_bytes_refuses(hd):
    with pytest.raises(N.NitroError) as e:
        kv_record_bytes(hd)
    assert e.value.status == N.UNSUPPORTED


@pytest.mark.parametrize("args,status", [
    ((0, 1, 4, 64), N.INVALID_ARGUMENT), ((8, 0, 4, 64), N.INVALID_ARGUMENT), ((8, 1, 0, 64), N.INVALID_ARGUMENT),
    ((8, 1, 4, 66), N.UNSUPPORTED), ((8, 1, 4, 260), N.UNSUPPORTED), ((8, 1, 1 << 30, 64), N.UNSUPPORTED),
    ((1 << 28, 1, 1, 64), N.UNSUPPORTED)])
def test_pool_arguments(args, status):
    out = ctypes.c_void_p()
    assert N.lib().nitro_kvpool_create_q8(*args, ctypes.byref(out)) == status
    assert not out.value
    assert N.lib().nitro_kvpool_wrap_q8(ctypes.c_void_p(4096), *args, ctypes.byref(out)) == status


def test_null_and_misaligned():
    L, out = N.lib(), ctypes.c_void_p()
    assert L.nitro_kvpool_create_q8(8, 1, 4, 64, None) == N.INVALID_ARGUMENT
    assert L.nitro_kvpool_wrap_q8(None, 8, 1, 4, 64, ctypes.byref(out)) == N.INVALID_ARGUMENT
    assert L.nitro_kvpool_wrap_q8(ctypes.c_void_p(4104), 8, 1, 4, 64, ctypes.byref(out)) == N.INVALID_ARGUMENT
    assert L.nitro_kvpool_q8_data(None, ctypes.byref(out)) == N.INVALID_ARGUMENT
    assert L.nitro_kvpool_q8_record_bytes(64, None) == N.INVALID_ARGUMENT
    assert L.nitro_kv_read(None, 0, None, None, None) == N.INVALID_ARGUMENT
    assert L.nitro_kv_read_prefill(None, 0, None, None, None) == N.INVALID_ARGUMENT


def test_plain_form_places_every_byte():
    """Every code and scale of a full page lies in its own bytes, and values() finds it."""
    hd, heads = 20, 2
    cache = kv_q8.Cache(np.full((3, 2, heads, kv_q8.record_bytes(hd)), 0xAA, np.uint8), hd)
    rng = np.random.default_rng(0)
    k, v = (rng.standard_normal((16, heads, hd)).astype(np.float32) for _ in range(2))
    cache.put(1, 2 * 16 + np.arange(16), k, v)
    assert (cache.data[:2] == 0xAA).all() and (cache.data[2, 0] == 0xAA).all()
    got_k, got_v = cache.values(1, [2], 16)
    for got, want in ((got_k, k), (got_v, v)):
        # half a step of the row's own scale
        assert (np.abs(got - want) <= np.abs(want).max(-1, keepdims=True) / 127 * (0.5 + 2.0 ** -15)).all()
    kc = kv_q8.quantise(k, v)[0]
    token, d = 7, 18
    assert cache.data[2, 1, 0, ((token // 4 * 2 + d // 16) * 4 + token % 4) * 16 + d % 16] == kc[token, 0, d].view(np.uint8)


def test_the_bound_counts_every_rounding():
    """It holds the sum of them: 128 weights that share a unit of the first one's, each off by
    half of it in the direction of the largest value; the integers of a score and of an output
    joined half of 256 units off; q's steps; six fp32 roundings of a score and one of exp2, for
    numerator and denominator; two for each of two tiles."""
    hd, n = 4, 128
    k, v = np.zeros((n, 1, hd)), np.ones((n, 1, hd))
    k[0] = 1
    for far in (5.0, 8.0, 12.0):
        q = np.full((1, 1, hd), far / hd * np.sqrt(hd), np.float32)  # the first score is `far`, the others 0
        bound = kv_q8.attention(q, [n - 1], k, v)[1][0, 0, 0]
        p = np.exp(-far)
        total = 1 + (n - 1) * p
        scores = 6e-8 * float(q.max()) * hd / np.sqrt(hd) + 128 / 8355000 * float(q.max()) / 127 / np.sqrt(hd)
        weights = n * 0.5 / 8355000 / total + 128 / 127 / 8355000 / total
        assert bound >= 2 * (scores + 6 * 2.0 ** -24 * far + 2.0 ** -22) + weights + 4 * 2.0 ** -24
