"""Host-side checks of the paged 8-bit KV cache and the packed attention: sizes, refusals that need no device."""
import ctypes

import pytest


def _cfg(native, **kw):
    c = dict(code=0, n_kv_heads=8, head_dim=64, page_size=64, n_pages=10, rope=0, rope_dim=0, original_max_pos=8192,
             rope_theta=1e4, rope_factor=0.0, low_freq_factor=1.0, high_freq_factor=4.0)
    c.update(kw)
    return native.KV8Config(**c)


@pytest.mark.parametrize("nkv,hd,page,n", [(1, 32, 16, 1), (8, 64, 64, 10), (3, 96, 32, 7), (8, 128, 128, 100000), (2, 256, 16, 3)])
def test_pool_bytes(native, nkv, hd, page, n):
    c = _cfg(native, n_kv_heads=nkv, head_dim=hd, page_size=page, n_pages=n)
    assert native.lib().pb_kv8_pool_bytes(ctypes.byref(c)) == n * nkv * (page // 16) * (32 * hd + 16)


@pytest.mark.parametrize("bad", [dict(code=2), dict(code=-1), dict(n_kv_heads=0), dict(n_kv_heads=2000), dict(head_dim=0),
                                 dict(head_dim=48), dict(head_dim=288), dict(page_size=8), dict(page_size=48),
                                 dict(page_size=256), dict(n_pages=0), dict(rope=3), dict(rope=1, rope_dim=0),
                                 dict(rope=2, rope_dim=33), dict(rope=1, rope_dim=66)])
def test_bad_configurations(native, bad):
    c = _cfg(native, **bad)
    assert native.lib().pb_kv8_pool_bytes(ctypes.byref(c)) == -1


def test_null_handles(native):
    L = native.lib()
    c = _cfg(native)
    out = ctypes.c_void_p()
    assert L.pb_kv8_pool_bytes(None) == -1
    assert L.pb_kv8_create(None, ctypes.byref(c), ctypes.byref(out)) == native.PB_ERR_ARG
    assert L.pb_kv8_free(None) == native.PB_OK
    assert L.pb_kv8_append(None, None, 0, None, 0, None, 0, None, 0, 0, None, None, None, 0, 0, 0, 0, None, 0, None, 0,
                           None, 0) == native.PB_ERR_ARG
    assert L.pb_kv8_read(None, None, None, None, None, 0, 0, 0, 0, None, 0, None, 0) == native.PB_ERR_ARG
    assert L.pb_kv8_attn(None, None, 0, None, 0, 0, None, None, None, 0, 0, 0, 1.0, None, 0) == native.PB_ERR_ARG
    assert L.pb_attn_packed(None, 1, None, 0, None, 0, None, 0, None, None, 0, 0, 0, 1, 1, 64, 1.0, 1, None,
                            0) == native.PB_ERR_ARG
