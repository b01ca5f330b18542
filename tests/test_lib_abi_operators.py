"""C entry points of the sampling, page, per-head norm and 8-bit operators: bad arguments are
refused, with a message, before anything touches a device.  No kernel is launched here."""

import ctypes

import pytest

from inferkernellab_b200 import _lib

OK, INVALID, LAYER = _lib.B200_OK, _lib.B200_ERR_INVALID, _lib.B200_ERR_LAYER
UNSUPPORTED, WORKSPACE = _lib.B200_ERR_UNSUPPORTED, _lib.B200_ERR_WORKSPACE
P = 4096  # a non-null address that no refused call may read


def _cache(**kw):
    return _lib.CacheDesc(**(dict(k_cache=P, v_cache=P, num_layers=1, num_blocks=4, block_size=16,
                                  num_kv_heads=2, head_dim=64, dtype=_lib.B200_BF16) | kw))


def _check(status, want, match):
    assert status == want, _lib.last_error()
    assert match in _lib.last_error()


@pytest.mark.parametrize("args,cache,want,match", [
    (dict(layer=1), {}, LAYER, "layer"),
    (dict(num_q_heads=3), {}, INVALID, "divisible"),
    (dict(rotary_dim=65), {}, INVALID, "rotary_dim"),
    (dict(rotary_dim=66), {}, INVALID, "rotary_dim"),
    (dict(eps=-1.0), {}, INVALID, "eps"),
    (dict(eps=float("nan")), {}, INVALID, "eps"),
    (dict(num_tokens=-1), {}, INVALID, "num_tokens"),
    (dict(num_tokens=2 ** 31), {}, UNSUPPORTED, "tokens"),
    ({}, dict(dtype=_lib.B200_F32), UNSUPPORTED, "float16"),
    ({}, dict(k_cache=None), INVALID, "null"),
    (dict(num_tokens=0), {}, OK, ""),
])
def test_qk_norm_rope_append(args, cache, want, match):
    a = _lib.QkNormArgs(**(dict(num_tokens=1, num_q_heads=4, layer=0, rotary_dim=64, eps=1e-6) | args))
    c = _cache(**cache)
    _check(_lib.load().b200_qk_norm_rope_append(ctypes.byref(c), ctypes.byref(a), P, P, P, P, P, P,
                                                P, P, P, None, None), want, match)


def test_pages():
    lib, c = _lib.load(), _cache()
    _check(lib.b200_copy_kv_pages(None, P, P, None, 0, 1, None, None), INVALID, "null")
    _check(lib.b200_copy_kv_pages(ctypes.byref(c), P, None, None, 0, 1, None, None), INVALID, "null")
    _check(lib.b200_copy_kv_pages(ctypes.byref(c), P, P, None, 5, 1, None, None), INVALID, "index dtype")
    _check(lib.b200_copy_kv_pages(ctypes.byref(c), P, P, None, 0, -1, None, None), INVALID, "count")
    _check(lib.b200_copy_kv_pages(ctypes.byref(c), P, P, None, 0, 2 ** 40, None, None), UNSUPPORTED, "pages")
    _check(lib.b200_copy_kv_pages(ctypes.byref(c), None, None, None, 0, 0, None, None), OK, "")
    _check(lib.b200_remap_block_tables(P, 7, 1, 1, 1, P, 4, P, 1, None, None), INVALID, "int32 or int64")
    _check(lib.b200_remap_block_tables(P, 0, 1, 1, 1, None, 4, P, 1, None, None), INVALID, "null")
    _check(lib.b200_remap_block_tables(P, 0, 1, 1, 1, P, 0, P, 1, None, None), INVALID, "pool size")
    _check(lib.b200_remap_block_tables(None, 0, 1, 0, 1, None, 4, None, 1, None, None), OK, "")


@pytest.mark.parametrize("args,want,match", [
    (dict(dtype=_lib.B200_E4M3), UNSUPPORTED, "float32"),
    (dict(vocab=0), INVALID, "vocab"),
    (dict(rows=-1), INVALID, "rows"),
    (dict(vocab=376833), UNSUPPORTED, "376832"),
    (dict(rows=2 ** 31), UNSUPPORTED, "rows"),
    (dict(rows=0), OK, ""),
])
def test_sample_tokens(args, want, match):
    a = _lib.SampleArgs(**(dict(rows=1, row_stride=8, vocab=8, dtype=_lib.B200_F32, temperature=1.0,
                                top_k=0, top_p=1.0, min_p=0.0) | args))
    lib = _lib.load()
    _check(lib.b200_sample_tokens(ctypes.byref(a), P, P, None, None, None, None, P, P, P, None), want, match)
    if want == OK:
        a.rows = 1
        _check(lib.b200_sample_tokens(ctypes.byref(a), P, None, None, None, None, None, P, P, P, None),
               INVALID, "null")


def test_quantize_fp8():
    call = _lib.load().b200_quantize_fp8
    _check(call(P, 1, 16, 16, _lib.B200_F32, 1, P, 16, P, 1, 1, None), UNSUPPORTED, "float16")
    _check(call(P, 1, 16, 16, _lib.B200_F16, 2, P, 16, P, 1, 1, None), INVALID, "128 rows")
    _check(call(P, 1, 0, 16, _lib.B200_F16, 1, P, 16, P, 1, 1, None), INVALID, "cols")
    _check(call(P, 1, 16, 16, _lib.B200_F16, 1, None, 16, P, 1, 1, None), INVALID, "null")
    _check(call(None, 0, 16, 16, _lib.B200_F16, 1, None, 16, None, 1, 1, None), OK, "")


@pytest.mark.parametrize("args,want,match", [
    (dict(dtype=_lib.B200_F32), UNSUPPORTED, "output"),
    (dict(x_dtype=_lib.B200_F16), INVALID, "e4m3"),
    (dict(k=0), INVALID, "columns"),
    (dict(m=-1), INVALID, "rows"),
    (dict(n=2 ** 31), UNSUPPORTED, "2^31"),
    (dict(w_stride=100), INVALID, "16-byte"),
    (dict(x_stride=100), INVALID, "16-byte"),
    (dict(w_stride=112), INVALID, "overlap"),
    (dict(m=2, x_stride=0), INVALID, "overlap"),
    (dict(m=0), OK, ""),
])
def test_fp8_linear(args, want, match):
    a = _lib.Fp8LinearArgs(**(dict(m=1, n=8, k=128, x_stride=128, w_stride=128, out_stride=8,
                                   x_scale_stride_row=1, x_scale_stride_block=1,
                                   w_scale_stride_row=1, w_scale_stride_block=1,
                                   dtype=_lib.B200_BF16, x_dtype=_lib.B200_E4M3) | args))
    call = _lib.load().b200_fp8_linear
    _check(call(ctypes.byref(a), P, P, P, P, None, P, None, 0, None, None), want, match)
    if want == OK:
        a.m = 1
        _check(call(ctypes.byref(a), P, None, P, P, None, P, None, 0, None, None), INVALID, "null")
        _check(call(None, P, P, P, P, None, P, None, 0, None, None), INVALID, "null")
