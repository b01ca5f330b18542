"""C entry points refuse outputs whose rows share memory.  No kernel is launched here."""

import ctypes

import pytest

from inferkernellab_b200 import _lib

P = 4096  # a non-null address that no refused call may read


def _refused(status):
    assert status == _lib.B200_ERR_INVALID and "overlap" in _lib.last_error(), _lib.last_error()


@pytest.mark.parametrize("stride", [0, 4, 7])
def test_fp8_linear(stride):
    a = _lib.Fp8LinearArgs(m=2, n=8, k=128, x_stride=128, w_stride=128, out_stride=stride,
                           x_scale_stride_row=1, x_scale_stride_block=1, w_scale_stride_row=1,
                           w_scale_stride_block=1, dtype=_lib.B200_BF16, x_dtype=_lib.B200_E4M3)
    _refused(_lib.load().b200_fp8_linear(ctypes.byref(a), P, P, P, P, None, P, None, 0, None, None))


@pytest.mark.parametrize("stride", [0, 5])
def test_remap_block_tables(stride):
    _refused(_lib.load().b200_remap_block_tables(P, 0, 6, 2, 6, P, 4, P, stride, None, None))


@pytest.mark.parametrize("tokens,heads,token_stride,head_stride", [
    (3, 4, 0, 64), (3, 4, 256, 0), (3, 4, 255, 64), (3, 4, 256, 63), (3, 4, 64, 191), (3, 4, 63, 192),
    (2, 2, 0, 128), (1, 4, 0, 63), (3, 2, 0, 0), (3, 2, 64, 128)])
def test_qk_norm_rope_append(tokens, heads, token_stride, head_stride):
    c = _lib.CacheDesc(k_cache=P, v_cache=P, num_layers=1, num_blocks=4, block_size=16,
                       num_kv_heads=heads // 2 or 1, head_dim=64, dtype=_lib.B200_BF16)
    a = _lib.QkNormArgs(num_tokens=tokens, num_q_heads=heads, layer=0, rotary_dim=64, eps=1e-6,
                        q_out_stride_token=token_stride, q_out_stride_head=head_stride)
    _refused(_lib.load().b200_qk_norm_rope_append(ctypes.byref(c), ctypes.byref(a), P, P, P, P, P,
                                                  P, P, P, P, None, None))
