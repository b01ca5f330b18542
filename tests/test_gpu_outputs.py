"""Outputs given by the caller: any layout of whole rows, none whose rows share memory."""

import pytest
import torch

from inferkernellab_b200 import (PagedKVCache, check_device_errors, fp8_linear, qk_norm_rope_append,
                                 quantize_fp8_weight, remap_block_tables)

pytestmark = pytest.mark.gpu


def _qk_norm(tokens, heads, out=None):
    gen = torch.Generator(device="cuda").manual_seed(3)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda").bfloat16()

    cache = PagedKVCache(2, 16, 1, 64, dtype=torch.bfloat16, device="cuda")
    return qk_norm_rope_append(normal(tokens, heads, 64), normal(tokens, 1, 64), normal(tokens, 1, 64),
                               normal(64), normal(64), normal(tokens, 64), normal(tokens, 64), cache,
                               torch.arange(tokens, dtype=torch.int32, device="cuda"), out=out)


def _empty(*shape, dtype=torch.bfloat16):
    return torch.zeros(shape, dtype=dtype, device="cuda")


def test_qk_norm_outputs():
    want = _qk_norm(5, 4)
    for out in (_empty(4, 5, 64).transpose(0, 1), _empty(5, 4, 80)[..., :64], _empty(5, 9, 64)[:, ::2][:, :4],
                _empty(7, 4, 64)[1:6], _empty(4, 6, 72)[:, 1:, 3:67].transpose(0, 1)):
        assert _qk_norm(5, 4, out) is out and torch.equal(out, want)
    for shape in ((1, 4), (5, 1), (1, 1)):  # a single token or head has no stride to clear
        out = _empty(64 * 20).as_strided((*shape, 64), (64 if shape[0] > 1 else 0, 64 if shape[1] > 1 else 0, 1))
        assert torch.equal(_qk_norm(*shape, out), _qk_norm(*shape))
    for out in (_empty(1, 4, 64).expand(5, 4, 64), _empty(5, 1, 64).expand(5, 4, 64),
                _empty(2000).as_strided((5, 4, 64), (256, 63, 1)),
                _empty(2000).as_strided((5, 4, 64), (255, 64, 1)),
                _empty(2000).as_strided((5, 4, 64), (64, 64, 1))):
        with pytest.raises(ValueError, match="overlap"):
            _qk_norm(5, 4, out)
    assert check_device_errors() == 0


def test_fp8_linear_outputs():
    x = torch.randn((6, 128), device="cuda").bfloat16()
    w, ws = quantize_fp8_weight(torch.randn((40, 128), device="cuda").bfloat16())
    want = fp8_linear(x, w, ws)
    for out in (_empty(12, 40)[::2], _empty(6, 48)[:, 5:45]):
        assert fp8_linear(x, w, ws, out=out) is out and torch.equal(out, want)
    one = _empty(40).as_strided((1, 40), (0, 1))
    assert torch.equal(fp8_linear(x[:1], w, ws, out=one), want[:1])
    for out in (_empty(1, 40).expand(6, 40), _empty(240).as_strided((6, 40), (39, 1))):
        with pytest.raises(ValueError, match="overlap"):
            fp8_linear(x, w, ws, out=out)


def test_remapped_table_outputs():
    tables = torch.randint(0, 9, (4, 7), device="cuda", dtype=torch.int32)
    page_map = torch.randperm(9, device="cuda").int()
    out = _empty(8, 7, dtype=torch.int32)[::2]
    assert torch.equal(remap_block_tables(tables, page_map, out=out), page_map[tables.long()])
    for out in (_empty(1, 7, dtype=torch.int32).expand(4, 7),
                _empty(40, dtype=torch.int32).as_strided((4, 7), (6, 1))):
        with pytest.raises(ValueError, match="overlap"):
            remap_block_tables(tables, page_map, out=out)
    shared = tables[:1].expand(4, 7)  # one row for several requests: read, but not in place
    assert torch.equal(remap_block_tables(shared, page_map), page_map[shared.long()])
    with pytest.raises(ValueError, match="overlap"):
        remap_block_tables(shared, page_map, out=shared)
