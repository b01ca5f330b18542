"""Page copies and block-table rewriting, bit for bit."""

import pytest
import torch

from inferkernellab_b200 import (PagedKVCache, _lib, check_device_errors, copy_kv_pages,
                                 remap_block_tables)

pytestmark = pytest.mark.gpu


def _cache(dtype=torch.bfloat16, blocks=40, block=16, kv=2, dim=64, layers=3, seed=0):
    cache = PagedKVCache(blocks, block, kv, dim, num_layers=layers, dtype=dtype, device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(seed)
    for t in (cache.k, cache.v):  # every bit pattern, NaNs among them
        t.view(torch.int16).copy_(torch.randint(-2 ** 15, 2 ** 15, t.shape, generator=gen,
                                                device="cuda", dtype=torch.int16))
    return cache


def _expected(t, src, dst, tokens):
    want = t.view(torch.int16).clone()
    for a, b, n in zip(src, dst, tokens):
        want[:, b, :n] = t.view(torch.int16)[:, a, :n]
    return want


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
@pytest.mark.parametrize("index", [torch.int32, torch.int64, list], ids=["i32", "i64", "list"])
@pytest.mark.parametrize("block,kv,dim,layers", [(16, 2, 64, 3), (1, 1, 16, 1), (256, 8, 128, 2),
                                                 (5, 3, 2, 4), (16, 1, 130, 1)])
def test_copies_whole_and_partial_pages(dtype, index, block, kv, dim, layers):
    n = 11
    gen = torch.Generator().manual_seed(block + dim)
    order = torch.randperm(40, generator=gen).tolist()
    src, dst = order[:n], order[n:2 * n]
    src[1] = src[0]  # one page may go to several places
    counts = torch.randint(0, block + 1, (n,), generator=gen).tolist()
    counts[0], counts[2] = block, 0

    def given(v):
        return list(v) if index is list else torch.tensor(v, dtype=index, device="cuda")

    for tokens in (None, counts):
        cache = _cache(dtype, block=block, kv=kv, dim=dim, layers=layers)
        want = [_expected(t, src, dst, tokens or [block] * n) for t in (cache.k, cache.v)]
        copy_kv_pages(cache, given(src), given(dst), tokens=None if tokens is None else given(tokens))
        for t, w in zip((cache.k, cache.v), want):
            assert torch.equal(t.view(torch.int16), w)
    assert check_device_errors() == 0


def test_ids_outside_the_pool_and_strided_ids():
    cache = _cache()
    src = torch.tensor([[1, 0], [-1, 0], [40, 0], [2, 0], [3, 0]], dtype=torch.int32, device="cuda")[:, 0]
    dst = torch.tensor([10, 11, 12, -5, 13], dtype=torch.int32, device="cuda")
    want = [_expected(t, [1, 3], [10, 13], [16, 16]) for t in (cache.k, cache.v)]
    copy_kv_pages(cache, src, dst)
    assert torch.equal(cache.k.view(torch.int16), want[0])
    assert torch.equal(cache.v.view(torch.int16), want[1])
    assert check_device_errors() == _lib.DEVERR_BAD_BLOCK
    counts = torch.tensor([99, -3, 4, 4, 5], dtype=torch.int32, device="cuda")  # clamped to the page
    want = [_expected(t, [1, 3], [20, 24], [16, 5]) for t in (cache.k, cache.v)]
    copy_kv_pages(cache, src, torch.tensor([20, 21, -1, 23, 24], dtype=torch.int32, device="cuda"),
                  tokens=torch.where(counts == 4, 0, counts))
    assert torch.equal(cache.k.view(torch.int16), want[0])
    assert torch.equal(cache.v.view(torch.int16), want[1])


def test_nothing_to_copy_and_refusals():
    cache = _cache()
    before = cache.k.view(torch.int16).clone()
    copy_kv_pages(cache, [], [])
    copy_kv_pages(cache, torch.empty(0, dtype=torch.int32, device="cuda"),
                  torch.empty(0, dtype=torch.int32, device="cuda"))
    for src, dst, match in (([1, 2], [3], "one entry"), ([1, 2], [3, 3], "destination"),
                            ([1, 2], [2, 3], "destination"), ([1], [40], "invalid physical"),
                            ([-1], [4], "invalid physical")):
        with pytest.raises(ValueError, match=match):
            copy_kv_pages(cache, src, dst)
    with pytest.raises(ValueError, match="tokens must lie"):
        copy_kv_pages(cache, [1], [2], tokens=[17])
    ids = torch.tensor([1], dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError, match="share"):
        copy_kv_pages(cache, ids, ids.long())
    with pytest.raises(ValueError, match="cache device"):
        copy_kv_pages(cache, ids, ids.cpu())
    with pytest.raises(ValueError, match="one entry"):
        copy_kv_pages(cache, ids, ids, tokens=ids.repeat(2))
    cpu = PagedKVCache(4, 16, 2, 64, device="cpu")
    with pytest.raises(ValueError, match="CUDA"):
        copy_kv_pages(cpu, [0], [1])
    assert torch.equal(cache.k.view(torch.int16), before)


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64], ids=["i32", "i64"])
@pytest.mark.parametrize("rows,width", [(1, 1), (7, 33), (300, 517)])
def test_tables_are_rewritten(dtype, rows, width):
    blocks = 977
    gen = torch.Generator(device="cuda").manual_seed(rows)
    page_map = torch.randperm(blocks, generator=gen, device="cuda").int()
    wide = torch.randint(0, blocks, (rows, width + 3), generator=gen, device="cuda").to(dtype)
    tables = wide[:, :width]
    tables[rows // 2, width // 2:] = -1  # unused columns
    want = torch.where(tables < 0, tables, page_map[tables.clamp(min=0).long()].to(dtype))
    assert torch.equal(remap_block_tables(tables, page_map), want)
    keep = wide[:, width:].clone()
    assert remap_block_tables(tables, page_map, out=tables) is tables  # in place, strided rows
    assert torch.equal(tables, want) and torch.equal(wide[:, width:], keep)
    assert check_device_errors() == 0
    tables[0, 0] = blocks + 4
    assert int(remap_block_tables(tables, page_map)[0, 0]) == blocks + 4
    assert check_device_errors() == _lib.DEVERR_BAD_BLOCK


def test_remap_refusals():
    tables = torch.zeros((2, 3), dtype=torch.int32, device="cuda")
    page_map = torch.zeros(4, dtype=torch.int32, device="cuda")
    assert remap_block_tables(tables[:0], page_map).shape == (0, 3)
    with pytest.raises(ValueError, match="2-D"):
        remap_block_tables(tables[0], page_map)
    with pytest.raises(ValueError, match="int32 or int64"):
        remap_block_tables(tables.float(), page_map)
    with pytest.raises(ValueError, match="page_map"):
        remap_block_tables(tables, page_map.long())
    with pytest.raises(ValueError, match="page_map"):
        remap_block_tables(tables, page_map.cpu())
    with pytest.raises(ValueError, match="out must"):
        remap_block_tables(tables, page_map, out=tables.long())
