"""The page, head-norm and 8-bit operators from host threads that do not wait for each other."""

import threading

import pytest
import torch

from inferkernellab_b200 import (PagedKVCache, check_device_errors, copy_kv_pages, fp8_linear,
                                 qk_norm_rope_append, quantize_fp8, quantize_fp8_weight,
                                 remap_block_tables)

pytestmark = pytest.mark.gpu


def _normal(*shape):
    return torch.randn(shape, device="cuda").bfloat16()


def _linear(m, n, k):
    x, (w, s) = _normal(m, k), quantize_fp8_weight(_normal(n, k))
    return lambda: fp8_linear(x, w, s)


def _quantize():
    x = _normal(130, 1000)
    return lambda: torch.cat([t.float() for t in quantize_fp8(x)], dim=1)


def _head_norm(tokens):
    cache = PagedKVCache(-(-tokens // 16), 16, 2, 64, dtype=torch.bfloat16, device="cuda")
    q, k, v = _normal(tokens, 8, 64), _normal(tokens, 2, 64), _normal(tokens, 2, 64)
    weights, cos, sin = (_normal(64), _normal(64)), _normal(tokens, 64), _normal(tokens, 64)
    slots = torch.arange(tokens, dtype=torch.int32, device="cuda")

    def call():
        out = qk_norm_rope_append(q, k, v, *weights, cos, sin, cache, slots)
        return torch.cat([out.flatten(), cache.k.flatten()[:k.numel()], cache.v.flatten()[:v.numel()]])

    return call


def _pages():
    cache = PagedKVCache(12, 16, 2, 64, num_layers=2, dtype=torch.bfloat16, device="cuda")
    cache.k.normal_()
    cache.v.normal_()
    tables = torch.randint(0, 12, (3, 5), device="cuda", dtype=torch.int32)
    page_map = torch.arange(12, device="cuda", dtype=torch.int32).flip(0)

    def call():
        copy_kv_pages(cache, [1, 2, 3], [7, 8, 9], tokens=[16, 3, 0])
        return torch.cat([cache.k.float().flatten(), cache.v.float().flatten(),
                          remap_block_tables(tables, page_map).float().flatten()])

    return call


def test_operators_from_several_threads():
    calls = [_linear(2500, 2560, 256), _linear(3, 640, 1024), _linear(200, 512, 512), _quantize(),
             _head_norm(1), _head_norm(300), _pages()]
    want = [call() for call in calls]
    torch.cuda.synchronize()
    start, wrong = threading.Barrier(len(calls)), []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                start.wait()
                for _ in range(60):
                    got = calls[i]()
                    if not torch.equal(got, want[i]):
                        wrong.append(i)
        except Exception as error:
            wrong.append((i, error))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(calls))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong, wrong
    assert check_device_errors() == 0
