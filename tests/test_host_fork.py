"""Forked requests on the host side: shared blocks, their holders, and the runtime."""

import pytest

from inferkernellab_b200 import (BlockAllocator, InferenceRuntime, PagedKVCache,
                                 TokenBudgetScheduler)


def test_named_holders_take_a_block_over():
    a = BlockAllocator(4)
    blocks = a.allocate(2, owner=1)
    a.share(blocks, owner=2)
    a.share(blocks, owner=3)
    a.free(blocks, owner=2)  # a holder in between
    assert [a.ref_count(b) for b in blocks] == [2, 2] and a.owner(blocks[0]) == 1
    a.free(blocks, owner=1)  # the owner: the next holder takes over
    assert [a.owner(b) for b in blocks] == [3, 3] and a.num_used_blocks == 2
    with pytest.raises(ValueError, match="not owned"):
        a.free(blocks, owner=1)
    a.free(blocks, owner=3)
    assert a.num_free_blocks == 4
    assert a.allocate(1, owner=5) == [blocks[-1]] and a.owner(blocks[-1]) == 5


def test_fork_of_full_blocks_shares_them():
    cache = PagedKVCache(8, 4, 2, 16, device="cpu")
    table = cache.allocate_request(1, 8)
    tables = cache.fork_request(table, 8, [2, 3])
    assert tables == [table, table]  # nothing to copy
    assert [cache.allocator.ref_count(b) for b in table] == [3, 3]
    for rid, t in ((1, table), (3, tables[1]), (2, tables[0])):
        cache.release_request(t, rid)
    assert cache.allocator.num_used_blocks == 0


def test_fork_is_all_or_nothing():
    cache = PagedKVCache(4, 4, 2, 16, device="cpu")
    table = cache.allocate_request(1, 6)
    with pytest.raises(RuntimeError, match="out of KV blocks"):
        cache.fork_request(table, 6, [2, 3, 4])
    assert [cache.allocator.ref_count(b) for b in table] == [1, 1]
    with pytest.raises(ValueError, match="shorter"):
        cache.fork_request(table, 9, [2])
    with pytest.raises(ValueError, match="positive"):
        cache.fork_request(table, 0, [2])


def test_runtime_forks_join_the_decode_batch():
    cache = PagedKVCache(12, 4, 2, 16, device="cpu")
    seen = []
    runtime = InferenceRuntime(cache, TokenBudgetScheduler(8, 64),
                               prefill_batch_fn=lambda *a: None,
                               decode_fn=lambda requests: seen.append([r.request_id for r in requests]))
    runtime.submit(0, 8, 3)
    with pytest.raises(ValueError, match="cached prompt"):
        runtime.fork(0, [1])
    runtime.step()
    forks = runtime.fork(0, [1, 2])
    assert [(f.cached_tokens, f.generated_tokens, f.status) for f in forks] == [(8, 0, "running")] * 2
    for bad in ([1], [5, 5]):
        with pytest.raises(ValueError, match="duplicate"):
            runtime.fork(0, bad)
    with pytest.raises(ValueError, match="cached prompt"):
        runtime.fork(9, [10])
    runtime.step()
    tables = [r.block_table for r in (runtime._requests[i] for i in range(3))]
    assert all(t[:2] == tables[0][:2] for t in tables)
    assert len({t[2] for t in tables}) == 3  # each writes its next tokens to its own block
    while runtime.scheduler.running:
        runtime.step()
    assert seen == [[0, 1, 2]] * 3
    assert cache.allocator.num_used_blocks == 0
    with pytest.raises(ValueError, match="cached prompt"):
        runtime.fork(0, [7])  # finished
