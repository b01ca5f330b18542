"""Forks released in any order, with and without naming who releases, and forks that fail."""

import itertools

import pytest

from inferkernellab_b200 import (BlockAllocator, InferenceRuntime, PagedKVCache, PrefixCache,
                                 TokenBudgetScheduler)


@pytest.mark.parametrize("unnamed", [u for n in range(4) for u in itertools.combinations((1, 2, 3), n)])
@pytest.mark.parametrize("order", list(itertools.permutations((1, 2, 3))))
def test_forks_release_in_any_order_named_or_not(order, unnamed):
    cache = PagedKVCache(8, 4, 2, 16, device="cpu")
    table = cache.allocate_request(1, 8)
    tables = {1: table} | dict(zip((2, 3), cache.fork_request(table, 8, [2, 3])))
    for i, rid in enumerate(order):
        assert [cache.allocator.ref_count(b) for b in table] == [3 - i] * 2
        cache.release_request(tables[rid], None if rid in unnamed else rid)
    assert cache.allocator.num_used_blocks == 0
    with pytest.raises(ValueError, match="not allocated"):
        cache.release_request(table, 1)


def test_a_named_release_is_still_checked():
    a = BlockAllocator(4)
    blocks = a.allocate(1, owner=1)
    a.share(blocks, owner=2)
    a.free(blocks)  # 1 or 2: who is left is not known
    with pytest.raises(ValueError, match="not owned"):
        a.free(blocks, owner=3)
    a.free(blocks, owner=2)
    blocks = a.allocate(1, owner=4)  # the same block: its holders of before are forgotten
    with pytest.raises(ValueError, match="not owned"):
        a.free(blocks, owner=2)
    a.free(blocks, owner=4)
    assert a.num_free_blocks == 4


def test_a_fork_whose_copy_fails_leaves_nothing_behind():
    cache = PagedKVCache(8, 4, 2, 16, device="cpu")  # the page copy needs a CUDA cache
    table = cache.allocate_request(1, 6)
    expected = PagedKVCache(8, 4, 2, 16, device="cpu")
    expected.allocate_request(1, 6)
    for _ in range(3):
        with pytest.raises(ValueError, match="CUDA"):
            cache.fork_request(table, 6, [2, 3])
    assert [cache.allocator.ref_count(b) for b in table] == [1, 1]
    assert [cache.allocator.owner(b) for b in table] == [1, 1]
    assert cache.allocator.num_used_blocks == 2
    with pytest.raises(ValueError, match="not owned"):
        cache.release_request(table, 2)  # a holder of the failed fork only
    # what is handed out next is what it would have been
    assert cache.allocator.allocate(6) == expected.allocator.allocate(6)
    cache.release_request(table, 1)


@pytest.mark.parametrize("first", [1, 2, 3])
def test_sharers_of_a_prefix_release_after_the_index_was_dropped(first):
    """Request 2 has request 1's prompt blocks through the index, 3 is a fork of 2; the index lets
    go of its reference while all of them still run."""
    cache = PagedKVCache(12, 4, 2, 16, device="cpu")
    prefix = PrefixCache(cache.allocator, 4)
    runtime = InferenceRuntime(cache, TokenBudgetScheduler(8, 64), prefix_cache=prefix,
                               prefill_batch_fn=lambda *a: None, decode_fn=lambda requests: None)
    prompt = tuple(range(8))
    requests = {1: runtime.submit(1, 8, 5, token_ids=prompt)}
    runtime.step()
    requests[2] = runtime.submit(2, 9, 5, token_ids=prompt + (9,))
    runtime.step()
    assert requests[2].block_table[:2] == requests[1].block_table[:2]
    tables = {rid: list(r.block_table[:2]) for rid, r in requests.items()}
    cache.allocator.share(tables[2], owner=3)
    prefix.clear()
    for rid in [first] + [r for r in (1, 2, 3) if r != first]:
        cache.release_request(tables.get(rid, tables[2]), rid)
    assert cache.allocator.num_used_blocks == 1  # request 2's own last block
