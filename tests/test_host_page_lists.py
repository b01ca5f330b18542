"""Page lists of ``copy_kv_pages``, alone and beside tensors, checked on the host."""

import pytest
import torch

from inferkernellab_b200 import CacheLayout
from inferkernellab_b200.ops import _page_lists

LAYOUT = CacheLayout(num_layers=1, num_blocks=40, block_size=16, num_kv_heads=2, head_dim=64)
CPU = torch.device("cpu")


def _tensor(*ids):
    return torch.tensor(ids, dtype=torch.int64)


@pytest.mark.parametrize("src,dst,tokens,match", [
    ([1, 40], _tensor(3, 4), None, "invalid physical"),
    (_tensor(3, 4), [-1, 5], None, "invalid physical"),
    (_tensor(3, 4), [5, 5], None, "destination"),
    (_tensor(3, 4), [5, 6], [17, 0], "tokens must lie"),
    ([3, 4], [5, 6], [0, -1], "tokens must lie"),
    ([1.5, 2], [5, 6], None, "whole"),
    (_tensor(3, 4), [5, 6.5], None, "whole"),
    ([3, 4], [5, 6], [1.5, 2], "whole"),
])
def test_lists_are_checked(src, dst, tokens, match):
    with pytest.raises(ValueError, match=match):
        _page_lists(LAYOUT, CPU, src, dst, tokens)


@pytest.mark.parametrize("src,dst,tokens", [
    ([1, 2], [3, 4], None), ([1, 1], (3, 4), [0, 16]), (_tensor(1, 2), [3, 4], None),
    ([1, 2], _tensor(3, 4), [5, 6]), (_tensor(1, 2), _tensor(3, 4), [5, 6]), ([], [], None)])
def test_lists_become_tensors_beside_them(src, dst, tokens):
    got = _page_lists(LAYOUT, CPU, src, dst, tokens)
    for value, given in zip(got, (src, dst, tokens)):
        assert (value is None) == (given is None)
        if given is not None:
            assert value.tolist() == list(given)
    assert len({v.dtype for v in got if v is not None}) == 1
