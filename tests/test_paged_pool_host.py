"""The page pool's bookkeeping (no GPU)."""
import pytest
import torch

from tinyserve_b200.paged import PagePool


def test_pages_are_handed_out_once_and_come_back():
    pool = PagePool(2, 6, 1, 16, 64, torch.bfloat16, torch.device("cpu"))
    assert [pool.pages_for(n) for n in (0, 1, 16, 17)] == [0, 1, 1, 2]
    a, b = pool.take(4), pool.take(2)
    assert sorted(a + b) == list(range(6)) and pool.free == 0
    with pytest.raises(RuntimeError):
        pool.take(1)
    pool.give_back(a)
    assert pool.free == 4 and sorted(pool.take(4)) == sorted(a)
    assert pool.k.shape == (2, 6, 1, 16, 64) and pool.v.dtype == torch.bfloat16
