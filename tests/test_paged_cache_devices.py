"""A page table on another device than its pages is refused when the cache is made: kernels read both (CPU)."""
import pytest
import torch

from treeattn_amd import kernels as K


def test_pool_and_table_share_a_device():
    pool = torch.zeros(4, 2, 8, 16)
    table = torch.zeros(1, 2, 2, dtype=torch.int32)
    assert K.PagedCache(pool, table, 16).tcap == 16
    for a, b in ((pool.to('meta'), table), (pool, table.to('meta'))):
        with pytest.raises(ValueError, match='table on'):
            K.PagedCache(a, b, 16)
