"""Calls at the edges of what the chunk operators' Python side takes, without a GPU."""
import numpy as np
import pytest

from snapmind_b200.block_pool import BlockPool


def host_pool(lens, free=100, width=8, block_size=16):
    """A pool's host side only: a call that gets past its checks fails for want of a device."""
    pool = BlockPool.__new__(BlockPool)
    pool.max_seqs, pool.block_size, pool.max_blocks_per_seq = len(lens), block_size, width
    pool._host_lens, pool._host_free = np.array(lens, dtype=np.int64), free
    return pool


@pytest.mark.parametrize("counts", [
    np.array([1, 2**63], dtype=np.uint64), np.array([2**64 - 1, 1], dtype=np.uint64), np.array([2**31, 0]),
    np.array([2**63 - 1, 0]), np.array([-1, 0]), [2**70, 0],
], ids=str)
def test_counts_no_length_can_hold(counts):
    pool = host_pool([40, 30])
    with pytest.raises(ValueError, match="reserve_each"):
        pool.reserve_each(counts)
    assert pool.host_lens.tolist() == [40, 30] and pool._host_free == 100
