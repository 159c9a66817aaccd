"""The chunk operators and the 8-bit cache at the ends of their ranges: counts from device memory,
exponents far apart, masked infinities, bad block ids."""
import pytest
import torch

import snapmind_b200._lib as lib

pytestmark = pytest.mark.gpu


def device_state(pool):
    return [t.tolist() for t in (pool.block_tables, pool.seq_lens, pool.free_stack, pool.free_top)]


@pytest.mark.parametrize("counts,word", [
    ([1, -1, 0], lib.DEVERR_TABLE),
    ([2**31 - 1, 0, 0], lib.DEVERR_TABLE),
    ([0, 2**31 - 1, 2**31 - 1], lib.DEVERR_TABLE),
    ([2**31 - 1, -(2**31), 3], lib.DEVERR_TABLE),
    ([0, 0, 4 * 16 - 50 + 1], lib.DEVERR_TABLE),   # one token past the table row
    ([24, 63, 14], lib.DEVERR_OUT_OF_BLOCKS),      # 4 blocks of 3 free ones
])
def test_device_counts_that_do_not_fit(cuda_device, counts, word):
    """reserve_each of counts in device memory: the error word tells, and nothing changes."""
    from snapmind_b200 import PagedKVPool

    pool = PagedKVPool(1, 1, 64, 11, 3, 4, dtype=torch.bfloat16)
    pool.reserve_each([40, 1, 50])
    before = device_state(pool)

    def reserve(n):
        n = torch.tensor(n, dtype=torch.int32, device="cuda")
        status = lib.load().snapmind_kv_reserve_each(
            pool.block_tables.data_ptr(), 4, 4, pool.seq_lens.data_ptr(), n.data_ptr(), 3, 16, pool.free_stack.data_ptr(),
            pool.free_top.data_ptr(), 11, pool.err.data_ptr(), lib.stream_handle(torch.device("cuda")))
        assert status == lib.OK
        return int(pool.err.item())

    assert reserve(counts) == word
    assert device_state(pool) == before
    pool.err.zero_()
    assert reserve([24, 47, 14]) == 0  # up to the rows' ends and the last block
    assert pool.seq_lens.tolist() == [64, 48, 64] and int(pool.free_top.item()) == 0
