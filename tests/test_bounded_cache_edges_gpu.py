"""The bounded cache where its calls could go wrong.  Tolerances of accumulated weights are those of test_evict_gpu.py."""
import pytest
import torch

import snapmind_b200._lib as lib
from test_chunk_gpu import DT, make_pool
from test_evict_gpu import U, dense, reference_mass

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("generic", [False, True])
@pytest.mark.parametrize("new", [150, None])
@pytest.mark.parametrize("dtype,group,d", [
    ("bf16", 1, 128), ("bf16", 3, 128), ("f16", 5, 128), ("bf16", 6, 128), ("bf16", 6, 64), ("f16", 7, 64), ("bf16", 8, 128),
    ("bf16", 12, 64), ("bf16", 50, 128), ("bf16", 71, 64), ("f32", 6, 64),
])
def test_keys_that_an_infinity_masks(dtype, group, d, new, generic):
    """Keys with an infinity in K that gives every query a score of -infinity weigh nothing, as keys that are not there."""
    n, hkv, t = 500, 2, new or 1
    pool, ks, _ = make_pool(DT[dtype], [n], hkv, d, 16, 7)
    g = torch.Generator(device="cuda").manual_seed(group)
    pool.mass = torch.rand((1, pool.num_blocks, hkv, 16), generator=g, device="cuda")
    before = dense(pool, pool.mass[0], 0, n).clone()
    q = torch.randn((t, hkv * group, d), generator=g, device="cuda").to(DT[dtype])
    q[..., 0] = 1
    masked = [0, 5, 129, 300, 349]  # none of them one of the new tokens
    for j in masked:
        pool.k[0, pool.block_tables[0, j // 16], :, j % 16, 0] = -torch.inf
    if new is None:
        out = pool.decode(0, q, accumulate=True, force_generic=generic)
    else:
        out = pool.attend_chunk(0, q, torch.tensor([0, t], dtype=torch.int32, device="cuda"), accumulate=True, force_generic=generic)
    pool.check()
    assert torch.isfinite(out).all()
    got = dense(pool, pool.mass[0], 0, n)
    assert torch.equal(got[:, masked], before[:, masked])
    rest = [j for j in range(n) if j not in masked]
    want, tol = reference_mass(q, ks[0][:, rest], 0, 0, d ** -0.5)
    old = before[:, rest].double()
    assert ((got[:, rest].double() - old - want).abs() <= tol + 2 * U * (old + want) + 1e-30).all()
    # a NaN in a query of kv head 0: in whatever it sees, and nowhere else
    q[t // 3, group - 1, 3] = torch.nan
    if new is None:
        pool.decode(0, q, accumulate=True, force_generic=generic)
    else:
        pool.attend_chunk(0, q, torch.tensor([0, t], dtype=torch.int32, device="cuda"), accumulate=True, force_generic=generic)
    got, sees = dense(pool, pool.mass[0], 0, n), n - t + t // 3 + 1
    assert torch.isnan(got[0, :sees]).all() and not torch.isnan(got[0, sees:]).any() and not torch.isnan(got[1]).any()


def test_new_tokens_after_an_error():
    """What an error word says of other calls does not keep a reserve's new tokens from weighing nothing; a reserve that
    failed leaves all weights as they are."""
    from snapmind_b200 import PagedKVPool

    for word in (lib.DEVERR_TABLE, lib.DEVERR_OUT_OF_BLOCKS, lib.DEVERR_TABLE | lib.DEVERR_BLOCK_ID):
        for how in ("reserve", "each", "device"):
            pool = PagedKVPool(2, 3, 64, 16, max_seqs=2, max_blocks_per_seq=8, mass=True)
            pool.reserve(20)
            pool.mass.fill_(7.0)
            pool.err.fill_(word)
            if how == "reserve":
                pool.reserve(5)
            elif how == "each":
                pool.reserve_each([5, 5])
            else:
                pool.reserve_device(5, 2)
            for layer in range(2):
                for b in range(2):
                    m = dense(pool, pool.mass[layer], b, 25)
                    assert (m[:, 20:] == 0).all() and (m[:, :20] == 7).all(), (word, how)
            assert int((pool.mass == 0).sum()) == 2 * 3 * 2 * 5
            assert int(pool.err.item()) == word
    # a reserve on the device that fails, one that succeeds behind it, without a check between them
    pool = PagedKVPool(1, 2, 64, 4, max_seqs=2, max_blocks_per_seq=8, mass=True)
    pool.reserve(20)
    pool.mass.fill_(7.0)
    pool.reserve_device(30, 2)
    assert (pool.mass == 7).all() and pool.seq_lens.tolist() == [20, 20]
    pool.reserve_device(12, 2)
    pool.account_host(12, 2)
    for b in range(2):
        m = dense(pool, pool.mass[0], b, 32)
        assert (m[:, 20:] == 0).all() and (m[:, :20] == 7).all()
    with pytest.raises(RuntimeError, match="out of blocks"):
        pool.check()
