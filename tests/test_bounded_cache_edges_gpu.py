"""The bounded cache where its calls could go wrong.  Tolerances of accumulated weights are those of test_evict_gpu.py."""
from types import SimpleNamespace

import numpy as np
import pytest
import torch
import torch.nn as nn

import snapmind_b200._lib as lib
from llama_harness import Rope
from test_budget_gpu import normed_attention, reference_layer
from test_chunk_gpu import DT, make_pool
from test_evict_gpu import U, check_mass, dense, reference_mass

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


@pytest.mark.parametrize("cache", ["same", "e4m3"])
def test_copies_without_blocks(cache):
    """A call whose targets find too few blocks on the device changes nothing, a target that holds as many tokens as it would
    end with among them, and names no kept token."""
    from snapmind_b200 import PagedKVPool, QuantizedKVPool

    cls = QuantizedKVPool if cache == "e4m3" else PagedKVPool
    pool = cls(2, 2, 64, 24, max_seqs=4, max_blocks_per_seq=8, dtype=torch.bfloat16, mass=True)
    pool.reserve_each([100, 90, 32, 0])
    g = torch.Generator(device="cuda").manual_seed(1)
    state = [pool.k, pool.v, pool.mass, pool.block_tables, pool.seq_lens, pool.free_stack, pool.free_top]
    for x in state[:2] + ([pool.scales] if cache == "e4m3" else []):
        x.view(torch.uint8).copy_(torch.randint(0, 256, x.view(torch.uint8).shape, generator=g, device="cuda", dtype=torch.int32).to(torch.uint8))
    if cache == "e4m3":
        state.append(pool.scales)
    pool.mass.copy_(torch.rand(pool.mass.shape, generator=g, device="cuda"))
    top = int(pool.free_top)
    pool.free_top.fill_(1)  # the host's count does not know: sequence 3 would need two
    held = [x.view(torch.uint8).clone() for x in state]
    kept = pool.evict(32, recent=3, seqs=[0, 1], into=[2, 3])
    for x, y in zip(state, held):
        assert torch.equal(x.view(torch.uint8), y)
    assert (kept == -1).all()
    with pytest.raises(RuntimeError, match="out of blocks"):
        pool.check()
    # with the blocks there, the same call is what it says
    pool.free_top.fill_(top)
    kept = pool.evict(32, recent=3, seqs=[0, 1], into=[2, 3])
    pool.check()
    assert pool.seq_lens.tolist() == [100, 90, 32, 32] and int(pool.free_top) == top - 2 and (kept >= 0).all()
    for layer in range(2):
        for b in range(2):
            i = kept[layer, b].long()
            for x in (pool.k, pool.v):
                a = dense(pool, x[layer].view(torch.uint8), b, 100 - 10 * b)
                z = dense(pool, x[layer].view(torch.uint8), 2 + b, 32)
                assert torch.equal(z, torch.gather(a, 1, i.unsqueeze(-1).expand(-1, -1, a.shape[-1])))


@pytest.mark.parametrize("dtype,cache,hq,hkv,d,bs,lens,new", [
    # layers of a number of weights that is no multiple of 4
    ("f32", "same", 2, 1, 40, 2, [30, 33], [5, 33]),
    ("bf16", "same", 3, 1, 128, 5, [31, 12], [7, 2]),
    ("bf16", "same", 3, 3, 64, 10, [31, 12], [7, 12]),
    ("f16", "e4m3", 2, 1, 64, 3, [31, 12], [7, 2]),
    ("f32", "same", 2, 1, 40, 2, [30, 33], None),
    ("bf16", "same", 3, 1, 128, 5, [31, 12], None),
    # what the kernels for larger blocks take
    ("bf16", "same", 32, 8, 128, 16, [700, 129], [130, 1]),
    ("bf16", "e4m3", 8, 2, 64, 32, [700, 129], [130, 1]),
    ("bf16", "same", 32, 8, 128, 16, [700, 129], None),
    ("f16", "e4m3", 8, 2, 128, 32, [700, 129], None),
])
def test_weights_of_a_later_layer(dtype, cache, hq, hkv, d, bs, lens, new):
    pool, ks, _ = make_pool(DT[dtype], lens, hkv, d, bs, 11, cache, layers=3)
    assert (pool.num_blocks * hkv * bs % 4 != 0) == (bs < 16)
    g = torch.Generator(device="cuda").manual_seed(2)
    pool.mass = torch.rand((3, pool.num_blocks, hkv, bs), generator=g, device="cuda")
    before = pool.mass.clone()
    counts = new or [1] * len(lens)
    q = torch.randn((sum(counts), hq, d), generator=g, device="cuda").to(DT[dtype])
    if new is None:
        pool.decode(2, q, accumulate=True)
    else:
        pool.attend_chunk(2, q, torch.tensor([0, *np.cumsum(new)], dtype=torch.int32, device="cuda"), accumulate=True)
    pool.check()
    assert torch.equal(pool.mass[:2], before[:2])
    last = SimpleNamespace(mass=pool.mass[2:], block_size=bs, block_tables=pool.block_tables)
    check_mass(last, before[2:], ks, q, counts, 0, 0, d ** -0.5)
    # another layer's weights first: layer 1 on its own
    pool.mass.copy_(before)
    pool.k[1].view(torch.uint8).copy_(pool.k[2].view(torch.uint8))
    pool.v[1].view(torch.uint8).copy_(pool.v[2].view(torch.uint8))
    if cache == "e4m3":
        pool.scales[1].copy_(pool.scales[2])
    if new is None:
        pool.decode(1, q, accumulate=True)
    else:
        pool.attend_chunk(1, q, torch.tensor([0, *np.cumsum(new)], dtype=torch.int32, device="cuda"), accumulate=True)
    assert torch.equal(pool.mass[0], before[0]) and torch.equal(pool.mass[2], before[2])
    check_mass(SimpleNamespace(mass=pool.mass[1:2], block_size=bs, block_tables=pool.block_tables), before[1:2], ks, q, counts, 0, 0, d ** -0.5)


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


class Normed(nn.Module):
    """A projection whose heads are normalised by a module and brought back to the projection's type."""

    def __init__(self, proj, norm, heads):
        super().__init__()
        self.proj, self.norm, self.heads = proj, norm, heads

    def forward(self, x):
        y = self.proj(x)
        z = self.norm(y.view(*y.shape[:-1], self.heads, -1).transpose(1, 2)).to(y.dtype)
        return z.transpose(1, 2).reshape(y.shape)


@pytest.mark.parametrize("where", ["pool", "weighing pool", "cache", "none"])
@pytest.mark.parametrize("rows,norms,auto", [
    (torch.bfloat16, torch.float32, False), (torch.float32, torch.bfloat16, False), (torch.float32, torch.float32, True),
    (torch.float16, torch.bfloat16, False),
])
@torch.no_grad()
def test_norms_of_another_type(rows, norms, auto, where):
    """Norms kept in another type than the projections' rows (or projections under autocast) are the modules' own, rounded to
    the rows' type: the bits of a layer without norms whose projections end with them."""
    from snapmind_b200 import PagedGroupedQueryAttention, PagedKVCache, PagedKVPool

    torch.manual_seed(2)
    rope = Rope(64, 128, 10000.0).cuda()
    layer = normed_attention(d_model=256, n_heads=8, n_kv_heads=2, pe=rope, head_dim=64).cuda()
    for m in (layer.q_norm, layer.k_norm):  # weights that every type holds
        m.weight.copy_(1 + torch.randint(-8, 9, (64,)) / 32)
    for m in (layer.q_proj, layer.k_proj, layer.v_proj, layer.out_proj):
        m.to(rows)
    layer.q_norm.to(norms), layer.k_norm.to(norms)
    plain = PagedGroupedQueryAttention(d_model=256, n_heads=8, n_kv_heads=2, pe=rope, head_dim=64).cuda()
    plain.q_proj, plain.k_proj = Normed(layer.q_proj, layer.q_norm, 8), Normed(layer.k_proj, layer.k_norm, 2)
    plain.v_proj, plain.out_proj = layer.v_proj, layer.out_proj
    x = torch.randn(1 if where in ("cache", "none") else 3, 40, 256, device="cuda").to(rows)
    held = torch.bfloat16 if auto else rows
    mask = torch.triu(torch.full((33, 33), -torch.inf), 1).cuda()
    got = []
    for m in (layer, plain):
        with torch.autocast("cuda", torch.bfloat16, enabled=auto):
            if where == "none":
                got.append(m(x[:, :33], mask=mask)[0])
                continue
            if where == "cache":
                view = PagedKVCache(64, 1, 2, 64, dtype=held, device="cuda").layer_dicts()[0]
            else:
                pool = PagedKVPool(1, 2, 64, 24, 3, 8, dtype=held, mass=where != "pool")
                view = pool.layer_views(3)[0]
                pool.reserve(33)
            out = [m(x[:, :33], kv_cache=view, mask=mask)[0]]
            for t in range(33, 40):
                if where != "cache":
                    pool.reserve(1)
                out.append(m(x[:, t:t + 1], kv_cache=view, position_ids=torch.full((len(x),), t, device="cuda"))[0])
            got.append(torch.cat(out, 1))
            if where != "cache":
                pool.check()
    assert torch.equal(*got)
    if rows == torch.float32 and not auto:  # and the formulas, as test_plugin_over_a_pool has them
        want = reference_layer(layer, x[:, :got[0].shape[1]], rope)
        assert (got[0].double() - want).abs().max() <= 2.0**-12 * want.abs().max()


@pytest.mark.parametrize("dtype,cache,hq,seqs,bs,few", [
    ("bf16", "same", 32, 4, 16, True), ("f16", "e4m3", 32, 4, 16, True), ("f32", "same", 32, 4, 16, True), ("bf16", "same", 32, 4, 8, True),
    ("bf16", "same", 32, 64, 16, False),
])
def test_workspace_of_a_decode(dtype, cache, hq, seqs, bs, few):
    """A decode that accumulates takes no more room than its own sequences' table rows, or the pool, have tokens for, and none
    for scores that it does not keep."""
    from snapmind_b200 import PagedKVPool, QuantizedKVPool

    nb, width, d, batch = 40960 // bs * 4, 2048 // bs, 128, 2 if few else seqs
    pool = (QuantizedKVPool if cache == "e4m3" else PagedKVPool)(1, 8, d, nb if few else seqs * 8, max_seqs=seqs, max_blocks_per_seq=width, block_size=bs,
                                                               dtype=DT[dtype], mass=True)
    pool.reserve(100)
    q = torch.randn((batch, hq, d), device="cuda").to(DT[dtype])
    pool.decode(0, q, accumulate=True)
    size = lib.load().snapmind_paged_gqa_chunk_mass_workspace_bytes
    base = size(d, batch, hq, 8, bs, pool.num_blocks, 0)
    scores = min(batch * width, pool.num_blocks) * bs * hq * 4 if DT[dtype] != torch.float32 and bs == 16 else 0
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    torch.cuda.reset_peak_memory_stats()
    held = torch.cuda.memory_allocated()
    pool.decode(0, q, accumulate=True)
    assert torch.cuda.max_memory_allocated() - held <= base + scores + (4 << 20)  # outputs, and what the allocator does not split off
    pool.check()


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("dtype,cache,hq,hkv,bs,window,sinks", [
    ("bf16", "same", 32, 8, 16, 0, 0), ("f16", "e4m3", 8, 2, 32, 0, 0), ("bf16", "same", 5, 5, 64, 300, 20), ("bf16", "e4m3", 14, 2, 128, 200, 130),
])
def test_scores_by_sequence_and_by_block(dtype, cache, hq, hkv, bs, window, sinks, wide):
    """Decodes of a few of a pool's sequences, and of all that a pool with long table rows holds."""
    lens = [900, 1, 401, 64, 777]
    pool, ks, _ = make_pool(DT[dtype], lens, hkv, 128, bs, 13, cache, spare=0 if wide else 400)
    batch = 5 if wide else 2
    assert (batch * pool.max_blocks_per_seq > pool.num_blocks) == wide
    g = torch.Generator(device="cuda").manual_seed(4)
    pool.mass = torch.rand((1, pool.num_blocks, hkv, bs), generator=g, device="cuda")
    before = pool.mass.clone()
    q = torch.randn((batch, hq, 128), generator=g, device="cuda").to(DT[dtype])
    pool.decode(0, q, accumulate=True, window=window, sinks=sinks)
    pool.check()
    check_mass(pool, before, ks[:batch], q, [1] * batch, window, sinks, 128 ** -0.5)
    first = pool.mass.clone()
    pool.mass.copy_(before)
    pool.decode(0, q, accumulate=True, window=window, sinks=sinks)
    assert torch.equal(pool.mass, first)


@pytest.mark.parametrize("dtype,cache,hq,hkv,d,bs,decode", [
    ("bf16", "same", 8, 2, 128, 16, True), ("bf16", "e4m3", 8, 2, 128, 16, True), ("bf16", "same", 8, 2, 128, 16, False),
    ("f16", "e4m3", 6, 2, 64, 16, False), ("f32", "same", 4, 2, 64, 16, False), ("f32", "same", 4, 2, 64, 16, True),
])
def test_many_sequences(dtype, cache, hq, hkv, d, bs, decode):
    """More sequences than a warp goes over when it plans."""
    rng = np.random.RandomState(5)
    lens = [int(x) for x in rng.randint(0, 200, 400)]
    new = [1] * 400 if decode else [int(min(n, rng.randint(0, 9))) for n in lens]
    pool, ks, _ = make_pool(DT[dtype], lens, hkv, d, bs, 17, cache)
    g = torch.Generator(device="cuda").manual_seed(6)
    pool.mass = torch.rand((1, pool.num_blocks, hkv, bs), generator=g, device="cuda")
    before = pool.mass.clone()
    q = torch.randn((sum(new), hq, d), generator=g, device="cuda").to(DT[dtype])
    if decode:
        pool.decode(0, q, accumulate=True)
    else:
        pool.attend_chunk(0, q, torch.tensor([0, *np.cumsum(new)], dtype=torch.int32, device="cuda"), accumulate=True)
    pool.check()
    check_mass(pool, before, ks, q, new, 0, 0, d ** -0.5)


@pytest.mark.parametrize("dtype,cache", [("bf16", "same"), ("f16", "e4m3")])
def test_a_decode_without_room_for_scores(dtype, cache):
    """The C entry with the workspace of a call that keeps none: the same output, and the weights from K."""
    lens = [900, 1, 401]
    pool, ks, _ = make_pool(DT[dtype], lens, 2, 128, 16, 19, cache)
    g = torch.Generator(device="cuda").manual_seed(7)
    pool.mass = torch.rand((1, pool.num_blocks, 2, 16), generator=g, device="cuda")
    before = pool.mass.clone()
    q = torch.randn((3, 8, 128), generator=g, device="cuda").to(DT[dtype])
    want = pool.decode(0, q, accumulate=True)
    pool.mass.copy_(before)
    need = lib.load().snapmind_paged_gqa_chunk_mass_workspace_bytes(128, 3, 8, 2, 16, pool.num_blocks, 0)
    ws, out, width = torch.empty(need, dtype=torch.uint8, device="cuda"), torch.empty_like(q), pool.max_blocks_per_seq
    args = (q.data_ptr(), 8 * 128, 128, lib.dtype_code(q.dtype), pool.k.data_ptr(), pool.v.data_ptr(),
            pool.scales.data_ptr() if cache == "e4m3" else None, lib.DTYPE_E4M3 if cache == "e4m3" else lib.dtype_code(q.dtype),
            pool.block_tables.data_ptr(), width, width, pool.seq_lens.data_ptr(), None, out.data_ptr(), 8 * 128, 128, 128 ** -0.5, 3, 3, 8, 2,
            128, 16, pool.num_blocks, 0, 0, 0, pool.mass.data_ptr(), ws.data_ptr())
    call = lib.load().snapmind_paged_gqa_chunk_mass
    assert call(*args, need, pool.err.data_ptr(), lib.stream_handle(torch.device("cuda"))) == lib.OK
    pool.check()
    assert torch.equal(out, want)
    check_mass(pool, before, ks, q, [1] * 3, 0, 0, 128 ** -0.5)
    assert call(*args, need - 1, pool.err.data_ptr(), lib.stream_handle(torch.device("cuda"))) == lib.ERR_BAD_ARGUMENT
