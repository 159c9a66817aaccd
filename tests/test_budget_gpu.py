"""The paths that norm, rotate, accumulate and evict together: the attention plugin, generation within a budget, captured
and overlapping calls."""
import math

import numpy as np
import pytest
import torch
import torch.nn as nn

from llama_harness import LlamaHarness, LlamaShape, Rope, init_weights
from test_evict_gpu import dense, kept_of, reference_mass, weights

pytestmark = pytest.mark.gpu


def normed_attention(**kw):
    from snapmind_b200 import PagedGroupedQueryAttention

    return PagedGroupedQueryAttention(qk_norm_eps=1e-5, **kw)


def reference_layer(layer, x, rope):
    """The layer's causal output for [B, T, d_model], in 64 bits: projections, norms, rotation, attention."""
    f = lambda m, y: y @ m.weight.double().t()  # noqa: E731
    b, t, _ = x.shape
    heads = lambda y, n: y.view(b, t, n, layer.head_dim).transpose(1, 2)  # noqa: E731
    x = x.double()
    q, k, v = (heads(f(m, x), n) for m, n in ((layer.q_proj, layer.n_heads), (layer.k_proj, layer.n_kv_heads), (layer.v_proj, layer.n_kv_heads)))
    norm = lambda y, m: y / torch.sqrt((y * y).mean(-1, keepdim=True) + m.eps) * m.weight.double()  # noqa: E731
    cos, sin = rope.cos_cached[:t].double(), rope.sin_cached[:t].double()
    turn = lambda y: y * cos + Rope._rotate_half(y) * sin  # noqa: E731
    q, k = turn(norm(q, layer.q_norm)), turn(norm(k, layer.k_norm))
    rep = layer.n_heads // layer.n_kv_heads
    k, v = k.repeat_interleave(rep, 1), v.repeat_interleave(rep, 1)
    s = q @ k.transpose(-1, -2) / math.sqrt(layer.head_dim)
    s = s.masked_fill(torch.ones(t, t, dtype=torch.bool, device=x.device).triu(1), -math.inf)
    return f(layer.out_proj, (torch.softmax(s, -1) @ v).transpose(1, 2).reshape(b, t, -1))


@pytest.mark.parametrize("mass", [False, True])
@torch.no_grad()
def test_plugin_over_a_pool(mass):
    """Prefill, then tokens one by one, against the formulas.  All f32: every stage is off by its length (256 terms at
    most) times 2^-24 of what it sums, six stages and softmax weights next to each other: 2^-12 of the largest output."""
    from snapmind_b200 import PagedKVPool

    torch.manual_seed(0)
    rope = Rope(64, 128, 10000.0).cuda()
    layer = normed_attention(d_model=256, n_heads=8, n_kv_heads=2, pe=rope, head_dim=64).cuda()
    layer.q_norm.weight.copy_(1 + 0.3 * torch.randn(64))
    layer.k_norm.weight.copy_(1 + 0.3 * torch.randn(64))
    x = torch.randn(3, 40, 256, device="cuda")
    want = reference_layer(layer, x, rope)
    pool = PagedKVPool(1, 2, 64, 24, 3, 8, dtype=torch.float32, mass=mass)
    view = pool.layer_views(3)[0]
    pool.reserve(33)
    mask = torch.triu(torch.full((33, 33), -math.inf), 1).cuda()
    got = [layer(x[:, :33], kv_cache=view, mask=mask)[0]]
    for t in range(33, 40):
        pool.reserve(1)
        got.append(layer(x[:, t:t + 1], kv_cache=view, position_ids=torch.full((3,), t, device="cuda"))[0])
    pool.check()
    err = (torch.cat(got, 1).double() - want).abs().max()
    assert err <= 2.0**-12 * want.abs().max(), float(err / want.abs().max())
    if mass:  # each query gives 1 in all for each head: 8 / 2 query heads a kv head, 40 queries
        for b in range(3):
            assert torch.allclose(dense(pool, pool.mass[0], b, 40).sum(1), torch.full((2,), 160.0, device="cuda"), rtol=1e-4)


@torch.no_grad()
def test_plugin_over_the_other_caches():
    from snapmind_b200 import PagedKVCache

    torch.manual_seed(1)
    rope = Rope(64, 128, 10000.0).cuda()
    layer = normed_attention(d_model=256, n_heads=8, n_kv_heads=2, pe=rope, head_dim=64).cuda()
    layer.q_norm.weight.copy_(1 + 0.3 * torch.randn(64))
    x = torch.randn(1, 40, 256, device="cuda")
    want = reference_layer(layer, x, rope)
    mask = torch.triu(torch.full((40, 40), -math.inf), 1).cuda()
    limit = 2.0**-12 * want.abs().max()
    assert (layer(x, mask=mask)[0].double() - want).abs().max() <= limit
    cache = PagedKVCache(64, 1, 2, 64, dtype=torch.float32, device="cuda")
    view = cache.layer_dicts()[0]
    got = [layer(x[:, :33], kv_cache=view, mask=mask[:33, :33])[0]]
    got += [layer(x[:, t:t + 1], kv_cache=view, position_ids=torch.tensor([t], device="cuda"))[0] for t in range(33, 40)]
    assert (torch.cat(got, 1).double() - want).abs().max() <= limit
    # a position encoding without tables, or gradients: the modules' own arithmetic
    class Plain(nn.Module):
        def apply_to_qk(self, q, k, position_ids=None):
            return rope.apply_to_qk(q, k, position_ids)

    layer.pe = Plain()
    assert (layer(x, mask=mask)[0].double() - want).abs().max() <= limit


SHAPE = LlamaShape(vocab_size=97, d_model=256, n_heads=8, n_kv_heads=2, n_layers=2, d_ff=256, max_seq_len=256)


def model(dtype=torch.float32):
    m = LlamaHarness(SHAPE, normed_attention)
    init_weights(m, 5)
    return m.to("cuda", dtype)


@pytest.mark.parametrize("cache", ["same", "e4m3"])
def test_generation_within_a_budget(cache):
    """Captured steps give the ids of eager ones, the sequences never hold more than the budget and its slack, and what
    they hold is what evicting by hand leaves."""
    from snapmind_b200 import PagedKVPool, QuantizedKVPool
    from snapmind_b200.engine import BatchedGraphDecoder

    cls = QuantizedKVPool if cache == "e4m3" else PagedKVPool
    m = model()
    prompts = torch.randint(0, 97, (3, 60), generator=torch.Generator().manual_seed(0)).cuda()
    ids, held = [], []
    for use_graph in (False, True):
        pool = cls(2, 2, 32, 3 * 4, 3, 4, dtype=torch.float32, mass=True)  # 64 tokens each: no more fit
        dec = BatchedGraphDecoder(m, pool, 3, use_graph=use_graph, budget=40, slack=9, recent=8, sinks=2)
        seen = []
        evict = pool.evict

        def spy(*a, **k):
            seen.append(int(pool.host_lens.max()))
            return evict(*a, **k)

        pool.evict = spy
        ids.append(dec.generate(prompts, 50))
        assert seen == [60] + [49] * 5 and pool.seq_lens.tolist() == list(pool.host_lens) == [44] * 3
        assert int(pool.free_top) == pool._host_free == 3
        held.append([t.clone() for t in (*pool.gather(), pool.mass)])
    assert ids[0] == ids[1] and len(ids[0][0]) == 50
    for a, b in zip(*held):
        assert torch.equal(a, b)


def test_a_budget_that_is_never_reached_changes_nothing():
    from snapmind_b200 import PagedKVPool
    from snapmind_b200.engine import BatchedGraphDecoder

    m = model()
    prompts = torch.randint(0, 97, (2, 30), generator=torch.Generator().manual_seed(1)).cuda()
    ids = []
    for kw in ({}, dict(budget=100, recent=10)):
        pool = PagedKVPool(2, 2, 32, 16, 2, 8, dtype=torch.float32, mass=True)
        ids.append(BatchedGraphDecoder(m, pool, 2, **kw).generate(prompts, 20))
    assert ids[0] == ids[1]
    with pytest.raises(ValueError, match="budget"):
        BatchedGraphDecoder(m, PagedKVPool(2, 2, 32, 16, 2, 8), 2, budget=10)


def fill(pool, g, kind="plain"):
    pool.k.copy_(torch.randn(pool.k.shape, generator=g, device="cuda"))
    pool.v.copy_(torch.randn(pool.v.shape, generator=g, device="cuda"))
    pool.mass.copy_(weights(pool.mass.shape, g, kind))


def test_a_captured_step_that_evicts():
    """reserve, a decode that accumulates and evict_device, captured once and replayed, against the same calls eagerly."""
    from snapmind_b200 import PagedKVPool

    results = []
    for captured in (False, True):
        pool = PagedKVPool(1, 2, 128, 40, max_seqs=3, max_blocks_per_seq=12, mass=True)
        g = torch.Generator(device="cuda").manual_seed(2)
        pool.reserve_each([50, 33, 120])
        fill(pool, g)
        q = torch.randn((3, 8, 128), generator=g, device="cuda").bfloat16()
        k = torch.randn((3, 2, 128), generator=g, device="cuda").bfloat16()
        out = torch.empty_like(q)

        def step():
            pool.reserve_device(3, 3)
            pool.append(0, k, k)
            pool.decode(0, q, out=out, accumulate=True)
            return pool.evict_device(48, recent=5, sinks=1, batch=3)

        if captured:
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.stream(side):
                kept = step()
            torch.cuda.current_stream().wait_stream(side)
            first = kept.clone()
            with torch.cuda.graph(graph):
                kept = step()
                with pytest.raises(RuntimeError, match="captured"):
                    pool.evict(8)
            steps = [first]
            for _ in range(3):
                graph.replay()
                steps.append(kept.clone())
        else:
            steps = [step() for _ in range(4)]
        for _ in range(4):
            pool.account_host(3, 3)
            pool.account_evict(48, 3)
        pool.check()
        assert pool.seq_lens.tolist() == list(pool.host_lens) == [48, 45, 48]
        assert int(pool.free_top) == pool._host_free
        results.append([*steps, out.clone(), *pool.gather(), pool.mass.clone(), pool.block_tables.clone()])
    for a, b in zip(*results):
        assert torch.equal(a, b)


def test_two_streams_and_another_stream():
    """Calls of two layers on two streams at once, and an eviction on a third: the bits of one stream's calls."""
    from snapmind_b200 import PagedKVPool

    def make():
        pool = PagedKVPool(2, 8, 128, 700, max_seqs=4, max_blocks_per_seq=300, mass=True)
        g = torch.Generator(device="cuda").manual_seed(4)
        pool.reserve_each([4000, 1200, 60, 3])
        fill(pool, g)
        return pool, torch.randn((4, 32, 128), generator=g, device="cuda").bfloat16()

    want, q = make()
    cu = torch.tensor([0, 1, 3, 3, 4], dtype=torch.int32, device="cuda")
    for layer in range(2):
        for _ in range(5):
            want.decode(layer, q, accumulate=True)
            want.attend_chunk(layer, q, cu, accumulate=True)
    kept = want.evict(500, recent=64)
    pool, q = make()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    for _ in range(5):
        for layer in range(2):
            with torch.cuda.stream(streams[layer]):
                pool.decode(layer, q, accumulate=True)
                pool.attend_chunk(layer, q, cu, accumulate=True)
    for s in streams[:2]:
        streams[2].wait_stream(s)
    with torch.cuda.stream(streams[2]):
        got = pool.evict(500, recent=64)
    torch.cuda.synchronize()
    assert torch.equal(got, kept) and torch.equal(pool.mass, want.mass) and torch.equal(pool.k, want.k)


@pytest.mark.parametrize("call", ["decode", "chunk"])
def test_nan_and_no_block(call):
    """A NaN query makes the tokens that it sees NaN, in its kv head alone; a table entry that is no block is flagged, and
    its tokens and all slots of other sequences keep their weight."""
    from snapmind_b200 import PagedKVPool

    pool = PagedKVPool(1, 2, 128, 64, max_seqs=2, max_blocks_per_seq=20, mass=True)
    g = torch.Generator(device="cuda").manual_seed(6)
    pool.reserve_each([200, 100])
    fill(pool, g)
    q = torch.randn((5, 8, 128), generator=g, device="cuda").bfloat16()
    cu = torch.tensor([0, 3, 5], dtype=torch.int32, device="cuda")
    run = (lambda x: pool.decode(0, x[:2], accumulate=True)) if call == "decode" else (lambda x: pool.attend_chunk(0, x, cu, accumulate=True))
    before = pool.mass.clone()
    bad = q.clone()
    bad[1, 1, 7] = float("nan")  # decode: sequence 1; chunk: the second of sequence 0's three new tokens; kv head 0
    run(bad)
    b, sees = (1, 100) if call == "decode" else (0, 199)
    m = dense(pool, pool.mass[0], b, 100 if call == "decode" else 200)
    assert torch.isnan(m[0, :sees]).all() and not torch.isnan(m[0, sees:]).any() and not torch.isnan(m[1]).any()
    assert not torch.isnan(dense(pool, pool.mass[0], 1 - b, 100 if b == 0 else 200)).any()
    pool.check()
    pool.mass.copy_(before)
    pool.block_tables[0, 3] = 64  # past the pool
    run(q)
    with pytest.raises(RuntimeError, match="block id"):
        pool.check()
    assert torch.isfinite(pool.mass).all()
    pool.block_tables[0, 3] = -1
    pool.mass.copy_(before)
    run(q)
    m = dense(pool, pool.mass[0], 1, 100)
    assert (m >= dense(pool, before[0], 1, 100)).all() and torch.isfinite(pool.mass).all()
    pool.err.zero_()


def test_out_is_q():
    """The queries as the output: the weights of the queries, not of what the call wrote over them."""
    from snapmind_b200 import PagedKVPool

    for dtype, d in ((torch.bfloat16, 128), (torch.float32, 64)):
        pool = PagedKVPool(1, 2, d, 64, max_seqs=2, max_blocks_per_seq=20, dtype=dtype, mass=True)
        g = torch.Generator(device="cuda").manual_seed(8)
        pool.reserve_each([200, 100])
        fill(pool, g)
        q = torch.randn((9, 8, d), generator=g, device="cuda").to(dtype)
        cu = torch.tensor([0, 7, 9], dtype=torch.int32, device="cuda")
        before = pool.mass.clone()
        out = pool.attend_chunk(0, q, cu, accumulate=True)
        mass = pool.mass.clone()
        pool.mass.copy_(before)
        x = q.clone()
        pool.attend_chunk(0, x, cu, out=x, accumulate=True)
        assert torch.equal(x, out) and torch.equal(pool.mass, mass)


def test_a_long_sequence():
    """Lengths whose weights do not fit shared memory at once, few of them apart, ties over the chunks' borders."""
    from snapmind_b200 import PagedKVPool

    n = 120001
    pool = PagedKVPool(1, 1, 64, n // 64 + 3, max_seqs=1, max_blocks_per_seq=n // 64 + 3, block_size=64, mass=True)
    pool.reserve(n)
    g = torch.Generator(device="cuda").manual_seed(9)
    fill(pool, g, "ties")
    m = dense(pool, pool.mass[0], 0, n).cpu().numpy()
    rows = dense(pool, pool.k[0], 0, n).clone()
    budget = 90000
    kept = pool.evict(budget, recent=1000, sinks=7)
    order = np.argsort(-m[0].astype(np.float64) - 10.0 * ((np.arange(n) < 7) | (np.arange(n) >= n - 1000)), kind="stable")
    want = np.sort(order[:budget])
    assert (kept[0, 0, 0].cpu().numpy() == want).all()
    assert torch.equal(dense(pool, pool.k[0], 0, budget), rows[:, torch.from_numpy(want).cuda()])
    q = torch.randn((1, 4, 64), generator=g, device="cuda").bfloat16()
    pool.mass.zero_()
    pool.decode(0, q, accumulate=True)
    w, tol = reference_mass(q, dense(pool, pool.k[0], 0, budget).double(), 0, 0, 64 ** -0.5)
    assert ((dense(pool, pool.mass[0], 0, budget).double() - w).abs() <= tol + 1e-30).all()
    assert kept_of(m[:, :50], 20, 3, 2).shape == (1, 20)


def test_the_whole_step_in_one():
    """append_rope, attend_chunk with weights and evict over many sequences, twice over: positions run on past evictions."""
    from snapmind_b200 import PagedKVPool

    from test_norm_rope_gpu import reference as rotated, tables as rope_tables

    hq, hkv, d, budget = 8, 2, 128, 48
    cos, sin = rope_tables(512, d)
    pool = PagedKVPool(1, hkv, d, 40, max_seqs=2, max_blocks_per_seq=12, dtype=torch.float32, mass=True)
    g = torch.Generator(device="cuda").manual_seed(10)
    w = [1 + 0.2 * torch.randn(d, generator=g, device="cuda") for _ in range(2)]
    at = np.zeros(2, np.int64)
    held = [torch.zeros((hkv, 0, d), dtype=torch.float64, device="cuda") for _ in range(2)]
    for new in ([70, 20], [5, 40], [1, 1]):
        pool.reserve_each(new)
        total = sum(new)
        q, k, v = (torch.randn((total, h, d), generator=g, device="cuda") for h in (hq, hkv, hkv))
        pos = torch.cat([torch.arange(a, a + n, device="cuda") for a, n in zip(at, new)])
        at += new
        cu = torch.tensor([0, new[0], total], dtype=torch.int32, device="cuda")
        qr = pool.append_rope(0, q, k, v, cos, sin, pos, cu_new=cu, q_norm=w[0], k_norm=w[1])
        pool.attend_chunk(0, qr, cu, accumulate=True)
        z, tol = rotated(k, w[1], cos, sin, pos, 1e-6)
        i = 0
        for b in range(2):
            n = int(pool.host_lens[b])
            got = dense(pool, pool.k[0], b, n).double()
            fresh = z[i:i + new[b]].transpose(0, 1)
            assert torch.equal(got[:, :n - new[b]], held[b])
            assert ((got[:, n - new[b]:] - fresh).abs() <= 2 * tol[i:i + new[b]].transpose(0, 1) + 2.0**-23 * fresh.abs()).all()
            held[b] = got
            i += new[b]
        m = [dense(pool, pool.mass[0], b, int(pool.host_lens[b])).cpu().numpy() for b in range(2)]
        pool.evict(budget, recent=8, sinks=2)
        for b in range(2):
            idx = torch.from_numpy(kept_of(m[b], budget, 8, 2)).cuda()
            held[b] = torch.gather(held[b], 1, idx.unsqueeze(-1).expand(-1, -1, d))
    pool.check()
