"""Attention that accumulates its weights, and eviction by them, against the formulas in 64 bits.

Tolerances (before any run).  With u = 2^-24, a score (D products in f32, in any order, the tensor core's sums
among them, the scale and log2 e folded in) is off by at most ds = 2 (D + 4) u scale sum_d |q_d k_d|, a weight's
numerator 2^(s - x) by a relative ds + 2^-21 (the subtraction, 2^x), and its 1 / sum by as much and n u.  So
a weight of the pass over the scores is off by a relative 4 ds + 2^-19 + 2 n u (both passes' scores), and a sum of
N weights on top of what was there by N u of it.  Kept indexes are exact; rows and weights move as bits."""
import numpy as np
import pytest
import torch

from test_chunk_gpu import DT, check, fp32_weights, make_pool, visible

pytestmark = pytest.mark.gpu

U = 2.0**-24


def reference_mass(q, k, window, sinks, scale):
    """(sum of weights [hkv, n], tolerance) of one sequence: q [t, hq, d], k [hkv, n, d]."""
    t, hq, d = q.shape
    hkv, n, _ = k.shape
    qd = q.double().view(t, hkv, hq // hkv, d).permute(1, 2, 0, 3)
    ok = visible(n, t, window, sinks)
    s = torch.einsum("hgtd,hnd->hgtn", qd, k) * scale
    sa = torch.einsum("hgtd,hnd->hgtn", qd.abs(), k.abs()).masked_fill(~ok, 0).amax(-1, keepdim=True) * abs(scale)
    m = s.masked_fill(~ok, -torch.inf).amax(-1, keepdim=True)
    p = torch.where(ok, torch.exp(s - torch.where(torch.isfinite(m), m, 0.0)), 0.0)
    z = p.sum(-1, keepdim=True)
    p = torch.where(z > 0, p / z, 0.0)
    rel = 4 * (2 * (d + 4) * U * sa) + 2.0**-19 + 2 * n * U
    rows = t * (hq // hkv)
    return p.sum((1, 2)), (p * rel).sum((1, 2)) + rows * U * p.sum((1, 2))


def dense(pool, x, b, n):
    """[heads, n, ...] of a paged tensor [blocks, heads, slots, ...] of sequence b."""
    bs = pool.block_size
    j = torch.arange(n, device="cuda")
    blocks = pool.block_tables[b].long()[j // bs]
    return x[blocks, :, j % bs].transpose(0, 1)


CASES = [
    # dtype, cache, hq, hkv, d, bs, lens, new (None: a decode), window, sinks
    ("f32", "same", 32, 4, 64, 16, [256, 40], [256, 17], 0, 0),
    ("f32", "same", 6, 2, 40, 12, [70, 1, 0, 33], [5, 1, 0, 33], 0, 0),
    ("f32", "same", 2, 2, 256, 16, [130], [130], 31, 3),
    ("f32", "e4m3", 8, 2, 96, 16, [90, 200], [3, 70], 64, 5),
    ("bf16", "same", 32, 8, 128, 16, [700, 129, 128, 64, 1], [130, 1, 128, 64, 1], 0, 0),
    ("bf16", "same", 32, 8, 128, 16, [3000, 517], [67, 517], 512, 4),
    ("bf16", "same", 32, 8, 128, 64, [2049, 777], [600, 3], 0, 0),
    ("bf16", "same", 12, 4, 128, 32, [1000, 333], [257, 333], 100, 40),
    ("bf16", "same", 71, 1, 64, 16, [500, 90], [9, 90], 0, 0),
    ("bf16", "same", 130, 1, 128, 16, [300], [5], 0, 0),
    ("bf16", "same", 16, 1, 128, 16, [260, 20], [70, 20], 17, 33),
    ("bf16", "same", 8, 8, 96, 16, [100, 260], [30, 4], 0, 0),
    ("bf16", "same", 8, 2, 64, 8, [400, 15], [100, 15], 1, 0),
    ("bf16", "same", 8, 2, 128, 256, [900, 15], [100, 15], 300, 2),
    ("f16", "same", 32, 8, 128, 16, [900, 0, 77], [257, 0, 12], 0, 0),
    ("f16", "same", 8, 1, 64, 32, [1500, 5], [300, 5], 200, 9),
    ("f16", "e4m3", 32, 8, 128, 16, [900, 400], [100, 400], 0, 0),
    ("bf16", "e4m3", 32, 8, 128, 16, [900, 400], [100, 3], 300, 6),
    ("bf16", "e4m3", 8, 2, 64, 32, [333, 400], [100, 1], 0, 0),
    ("bf16", "same", 32, 8, 128, 16, [700, 1, 0, 4097, 64], None, 0, 0),
    ("bf16", "same", 32, 8, 128, 16, [3000, 517, 5], None, 512, 4),
    ("f16", "same", 24, 8, 128, 32, [1000, 65], None, 0, 0),
    ("bf16", "same", 5, 5, 128, 64, [1000, 65], None, 0, 0),
    ("bf16", "same", 16, 2, 128, 128, [1000, 65], None, 100, 1),
    ("bf16", "same", 32, 4, 64, 16, [700, 33], None, 0, 0),
    ("f32", "same", 32, 4, 64, 16, [700, 33], None, 0, 0),
    ("f16", "e4m3", 32, 8, 128, 16, [900, 0, 401], None, 0, 0),
    ("bf16", "e4m3", 14, 2, 128, 32, [900, 401], None, 90, 3),
    ("f32", "e4m3", 4, 2, 80, 16, [90, 41], None, 0, 0),
    ("bf16", "same", 8, 2, 128, 512, [4000, 700], [40, 3], 500, 3),  # tiles of a sink block that nobody sees
    ("bf16", "e4m3", 8, 2, 128, 1024, [4000, 700], [40, 3], 500, 3),
    ("bf16", "same", 6, 1, 128, 16, [4000], [1200], 0, 0),  # heads that do not divide a step, many steps of whole rows
    ("f16", "same", 4, 1, 64, 16, [3000, 100], [900, 100], 700, 5),
    ("bf16", "same", 300, 1, 64, 16, [500], [4], 0, 0),  # several slices of heads
    # decodes that another kernel than the one that keeps its scores takes
    ("bf16", "same", 8, 2, 128, 8, [300, 20], None, 0, 0),
    ("bf16", "same", 8, 2, 128, 24, [300, 20], None, 0, 0),
    ("bf16", "same", 32, 2, 128, 16, [300, 1000], None, 200, 4),
    ("f16", "e4m3", 32, 2, 128, 16, [300, 1000], None, 0, 0),
]


def call(pool, q, cu, window, sinks, **kw):
    if cu is None:
        return pool.decode(0, q, window=window, sinks=sinks, **kw)
    return pool.attend_chunk(0, q, cu, window=window, sinks=sinks, **kw)


def setup(case, seed=3, values=False):
    dtype, cache, hq, hkv, d, bs, lens, new, window, sinks = case
    pool, ks, vs = make_pool(DT[dtype], lens, hkv, d, bs, seed, cache)
    g = torch.Generator(device="cuda").manual_seed(seed)
    pool.mass = torch.rand((1, pool.num_blocks, hkv, bs), generator=g, device="cuda")
    counts = [1] * len(lens) if new is None else new
    q = torch.randn((sum(counts), hq, d), generator=g, device="cuda").to(DT[dtype])
    cu = None if new is None else torch.tensor([0] + list(np.cumsum(new)), dtype=torch.int32, device="cuda")
    return (pool, ks, q, cu, counts, vs) if values else (pool, ks, q, cu, counts)


def check_mass(pool, before, ks, q, counts, window, sinks, scale):
    seen = torch.zeros(pool.mass.shape[1:], dtype=torch.bool, device="cuda")
    at = 0
    for b, (k, t) in enumerate(zip(ks, counts)):
        n = k.shape[1]
        if n and t:
            want, tol = reference_mass(q[at:at + t], k, window, sinks, scale)
            old = dense(pool, before[0], b, n).double()
            got = dense(pool, pool.mass[0], b, n).double()
            tol = tol + 2 * U * (old + want) + 1e-30
            err = (got - old - want).abs()
            assert (err <= tol).all(), f"sequence {b}: {float((err / tol).max()):.2f} x the tolerance"
            bs = pool.block_size
            j = torch.arange(n, device="cuda")
            seen[pool.block_tables[b].long()[j // bs], :, j % bs] = True
        at += t
    assert torch.equal(pool.mass[0][~seen], before[0][~seen])  # slots without a token


@pytest.mark.parametrize("generic", [False, True])
@pytest.mark.parametrize("case", CASES, ids=[f"{i}" for i in range(len(CASES))])
def test_accumulated_weights(case, generic):
    window, sinks = case[-2:]
    pool, ks, q, cu, counts, vs = setup(case, values=True)
    before = pool.mass.clone()
    plain = call(pool, q, cu, window, sinks, force_generic=generic)
    assert torch.equal(pool.mass, before)
    out = call(pool, q, cu, window, sinks, force_generic=generic, accumulate=True)
    pool.check()
    if cu is not None:
        assert torch.equal(out, plain)
    else:  # the weights of a bf16 decode that accumulates are off by 2^-16 (two bf16 terms), others' by their type's half step
        two = case[:2] == ("bf16", "same") and case[4] == 128 and case[2] // case[3] <= 8 and case[5] in (16, 32, 64, 128)
        half = 0.0 if generic else 2.0**-16 if two else fp32_weights(q.dtype)
        check(out, q, np.cumsum([0, *counts]).tolist(), ks, vs, window, sinks, half if case[1] == "same" else max(half, 2.0**-11))
    check_mass(pool, before, ks, q, counts, window, sinks, q.shape[-1] ** -0.5)
    # the same bits every time
    first = pool.mass.clone()
    pool.mass.copy_(before)
    call(pool, q, cu, window, sinks, force_generic=generic, accumulate=True)
    assert torch.equal(pool.mass, first)


@pytest.mark.parametrize("scale", [-0.2, 0.0, 1.5])
@pytest.mark.parametrize("case", [CASES[4], CASES[16], CASES[19], CASES[0]], ids=["chunk", "quant", "decode", "f32"])
def test_scales(case, scale):
    window, sinks = case[-2:]
    pool, ks, q, cu, counts = setup(case)
    before = pool.mass.clone()
    call(pool, q, cu, window, sinks, scale=scale, accumulate=True)
    check_mass(pool, before, ks, q, counts, window, sinks, scale)


def test_rows_that_f16_does_not_hold():
    """f16 queries over 8-bit rows of V past f16's range: the call is done over in f32, and its statistics count."""
    case = ("f16", "e4m3", 8, 2, 128, 16, [700, 90], [130, 7], 0, 0)
    pool, ks, q, cu, counts = setup(case)
    pool.scales[0, pool.block_tables[0, 3].item(), 1, 1, 5] = 127 + 30
    before = pool.mass.clone()
    pool.attend_chunk(0, q, cu, accumulate=True)
    pool.check()
    check_mass(pool, before, ks, q, counts, 0, 0, 128 ** -0.5)


# ------------------------------------------------------------------ eviction
def kept_of(mass, budget, recent, sinks):
    """[heads, kept] indexes of one (layer, sequence): plain, in order of (forced, weight, lowest index)."""
    heads, n = mass.shape
    if n <= budget:
        return np.tile(np.arange(n), (heads, 1))
    got = []
    for h in range(heads):
        forced = set(range(min(sinks, n))) | set(range(n - recent, n))
        rest = sorted((j for j in range(n) if j not in forced),
                      key=lambda j: (-(np.inf if np.isnan(mass[h, j]) else float(mass[h, j])), not np.isnan(mass[h, j]), j))
        got.append(sorted(forced | set(rest[:budget - len(forced)])))
    return np.array(got)


EVICT = [
    # dtype, cache, layers, hkv, d, bs, lens, budget, recent, sinks
    ("bf16", "same", 2, 4, 128, 16, [700, 129, 128, 64, 1, 0], 128, 16, 4),
    ("bf16", "same", 1, 2, 64, 16, [1000], 1, 0, 0),
    ("bf16", "same", 1, 2, 64, 16, [1000], 1, 1, 0),
    ("bf16", "same", 1, 2, 64, 16, [1000, 998], 997, 900, 97),
    ("f16", "same", 3, 1, 40, 12, [77, 300, 12], 33, 0, 0),
    ("f32", "same", 1, 3, 9, 5, [77, 31], 30, 7, 3),
    ("f16", "same", 1, 1, 9, 16, [300], 100, 10, 0),
    ("bf16", "e4m3", 2, 4, 128, 16, [700, 129, 33], 100, 31, 4),
    ("f32", "e4m3", 1, 2, 72, 8, [200, 129], 100, 0, 1),
    ("bf16", "same", 1, 2, 128, 16, [20000, 8195, 8300], 3000, 64, 4),
    ("bf16", "same", 1, 1, 128, 64, [20000], 15000, 100, 0),
    ("f32", "same", 1, 2, 256, 256, [3000], 700, 100, 9),
]


def weights(shape, g, kind):
    if kind == "ties":
        return torch.randint(0, 3, shape, generator=g, device="cuda").float()
    if kind == "equal":
        return torch.full(shape, 0.25, device="cuda")
    x = torch.empty(shape, device="cuda").exponential_(generator=g)
    if kind == "odd":
        r = torch.rand(shape, generator=g, device="cuda")
        x = torch.where(r < 0.05, torch.full_like(x, float("nan")), x)
        x = torch.where((r > 0.05) & (r < 0.1), torch.full_like(x, float("inf")), x)
        x = torch.where((r > 0.1) & (r < 0.2), -x, x)
        x = torch.where(r > 0.98, torch.full_like(x, float("-inf")), x)
        x = torch.where((r > 0.2) & (r < 0.3), x * 1e-42, x)
        x = torch.where((r > 0.3) & (r < 0.32), torch.zeros_like(x), x)
        x = torch.where((r > 0.32) & (r < 0.34), -torch.zeros_like(x), x)
    return x


def bits(x):
    return x.contiguous().view(torch.uint8)


def run_evict(case, kind, into, seed=5):
    dtype, cache, layers, hkv, d, bs, lens, budget, recent, sinks = case
    n = len(lens)
    kept_blocks = sum((min(x, budget) + bs - 1) // bs for x in lens)
    from snapmind_b200 import PagedKVPool, QuantizedKVPool

    g = torch.Generator(device="cuda").manual_seed(seed)
    rng = np.random.RandomState(seed)
    blocks = [(x + bs - 1) // bs for x in lens]
    nb = sum(blocks) + 5 + (kept_blocks if into else 0)
    perm = rng.permutation(nb)
    width = max(max(blocks), 1) + 1
    rows = 2 * n if into else n
    tables = np.zeros((rows, width), np.int64)
    at = 0
    for b, x in enumerate(blocks):
        tables[b, :x] = perm[at:at + x]
        at += x
    lens_all = list(lens) + [0] * (rows - n)
    if into and n > 1:  # a target that holds something already
        tables[n, :2] = perm[at:at + 2]
        at += 2
        lens_all[n] = bs + 1
    cls = QuantizedKVPool if cache == "e4m3" else PagedKVPool
    pool = cls(layers, hkv, d, nb, max_seqs=rows, max_blocks_per_seq=width, block_size=bs, dtype=DT[dtype], mass=True)
    pool.set_state(tables, np.array(lens_all), perm[at:])
    for t in (pool.k, pool.v) + ((pool.scales,) if cache == "e4m3" else ()):
        t.view(torch.uint8).copy_(torch.randint(0, 256, t.view(torch.uint8).shape, generator=g, device="cuda", dtype=torch.int32).to(torch.uint8))
    pool.mass.copy_(weights(pool.mass.shape, g, kind))
    held = {x: getattr(pool, x).clone() for x in ("k", "v", "mass")}
    scales = pool.scales.clone() if cache == "e4m3" else None
    want = {}
    for layer in range(layers):
        for b, x in enumerate(lens):
            m = dense(pool, held["mass"][layer], b, x).cpu().numpy()
            want[layer, b] = kept_of(m, budget, recent, sinks)
    old_tables = pool.block_tables.clone()
    if into:
        kept = pool.evict(budget, recent=recent, sinks=sinks, seqs=list(range(n)), into=list(range(n, 2 * n)))
    else:
        kept = pool.evict(budget, recent=recent, sinks=sinks)
    pool.check()
    ends = [min(x, budget) for x in lens]
    assert pool.seq_lens.tolist() == (list(lens) + ends if into else ends)
    assert list(pool.host_lens) == pool.seq_lens.tolist()
    assert int(pool.free_top) == pool._host_free == nb - sum((x + bs - 1) // bs for x in pool.host_lens)
    # no block is held twice
    ids = pool.free_stack[:int(pool.free_top)].tolist()
    for b, x in enumerate(pool.host_lens):
        ids += pool.block_tables[b, :(x + bs - 1) // bs].tolist()
    assert sorted(ids) == list(range(nb))
    assert kept.shape == (layers, n, hkv, budget)

    def rows_of(x, b, idx, tab):  # [heads, kept, ...]
        i = torch.from_numpy(idx).cuda()
        h = torch.arange(hkv, device="cuda").view(-1, 1)
        return x[tab[b].long()[i // bs], h, i % bs]

    for layer in range(layers):
        for b, x in enumerate(lens):
            idx = want[layer, b]
            m = idx.shape[1]
            got = kept[layer, b].cpu().numpy()
            assert (got[:, :m] == idx).all() and (got[:, m:] == -1).all()
            to = np.tile(np.arange(m), (hkv, 1))
            t = n + b if into else b
            for name in ("k", "v", "mass"):
                a = rows_of(held[name][layer], b, idx, old_tables)
                z = rows_of(getattr(pool, name)[layer], t, to, pool.block_tables)
                assert torch.equal(bits(a), bits(z)), name
            if scales is not None:
                for kv in range(2):
                    assert torch.equal(rows_of(scales[layer, :, :, kv], b, idx, old_tables),
                                       rows_of(pool.scales[layer, :, :, kv], t, to, pool.block_tables))
            if into:  # the whole stays as it was
                whole = np.tile(np.arange(x), (hkv, 1))
                for name in ("k", "v", "mass"):
                    assert torch.equal(bits(rows_of(held[name][layer], b, whole, old_tables)),
                                       bits(rows_of(getattr(pool, name)[layer], b, whole, pool.block_tables)))


@pytest.mark.parametrize("into", [False, True])
@pytest.mark.parametrize("case", EVICT, ids=[f"{i}" for i in range(len(EVICT))])
def test_evict(case, into):
    run_evict(case, "plain", into)


@pytest.mark.parametrize("kind", ["ties", "equal", "odd"])
@pytest.mark.parametrize("case", [EVICT[0], EVICT[7], EVICT[9]], ids=["b", "q", "long"])
def test_evict_orders(case, kind):
    run_evict(case, kind, False)


def test_evict_refusals():
    from snapmind_b200 import PagedKVPool

    plain = PagedKVPool(1, 2, 64, 32, max_seqs=4, max_blocks_per_seq=8)
    with pytest.raises(ValueError, match="mass"):
        plain.evict(16)
    q = torch.zeros((4, 2, 64), dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError, match="mass"):
        plain.decode(0, q, accumulate=True)
    with pytest.raises(ValueError, match="mass"):
        plain.attend_chunk(0, q, torch.tensor([0, 4], dtype=torch.int32, device="cuda"), accumulate=True)
    pool = PagedKVPool(1, 2, 64, 12, max_seqs=4, max_blocks_per_seq=8, mass=True)
    pool.reserve(80, batch=2)  # 5 blocks each, 2 left
    for kw in (dict(budget=0), dict(budget=8, recent=5, sinks=4), dict(budget=8, recent=-1), dict(budget=8, sinks=-1),
               dict(budget=8, batch=5), dict(budget=8, seqs=[0, 0]), dict(budget=8, seqs=[4]), dict(budget=8, seqs=[-1]),
               dict(budget=8, seqs=[0], batch=1), dict(budget=8, into=[1]), dict(budget=8, seqs=[0], into=[0]),
               dict(budget=8, seqs=[0, 1], into=[2]), dict(budget=8, seqs=[0, 1], into=[1, 2]),
               dict(budget=8, seqs=[0, 1], into=[2, 2])):
        with pytest.raises(ValueError):
            pool.evict(**kw)
    with pytest.raises(RuntimeError, match="out of blocks"):
        pool.evict(40, seqs=[0, 1], into=[2, 3])  # 3 blocks each
    assert list(pool.host_lens) == [80, 80, 0, 0] and pool._host_free == 2
    pool.evict(16, seqs=[0, 1], into=[2, 3])
    assert list(pool.host_lens) == [80, 80, 16, 16] and pool._host_free == 0
    pool.evict(16, seqs=[])
    pool.evict(16, batch=0)
    pool.check()


def test_new_tokens_weigh_nothing():
    """Slots of evicted and released tokens come back with weight 0, and only they."""
    from snapmind_b200 import PagedKVPool

    pool = PagedKVPool(2, 3, 64, 64, max_seqs=3, max_blocks_per_seq=16, mass=True)
    pool.mass.fill_(7.0)
    pool.reserve(20)
    for b in range(3):
        assert (dense(pool, pool.mass[0], b, 20) == 0).all() and (dense(pool, pool.mass[1], b, 20) == 0).all()
    assert int((pool.mass == 0).sum()) == 2 * 3 * 3 * 20
    pool.mass.fill_(5.0)
    pool.reserve_each([3, 0, 40])
    lens = [23, 20, 60]
    for b, fresh in enumerate([3, 0, 40]):
        for layer in range(2):
            m = dense(pool, pool.mass[layer], b, lens[b])
            assert (m[:, lens[b] - fresh:] == 0).all() and (m[:, :lens[b] - fresh] == 5).all()
    pool.reserve_device(2, 2)
    pool.account_host(2, 2)
    assert (dense(pool, pool.mass[1], 1, 22)[:, 20:] == 0).all() and (dense(pool, pool.mass[1], 1, 22)[:, :20] == 5).all()


def test_growing_and_evicting_in_turn_keeps_the_blocks():
    from snapmind_b200 import PagedKVPool

    pool = PagedKVPool(1, 2, 64, 64, max_seqs=3, max_blocks_per_seq=16, mass=True)
    pool.reserve(40)
    held = None
    for _ in range(3):
        pool.reserve(50)
        now = pool.block_tables[:, :6].clone()
        assert held is None or torch.equal(held, now)
        held = now
        pool.evict(40, recent=8)


@pytest.mark.parametrize("cache", ["same", "e4m3"])
def test_a_run_within_a_budget(cache):
    """A pool that takes chunks, attends with accumulated weights and goes back to its budget, against the same steps
    on plain tensors in 64 bits (rows as the pool holds them, weights as it accumulated them)."""
    from snapmind_b200 import PagedKVPool, QuantizedKVPool

    hq, hkv, d, bs, budget, recent, sinks = 8, 2, 128, 16, 64, 12, 3
    cls = QuantizedKVPool if cache == "e4m3" else PagedKVPool
    pool = cls(1, hkv, d, 64, max_seqs=3, max_blocks_per_seq=12, block_size=bs, dtype=torch.bfloat16, mass=True)
    g = torch.Generator(device="cuda").manual_seed(1)
    for step, new in enumerate([[70, 3, 0], [1, 1, 1], [5, 90, 64], [1, 1, 1], [1, 0, 2]]):
        pool.reserve_each(new)
        total = sum(new)
        k, v = (torch.randn((total, hkv, d), generator=g, device="cuda").bfloat16() for _ in range(2))
        q = torch.randn((total, hq, d), generator=g, device="cuda").bfloat16()
        cu = torch.tensor([0] + list(np.cumsum(new)), dtype=torch.int32, device="cuda")
        pool.append_packed(0, k, v, cu)
        before = pool.mass.clone()
        pool.attend_chunk(0, q, cu, accumulate=True)
        kd, vd = pool.gather()
        lens = [int(x) for x in pool.host_lens]
        ks, at = [], 0
        for n in lens:
            ks.append(kd[0, at:at + n * hkv * d].view(hkv, n, d).double())
            at += n * hkv * d
        check_mass(pool, before, ks, q, new, 0, 0, d ** -0.5)
        m = [dense(pool, pool.mass[0], b, n).cpu().numpy() for b, n in enumerate(lens)]
        kept = pool.evict(budget, recent=recent, sinks=sinks)
        kd2, _ = pool.gather()
        at = 0
        for b, n in enumerate(lens):
            idx = kept_of(m[b], budget, recent, sinks)
            assert (kept[0, b, :, :idx.shape[1]].cpu().numpy() == idx).all()
            rows = torch.gather(ks[b], 1, torch.from_numpy(idx).cuda().unsqueeze(-1).expand(-1, -1, d))
            size = rows.numel()
            assert torch.equal(kd2[0, at:at + size].double(), rows.reshape(-1))
            at += size
    pool.check()
