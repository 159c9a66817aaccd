"""Chunk attention over the paged pool, windowed decode with sinks, and the 8-bit pool,
against the formulas in 64 bits.

Tolerances (before any run).  With u = 2^-24, D the head dim and n the visible keys, in f32:
a score's error is at most (D + 4) u scale sum_d |q_d k_d| (D products summed in any order, the
scale and log2 e folded in), that of 2^x at most 2^-21, so a weight is off by a relative
w = 2^-21 + 2 ds, numerator and denominator together by 2 w + 2 n u; the tensor-core kernels
round each weight of the numerator by half a step of its type (bf16 2^-8, f16 2^-11).
All of that multiplies sum_p p |v|; the output's own rounding is half a step of |o|.
A weight below f16's normal range is off by at most 2^-25 of the largest weight."""
import itertools

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
HALF = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}


def fp32_weights(dtype):
    return 0.0 if dtype == torch.float32 else HALF[dtype]


def make_pool(dtype, lens, hkv, d, bs, seed, cache="same", layers=1, spare=0):
    """A shuffled pool whose slots without a token hold NaN; returns (pool, K, V) with K, V
    lists of the sequences' rows [heads, len, dim] in f64 as the pool holds them."""
    from snapmind_b200 import PagedKVPool, QuantizedKVPool

    rng = np.random.RandomState(seed)
    blocks = [(n + bs - 1) // bs for n in lens]
    nb = sum(blocks) + 3 + spare
    perm = rng.permutation(nb)
    width = max(max(blocks), 1) + 2
    tables = np.zeros((len(lens), width), np.int64)
    at = 0
    for b, n in enumerate(blocks):
        tables[b, :n] = perm[at:at + n]
        at += n
    cls = QuantizedKVPool if cache == "e4m3" else PagedKVPool
    pool = cls(layers, hkv, d, nb, max_seqs=len(lens), max_blocks_per_seq=width, block_size=bs, dtype=dtype)
    pool.set_state(tables, np.array(lens), perm[at:])
    g = torch.Generator(device="cuda").manual_seed(seed)
    holds = torch.zeros((nb, bs), dtype=torch.bool)
    for b, n in enumerate(lens):
        row = torch.zeros(blocks[b] * bs, dtype=torch.bool)
        row[:n] = True
        holds[tables[b, :blocks[b]]] = row.view(blocks[b], bs)
    empty = ~holds.cuda().view(nb, 1, bs, 1)
    kv = []
    for l in range(layers):
        for i, t in enumerate((pool.k, pool.v)):
            x = torch.randn((nb, hkv, bs, d), generator=g, device="cuda")
            if cache == "e4m3":
                codes = (x * 100).clamp(-448, 448).to(torch.float8_e4m3fn)
                codes.view(torch.uint8).masked_fill_(empty, 0x7F)
                t[l].view(torch.uint8).copy_(codes.view(torch.uint8))
                e = torch.randint(-9, -5, (nb, hkv, bs), generator=g, device="cuda")
                pool.scales[l, :, :, i] = torch.where(empty[..., 0].expand_as(e), torch.full_like(e, 255), e + 127).to(torch.uint8)
                val = codes.double() * torch.exp2(e.double()).unsqueeze(-1)
            else:
                t[l].copy_(x.masked_fill_(empty, float("nan")))
                val = t[l].double()
            if l == layers - 1:
                kv.append([val[torch.from_numpy(tables[b, :blocks[b]]).cuda()].permute(1, 0, 2, 3).reshape(hkv, -1, d)[:, :n]
                           for b, n in enumerate(lens)])
    return pool, kv[0], kv[1]


def visible(n, t, window, sinks):
    i = torch.arange(n - t, n, device="cuda").view(t, 1)
    j = torch.arange(n, device="cuda").view(1, n)
    ok = j <= i
    if window:
        ok = ok & ((j > i - window) | (j < sinks))
    return ok


def reference(q, k, v, window, sinks, weight_half, scale=None):
    """(o, tolerance) of one sequence: q [t, hq, d], k and v [hkv, n, d], in f64."""
    t, hq, d = q.shape
    hkv, n, _ = k.shape
    scale = d ** -0.5 if scale is None else scale
    q = q.double().view(t, hkv, hq // hkv, d).permute(1, 2, 0, 3)  # [hkv, G, t, d]
    ok = visible(n, t, window, sinks)
    o = torch.zeros((t, hq, d), dtype=torch.float64, device="cuda")
    tol = torch.zeros_like(o)
    if n == 0:
        return o, tol
    for h in range(hkv):
        s = torch.einsum("gtd,nd->gtn", q[h], k[h]) * scale
        sa = torch.einsum("gtd,nd->gtn", q[h].abs(), k[h].abs()).masked_fill(~ok, 0).amax(-1, keepdim=True) * scale
        m = s.masked_fill(~ok, -torch.inf).amax(-1, keepdim=True)
        p = torch.where(ok, torch.exp(s - torch.where(torch.isfinite(m), m, 0.0)), 0.0)
        z = p.sum(-1, keepdim=True)
        p = torch.where(z > 0, p / z, 0.0)
        oh = torch.einsum("gtn,nd->gtd", p, v[h])
        oa = torch.einsum("gtn,nd->gtd", p, v[h].abs())
        u = 2.0**-24
        w = 2.0**-21 + 2 * (d + 4) * u * sa
        top = torch.where(z > 0, 1 / z, 0.0) * (ok.double() @ v[h].abs())
        rel = oa * (2 * w + 2 * n * u + weight_half) + 2.0**-25 * top * (weight_half > 0)
        g = hq // hkv
        o[:, h * g:(h + 1) * g] = oh.permute(1, 0, 2)
        tol[:, h * g:(h + 1) * g] = rel.permute(1, 0, 2)
    return o, tol


def check(out, q, cu, ks, vs, window, sinks, weight_half, scale=None):
    assert torch.isfinite(out[: cu[-1]]).all()
    for b in range(len(ks)):
        if cu[b + 1] == cu[b]:
            continue
        o, tol = reference(q[cu[b]:cu[b + 1]], ks[b], vs[b], window, sinks, weight_half, scale)
        err = (out[cu[b]:cu[b + 1]].double() - o).abs()
        tol = tol + HALF[out.dtype] * o.abs() * (1 + 2.0**-6) + 1e-30
        if out.dtype == torch.float16:
            tol = tol + 2.0**-25
        bad = err > tol
        assert not bad.any(), f"sequence {b}: worst {float((err / tol).max()):.2f} x the tolerance, {int(bad.sum())} values"


CASES = [
    # dtype, cache, hq, hkv, d, bs, lens, new, window, sinks
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
    ("f16", "same", 32, 8, 128, 16, [1500, 300], [300, 40], 1024, 4),
    ("f16", "same", 15, 5, 64, 32, [640, 641], [1, 64], 0, 0),
    ("bf16", "e4m3", 32, 8, 128, 16, [900, 130, 1, 257], [200, 130, 1, 2], 0, 0),
    ("bf16", "e4m3", 16, 4, 64, 32, [600, 70], [31, 70], 128, 20),
    ("f16", "e4m3", 12, 2, 128, 64, [800, 64], [90, 64], 200, 1),
    ("bf16", "e4m3", 7, 7, 128, 16, [140], [139], 0, 0),
    ("bf16", "e4m3", 6, 2, 80, 16, [140, 50], [20, 50], 30, 4),
]


@pytest.mark.parametrize("generic", [False, True])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(x) for x in c[:6]))
def test_chunk(cuda_device, case, generic):
    dtype, cache, hq, hkv, d, bs, lens, new, window, sinks = case
    dtype = DT[dtype]
    pool, ks, vs = make_pool(dtype, lens, hkv, d, bs, 11, cache)
    g = torch.Generator(device="cuda").manual_seed(5)
    cu = [0] + list(np.cumsum(new))
    # a strided view with two rows behind the last sequence, which stay as they are
    q = (1.5 * torch.randn((cu[-1] + 2, hq + 3, d), generator=g, device="cuda")).to(dtype)[:, 1:hq + 1]
    out = torch.full((cu[-1] + 2, hq, d), 7.0, dtype=dtype, device="cuda")
    cud = torch.tensor(cu, dtype=torch.int32, device="cuda")
    got = pool.attend_chunk(0, q, cud, out=out, window=window, sinks=sinks, force_generic=generic)
    assert got is out
    pool.check()
    check(out, q, cu, ks, vs, window, sinks, fp32_weights(dtype))
    assert (out[cu[-1]:] == 7.0).all()


DECODE = [
    ("bf16", "same", 32, 8, 128, 16, [5000, 1, 64, 0, 1023, 2100], 1024, 4),
    ("bf16", "same", 32, 8, 128, 16, [700, 65, 16], 16, 0),
    ("f16", "same", 8, 8, 128, 64, [900, 1200, 63], 100, 70),
    ("f16", "same", 64, 8, 128, 32, [3000], 1, 1),
    ("bf16", "same", 48, 4, 128, 16, [300, 20], 50, 4),
    ("bf16", "same", 32, 4, 64, 16, [300, 20], 50, 4),
    ("f32", "same", 32, 4, 64, 16, [300, 20, 1], 50, 4),
    ("bf16", "e4m3", 32, 8, 128, 16, [5000, 1, 64, 0, 1023], 0, 0),
    ("bf16", "e4m3", 32, 8, 128, 32, [2000, 17, 64], 300, 5),
    ("f16", "e4m3", 12, 2, 128, 64, [2000, 17, 640], 0, 0),
    ("f16", "e4m3", 12, 2, 64, 16, [2000, 17, 640], 0, 0),
    ("f32", "e4m3", 12, 2, 128, 16, [200, 17, 64], 0, 0),
]


@pytest.mark.parametrize("generic", [False, True])
@pytest.mark.parametrize("case", DECODE, ids=lambda c: "-".join(str(x) for x in c[:6]))
def test_decode(cuda_device, case, generic):
    dtype, cache, hq, hkv, d, bs, lens, window, sinks = case
    dtype = DT[dtype]
    pool, ks, vs = make_pool(dtype, lens, hkv, d, bs, 3, cache)
    g = torch.Generator(device="cuda").manual_seed(6)
    q = (1.5 * torch.randn((len(lens), hq, d), generator=g, device="cuda")).to(dtype)
    out = pool.decode(0, q, window=window, sinks=sinks, force_generic=generic)
    pool.check()
    cu = list(range(len(lens) + 1))
    half = fp32_weights(dtype)
    check(out, q, cu, ks, vs, window, sinks, half)
    for b, n in enumerate(lens):
        if n == 0:
            assert (out[b] == 0).all()


def test_decode_equals_plain_decode_inside_the_window(cuda_device):
    """A window that covers every sequence gives what the decode without one gives (both within tolerance)."""
    pool, ks, vs = make_pool(torch.bfloat16, [400, 77], 8, 128, 16, 9)
    q = torch.randn((2, 32, 128), device="cuda").bfloat16()
    a, b = pool.decode(0, q), pool.decode(0, q, window=1 << 30, sinks=7)
    check(a, q, [0, 1, 2], ks, vs, 0, 0, 2.0**-8)
    check(b, q, [0, 1, 2], ks, vs, 0, 0, 2.0**-8)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_query_scales(cuda_device, dtype):
    """Queries and cache rows far from one: 8-bit decodes keep them (a row's exponent, a query's range)."""
    dtype = DT[dtype]
    lens = [130, 260]
    pool, ks, vs = make_pool(dtype, lens, 2, 128, 16, 21, "e4m3")
    e = torch.randint(-12, 4, pool.scales.shape, device="cuda")
    keep = pool.scales == 255
    pool.scales.copy_(torch.where(keep, pool.scales, (e + 127).to(torch.uint8)))
    val = [x.double() * torch.exp2(e[:, :, :, i].double()).unsqueeze(-1) for i, x in enumerate((pool.k, pool.v))]
    tables = pool.block_tables.long()
    ks, vs = [[x[0][tables[b, :(n + 15) // 16]].permute(1, 0, 2, 3).reshape(2, -1, 128)[:, :n] for b, n in enumerate(lens)]
              for x in val]
    for size in (1e-4, 30.0):
        q = (size * torch.randn((2, 8, 128), device="cuda")).to(dtype)
        scale = 0.002 / size
        check(pool.decode(0, q, scale=scale), q, [0, 1, 2], ks, vs, 0, 0, fp32_weights(dtype), scale)
        cu = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
        check(pool.attend_chunk(0, q, cu, scale=scale), q, [0, 1, 2], ks, vs, 0, 0, fp32_weights(dtype), scale)


def quantise64(x):
    """Values, exponents of rows by the definition, in f64."""
    x = x.double()
    a = torch.where(torch.isfinite(x), x.abs(), 0.0).amax(-1)
    e = torch.full_like(a, -100.0)
    for cand in range(-99, 121):
        e = torch.where(a > 448.0 * 2.0 ** (cand - 1), float(cand), e)
    y = x / torch.exp2(e).unsqueeze(-1)
    _, k = torch.frexp(y)
    grid = torch.exp2((k - 4).clamp(min=-9).double())
    y = torch.round(y / grid) * grid
    y = torch.where(torch.isfinite(x), y, torch.nan)
    return y * torch.exp2(e).unsqueeze(-1), e


@pytest.mark.parametrize("src", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("hkv,d,bs,T", [(8, 128, 16, 37), (4, 64, 32, 1), (3, 40, 16, 5), (2, 256, 64, 130)])
def test_quantised_rows_and_read_back(cuda_device, src, hkv, d, bs, T):
    from snapmind_b200 import QuantizedKVPool

    B, L = 3, 2
    pool = QuantizedKVPool(L, hkv, d, 40, B, 12, block_size=bs, dtype=DT[src])
    pool.reserve(T, batch=B)
    x = torch.randn((2, L, B, hkv, T, d), device="cuda") * torch.exp2(torch.randint(-20, 8, (2, L, B, hkv, T, 1), device="cuda").float())
    x[0, 0, 0, 0, 0] = 0
    x[1, 0, 0, 0, 0, 0] = 448.0
    x[1, 0, 0, 0, 0, 1:] = torch.arange(1, d, device="cuda") * 0.5  # ties among them
    x = x.to(DT[src])
    pool.append(None, x[0], x[1])
    got = pool.gather(batch=B)
    pool.check()
    for i in range(2):
        want, e = quantise64(x[i])
        top = torch.finfo(DT[src]).max
        want = want.clamp(-top, top).to(DT[src])  # exact in bf16 and f32; one rounding below f16's normal range
        assert torch.equal(got[i].view(L, B, hkv, T, d), want)
        # the stored bytes themselves
        for b, t in itertools.product(range(B), {0, T // 2, T - 1}):
            blk = int(pool.block_tables[b, t // bs])
            assert torch.equal(pool.scales[:, blk, :, i, t % bs].double() - 127, e[:, b, :, t])


def test_quantised_extremes(cuda_device):
    from snapmind_b200 import QuantizedKVPool

    pool = QuantizedKVPool(1, 1, 64, 4, 1, 4, dtype=torch.float32)
    pool.reserve(5, batch=1)
    x = torch.zeros((1, 1, 5, 64), device="cuda")
    x[0, 0, 0, :3] = torch.tensor([float("nan"), float("inf"), 2.0])
    x[0, 0, 1, :2] = torch.tensor([3.4e38, -3.4e38])
    x[0, 0, 2, :2] = torch.tensor([1e-40, -1e-35])
    x[0, 0, 3, :2] = torch.tensor([449.0, 448.0])
    x[0, 0, 4, :3] = torch.tensor([1.0, 2.0**-9 * 1.5, -2.0**-18])
    pool.append(0, x, x)
    k, v = pool.gather()
    pool.check()
    want, e = quantise64(x[0, 0])
    top = torch.finfo(torch.float32).max
    assert torch.equal(torch.nan_to_num(k.view(5, 64).double(), nan=123.0), torch.nan_to_num(want.clamp(-top, top), nan=123.0))
    assert torch.equal(pool.scales[0, int(pool.block_tables[0, 0]), 0, 1, :5].double() - 127, e)
    half = QuantizedKVPool(1, 1, 64, 4, 1, 4, dtype=torch.float16)
    half.reserve(1, batch=1)
    y = torch.full((1, 1, 1, 64), 65504.0, device="cuda").half()
    half.append(0, y, -y)
    k, v = half.gather()
    assert (k == 65504.0).all() and (v == -65504.0).all()  # 65536 held to f16's largest


@pytest.mark.parametrize("cache,dtype", [("same", "bf16"), ("same", "f32"), ("e4m3", "bf16"), ("e4m3", "f32")])
def test_a_run_of_steps(cuda_device, cache, dtype):
    """Prompts in ragged pieces, then single tokens, through reserve_each, append_packed,
    attend_chunk and decode, two layers, against the whole history."""
    from snapmind_b200 import PagedKVPool, QuantizedKVPool

    dtype = DT[dtype]
    B, hq, hkv, d, bs, L = 3, 8, 2, 128, 16, 2
    cls = QuantizedKVPool if cache == "e4m3" else PagedKVPool
    pool = cls(L, hkv, d, 120, B, 40, block_size=bs, dtype=dtype)
    g = torch.Generator(device="cuda").manual_seed(1)
    hist = [[[torch.zeros((hkv, 0, d), dtype=torch.float64, device="cuda") for _ in range(B)] for _ in range(2)] for _ in range(L)]
    for new in ([40, 0, 7], [1, 130, 1], [33, 1, 0], [1, 1, 1]):
        total = sum(new)
        pool.reserve_each(new)
        cu = [0] + list(np.cumsum(new))
        cud = torch.tensor(cu, dtype=torch.int32, device="cuda")
        kn, vn = (torch.randn((L, total, hkv, d), generator=g, device="cuda").to(dtype) for _ in range(2))
        q = torch.randn((L, total, hq, d), generator=g, device="cuda").to(dtype)
        pool.append_packed(None, kn, vn, cud)
        for l in range(L):
            for i, x in enumerate((kn, vn)):
                val = quantise64(x[l])[0] if cache == "e4m3" else x[l].double()
                for b in range(B):
                    hist[l][i][b] = torch.cat([hist[l][i][b], val[cu[b]:cu[b + 1]].transpose(0, 1)], 1)
            for window, sinks in ((0, 0), (25, 4)):
                out = pool.attend_chunk(l, q[l], cud, window=window, sinks=sinks)
                check(out, q[l], cu, hist[l][0], hist[l][1], window, sinks, fp32_weights(dtype))
                if new == [1, 1, 1]:
                    out = pool.decode(l, q[l], window=window, sinks=sinks)
                    check(out, q[l], cu, hist[l][0], hist[l][1], window, sinks, fp32_weights(dtype))
    pool.check()
    k, _ = pool.gather(batch=B)
    at = 0
    for b in range(B):
        n = hist[1][0][b].numel()
        assert torch.equal(k[1, at:at + n].double(), hist[1][0][b].reshape(-1))
        at += n


@pytest.mark.parametrize("cache", ["same", "e4m3"])
def test_masked_places(cuda_device, cache):
    """NaN in K and V before the window (a block that is read, too) reaches nothing; in
    decode and in a chunk whose queries' windows all start after it."""
    lens, window, sinks = [200, 330], 50, 3
    pool, ks, vs = make_pool(torch.bfloat16, lens, 2, 128, 64, 17, cache)
    new = [4, 9]
    cu = [0, 4, 13]
    for b, n in enumerate(lens):
        for pos in list(range(sinks, 64)) + list(range(64, n - new[b] - window + 1)):
            blk = int(pool.block_tables[b, pos // 64])
            for t in (pool.k, pool.v):
                t[0, blk, :, pos % 64].view(torch.uint8).fill_(0x7F if cache == "e4m3" else 0xFF)
            ks[b][:, pos], vs[b][:, pos] = 0, 0
    q = torch.randn((13, 8, 128), device="cuda").bfloat16()
    cud = torch.tensor(cu, dtype=torch.int32, device="cuda")
    check(pool.attend_chunk(0, q, cud, window=window, sinks=sinks), q, cu, ks, vs, window, sinks, 2.0**-8)
    check(pool.decode(0, q[:2], window=window, sinks=sinks), q[:2], [0, 1, 2], ks, vs, window, sinks, 2.0**-8)
    pool.check()


def test_lengths_that_do_not_fit(cuda_device):
    """More new tokens than cached ones (the first see nothing: zeros), offsets past the
    rows, a table entry outside the pool: no access out of range, an error where one is due."""
    pool, ks, vs = make_pool(torch.bfloat16, [40, 30], 2, 128, 16, 4)
    q = torch.randn((60, 8, 128), device="cuda").bfloat16()
    cu = torch.tensor([0, 50, 60], dtype=torch.int32, device="cuda")
    out = pool.attend_chunk(0, q, cu)
    pool.check()
    assert (out[:10] == 0).all()
    check(out[10:], q[10:], [0, 40, 50], ks, vs, 0, 0, 2.0**-8)
    out = torch.full_like(q, 3.0)
    pool.attend_chunk(0, q, torch.tensor([-5, 20, 1000], dtype=torch.int32, device="cuda"), out=out)
    pool.check()
    pool.block_tables[1, 1] = 10**6
    pool.attend_chunk(0, q, cu)
    with pytest.raises(RuntimeError, match="block id"):
        pool.check()
    pool.decode(0, q[:2], window=20)
    with pytest.raises(RuntimeError, match="block id"):
        pool.check()


def test_refusals(cuda_device):
    from snapmind_b200 import PagedKVPool

    pool, _, _ = make_pool(torch.bfloat16, [40, 30], 2, 128, 16, 4)
    qp, _, _ = make_pool(torch.bfloat16, [40, 30], 2, 128, 16, 4, "e4m3")
    q = torch.randn((2, 8, 128), device="cuda").bfloat16()
    cu = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
    for p in (pool, qp):
        with pytest.raises(TypeError):
            p.attend_chunk(0, q.half(), cu)
        with pytest.raises(ValueError):
            p.attend_chunk(0, q, cu.long())
        with pytest.raises(ValueError):
            p.attend_chunk(0, q, cu.cpu())
        with pytest.raises(ValueError):
            p.attend_chunk(1, q, cu)
        with pytest.raises(ValueError):
            p.attend_chunk(0, q[..., :64], cu)
        with pytest.raises(ValueError):
            p.attend_chunk(0, q[:, :7], cu)
        with pytest.raises(ValueError):
            p.attend_chunk(0, q, cu, window=-1)
        with pytest.raises(ValueError):
            p.attend_chunk(0, q, cu, sinks=4)
        with pytest.raises(ValueError):
            p.decode(0, q, window=0, sinks=4)
        with pytest.raises(ValueError):
            p.attend_chunk(0, q, torch.zeros(4, dtype=torch.int32, device="cuda"))
        with pytest.raises(ValueError):
            p.attend_chunk(0, q, cu, out=torch.empty_like(q[:1]))
        with pytest.raises(ValueError):
            p.append_packed(0, q, q, cu)  # 8 heads, not 2
        with pytest.raises(ValueError):
            p.append_packed(1, q[:, :2], q[:, :2], cu)
        with pytest.raises(ValueError):
            p.reserve_each([1, -1])
        with pytest.raises(ValueError):
            p.reserve_each([1, 1, 1])
        with pytest.raises(RuntimeError, match="out of blocks"):
            p.reserve_each([100, 10])
        assert p.host_lens.tolist() == [40, 30]
    with pytest.raises(ValueError):
        pool.decode(0, q, window=5, peers=object())
    with pytest.raises(ValueError):
        qp.decode(0, q, peers=object())
    with pytest.raises(NotImplementedError):
        qp.decode_layers(q.unsqueeze(0))
    with pytest.raises(ValueError):
        PagedKVPool(1, 2, 300, 4, 1, 2, dtype=torch.bfloat16).attend_chunk(0, torch.zeros((1, 2, 300), device="cuda").bfloat16(), cu[:2])


@pytest.mark.parametrize("cache", ["same", "e4m3"])
def test_two_streams_and_a_captured_step(cuda_device, cache):
    """Calls on two streams at once, and a captured step replayed as the lengths grow."""
    lens = [900, 650]
    pool, ks, vs = make_pool(torch.bfloat16, lens, 4, 128, 16, 8, cache, spare=8)
    g = torch.Generator(device="cuda").manual_seed(2)
    qs = [torch.randn((70, 16, 128), generator=g, device="cuda").bfloat16() for _ in range(4)]
    cu = [0, 64, 70]
    cud = torch.tensor(cu, dtype=torch.int32, device="cuda")
    streams = [torch.cuda.Stream() for _ in range(4)]
    torch.cuda.synchronize()
    outs = []
    for s, q in zip(streams, qs):
        with torch.cuda.stream(s):
            for _ in range(3):
                o = pool.attend_chunk(0, q, cud, window=600, sinks=4)
            outs.append(o)
    torch.cuda.synchronize()
    for o, q in zip(outs, qs):
        check(o, q, cu, ks, vs, 600, 4, 2.0**-8)
    # a captured decode step: reserve, append, attend; two graphs over the same pool
    kn, vn = (torch.randn((2, 4, 128), generator=g, device="cuda").bfloat16() for _ in range(2))
    q1 = qs[0][:2].clone()
    one = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
    graphs, res = [], []
    pool.decode(0, q1, window=300, sinks=2)
    for window in (300, 0):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            pool.reserve_device(1, 2)
            pool.append(0, kn, vn)
            if window:
                out = pool.decode(0, q1, window=window, sinks=2)
            else:
                out = pool.attend_chunk(0, q1, one)
        graphs.append(gr)
        res.append((out, window))
    for step in range(6):
        gr, (out, window) = graphs[step % 2], res[step % 2]
        kn.normal_(generator=g)
        vn.normal_(generator=g)
        gr.replay()
        pool.account_host(1, 2)
        for b in range(2):
            for hist, x in ((ks, kn), (vs, vn)):
                val = quantise64(x[b])[0] if cache == "e4m3" else x[b].double()
                hist[b] = torch.cat([hist[b], val.unsqueeze(1)], 1)
        check(out, q1, [0, 1, 2], ks, vs, window, 2 if window else 0, 2.0**-8)
    pool.check()


@pytest.mark.parametrize("cache", ["same", "e4m3"])
def test_many_sequences(cuda_device, cache):
    """Hundreds of sequences of any length, empty ones among them (more than a CTA has threads)."""
    rng = np.random.RandomState(0)
    lens = [int(x) for x in rng.randint(0, 60, 700)]
    new = [min(n, int(x)) for n, x in zip(lens, rng.randint(0, 6, 700))]
    pool, ks, vs = make_pool(torch.bfloat16, lens, 2, 128, 16, 30, cache)
    cu = [0] + list(np.cumsum(new))
    q = torch.randn((cu[-1], 4, 128), device="cuda").bfloat16()
    out = pool.attend_chunk(0, q, torch.tensor(cu, dtype=torch.int32, device="cuda"))
    pool.check()
    check(out, q, cu, ks, vs, 0, 0, 2.0**-8)
    q = torch.randn((700, 4, 128), device="cuda").bfloat16()
    out = pool.decode(0, q, window=20, sinks=2)
    check(out, q, list(range(701)), ks, vs, 20, 2, 2.0**-8)
    pool.check()


def test_generator_on_a_quantised_pool(cuda_device):
    """gqa_paged over a QuantizedKVPool: prefill and decode through the plugin equal the operators' own calls."""
    from snapmind_b200 import PagedGroupedQueryAttention, QuantizedKVPool

    torch.manual_seed(0)
    attn = PagedGroupedQueryAttention(256, 4, 2, head_dim=64).cuda().to(torch.bfloat16)
    pool = QuantizedKVPool(1, 2, 64, 32, 2, 8, dtype=torch.bfloat16)
    view = pool.layer_views(2)[0]
    x = torch.randn((2, 21, 256), device="cuda").bfloat16()
    with torch.no_grad():
        pool.reserve(20, batch=2)
        y, _ = attn(x[:, :20], kv_cache=view)
        pool.reserve(1, batch=2)
        z, _ = attn(x[:, 20:], kv_cache=view)
        q = attn._split_heads(attn.q_proj(x), 4)
        k, v = (quantise64(attn._split_heads(f(x), 2))[0] for f in (attn.k_proj, attn.v_proj))
        for b in range(2):
            o, _ = reference(q[b].transpose(0, 1), k[b], v[b], 0, 0, 0.0)
            want = attn.out_proj(o.to(torch.bfloat16).reshape(1, 21, 256))
            got = torch.cat([y[b:b + 1], z[b:b + 1]], 1)
            # the attention rows and the projected rows are each rounded to bf16: a relative 2^-8
            # of the row's size per rounding, twice, and the weights' own
            assert (got - want).abs().max() <= 4 * 2.0**-8 * want.abs().max()
    pool.check()


KERNELS = [  # (cache, head dim, one token per sequence, force_generic): every attention kernel
    ("same", 128, False, False), ("same", 64, False, False), ("e4m3", 128, False, False), ("same", 128, True, False),
    ("e4m3", 128, True, False), ("same", 128, False, True), ("e4m3", 64, True, True),
]


@pytest.mark.parametrize("scale", [-0.07, 0.0, 1e-3, 0.9])
@pytest.mark.parametrize("cache,d,single,generic", KERNELS)
def test_scales(cuda_device, cache, d, single, generic, scale):
    """Any softmax scale: a negative one turns the scores round, zero gives the mean of V."""
    lens = [300, 77]
    pool, ks, vs = make_pool(torch.bfloat16, lens, 2, d, 16, 40, cache)
    cu = [0, 1, 2] if single else [0, 40, 45]
    q = torch.randn((cu[-1], 8, d), device="cuda").bfloat16()
    if single:
        out = pool.decode(0, q, scale=scale, window=90, sinks=2, force_generic=generic)
    else:
        out = pool.attend_chunk(0, q, torch.tensor(cu, dtype=torch.int32, device="cuda"), scale=scale, window=90, sinks=2,
                                force_generic=generic)
    pool.check()
    check_scaled(out, q, cu, ks, vs, 90, 2, scale)


def check_scaled(out, q, cu, ks, vs, window, sinks, scale):
    # a negative scale is the positive one of -q: the tolerance's sum of magnitudes is the same
    s = -1 if scale < 0 else 1
    check(out, q * s, cu, ks, vs, window, sinks, 2.0**-8, abs(scale))


@pytest.mark.parametrize("single", [False, True])
@pytest.mark.parametrize("cache", ["same", "e4m3"])
def test_rows_off_every_boundary(cuda_device, cache, single):
    """q and out one element off a 16-byte boundary, offsets that do not start at 0, odd strides."""
    lens = [130, 64]
    pool, ks, vs = make_pool(torch.bfloat16, lens, 2, 128, 16, 41, cache)
    cu = [0, 1, 2] if single else [3, 60, 71]
    flat = torch.randn(75 * 9 * 129 + 1, device="cuda").bfloat16()
    q = flat[1:].view(75, 9, 129)[:cu[-1], :8, :128]
    out = torch.full_like(flat, 5.0)[1:].view(75, 9, 129)[:cu[-1], :8, :128]
    if single:
        pool.decode(0, q, out=out, window=100, sinks=4)
    else:
        pool.attend_chunk(0, q, torch.tensor(cu, dtype=torch.int32, device="cuda"), out=out, window=100, sinks=4)
    pool.check()
    if not single:
        assert (out[:3] == 5.0).all()
    check(out[cu[0]:], q[cu[0]:], [c - cu[0] for c in cu], ks, vs, 100, 4, 2.0**-8)


@pytest.mark.parametrize("cache", ["same", "e4m3"])
def test_offsets_past_32_bits(cuda_device, cache):
    """Blocks at the end of a pool of more than 2^32 bytes (and rows whose elements pass 2^32): written,
    read back, attended."""
    from snapmind_b200 import PagedKVPool, QuantizedKVPool

    hkv, d, bs, n = 8, 128, 16, 200
    quant = cache == "e4m3"
    nb = 290_000 if quant else 270_000  # x 16 KB of elements
    pool = (QuantizedKVPool if quant else PagedKVPool)(1, hkv, d, nb, 1, 16, block_size=bs, dtype=torch.bfloat16)
    assert (nb - 20) * hkv * bs * d > 2**32
    pool.set_state(np.arange(nb - 13, nb)[::-1][None].copy(), np.array([0]), np.arange(4))
    pool.block_tables[0, :13] = torch.arange(nb - 1, nb - 14, -1, device="cuda", dtype=torch.int32)
    pool.seq_lens[0] = n
    pool._host_lens[0] = n
    k, v = (torch.randn((1, n, hkv, d), device="cuda").bfloat16() for _ in range(2))
    cu = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    pool.append_packed(None, k, v, cu)
    ks, vs = ([(quantise64(x[0])[0] if quant else x[0].double()).transpose(0, 1)] for x in (k, v))
    kg, vg = pool.gather()
    assert torch.equal(kg.view(hkv, n, d).double(), ks[0]) and torch.equal(vg.view(hkv, n, d).double(), vs[0])
    q = torch.randn((n, 32, d), device="cuda").bfloat16()
    check(pool.attend_chunk(0, q, cu), q, [0, n], ks, vs, 0, 0, 2.0**-8)
    check(pool.decode(0, q[:1], window=150, sinks=3), q[:1], [0, 1], ks, vs, 150, 3, 2.0**-8)
    check(pool.attend_chunk(0, q, cu, force_generic=True), q, [0, n], ks, vs, 0, 0, 2.0**-8)
    pool.check()


@pytest.mark.parametrize("cache", ["same", "e4m3"])
def test_decode_that_stores_its_token(cuda_device, cache):
    """decode(append=) with a window, and over an 8-bit pool; only the first sequences of the pool."""
    pool, ks, vs = make_pool(torch.bfloat16, [70, 31, 50], 2, 128, 16, 42, cache, spare=4)
    pool.reserve(1, batch=2)
    kn, vn = (torch.randn((2, 2, 128), device="cuda").bfloat16() for _ in range(2))
    q = torch.randn((3, 8, 128), device="cuda").bfloat16()
    out = pool.decode(0, q, append=(kn, vn), window=40, sinks=1, batch=2)
    pool.check()
    assert out.shape == (2, 8, 128)
    for b in range(2):
        for hist, x in ((ks, kn), (vs, vn)):
            val = quantise64(x[b])[0] if cache == "e4m3" else x[b].double()
            hist[b] = torch.cat([hist[b], val.unsqueeze(1)], 1)
    check(out, q[:2], [0, 1, 2], ks[:2], vs[:2], 40, 1, 2.0**-8)


@pytest.mark.parametrize("single,generic", [(False, False), (True, False), (False, True)])
def test_a_length_past_the_table(cuda_device, single, generic):
    pool, _, _ = make_pool(torch.bfloat16, [40], 2, 128, 16, 43)
    pool.seq_lens[0] = 16 * pool.max_blocks_per_seq + 9
    q = torch.randn((1, 8, 128), device="cuda").bfloat16()
    cu = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    pool.block_tables.fill_(0)
    if single:
        pool.decode(0, q, window=30)
    else:
        pool.attend_chunk(0, q, cu, force_generic=generic)
    with pytest.raises(RuntimeError, match="table"):
        pool.check()


def test_generator_graph_on_a_quantised_pool(cuda_device):
    """BatchedGraphDecoder over a QuantizedKVPool: the captured steps give the ids of eager steps."""
    import torch.nn as nn

    from snapmind_b200 import PagedGroupedQueryAttention, QuantizedKVPool
    from snapmind_b200.engine import BatchedGraphDecoder

    class Tiny(nn.Module):
        def __init__(self):
            super().__init__()
            self.emb = nn.Embedding(50, 64)
            self.attn = PagedGroupedQueryAttention(64, 4, 2, head_dim=64)
            self.head = nn.Linear(64, 50)

        def forward(self, ids, kv_cache, position_ids=None):
            x = self.emb(ids)
            return self.head(x + self.attn(x, kv_cache=kv_cache[0], position_ids=position_ids)[0])

    torch.manual_seed(3)
    model = Tiny().cuda()
    prompts = torch.randint(0, 50, (3, 19), generator=torch.Generator().manual_seed(0)).cuda()
    ids = []
    for use_graph in (False, True):
        pool = QuantizedKVPool(1, 2, 64, 24, 3, 8, dtype=torch.float32)
        ids.append(BatchedGraphDecoder(model, pool, 3, use_graph=use_graph).generate(prompts, 12))
    assert ids[0] == ids[1]


@pytest.mark.parametrize("cache,d,single,generic", KERNELS)
def test_nan_is_not_hidden(cuda_device, cache, d, single, generic):
    """A NaN in a query makes that (row, head) NaN, one in a key every row and head that sees it, on
    one CTA or on many; the others keep their values."""
    lens, new = ([5000, 40, 0], [1, 1, 1]) if single else ([5000, 40, 0], [3, 20, 0])
    pool, ks, vs = make_pool(torch.bfloat16, lens, 2, d, 16, 44, cache)
    cu = [0, *itertools.accumulate(new)]
    cud = torch.tensor(cu, dtype=torch.int32, device="cuda")
    q = torch.randn((cu[-1], 8, d), device="cuda").bfloat16()

    def run(x, window):
        if single:
            return pool.decode(0, x, window=window, sinks=min(window, 2), force_generic=generic)
        return pool.attend_chunk(0, x, cud, window=window, sinks=min(window, 2), force_generic=generic)

    # one (row, head) whose every score is NaN
    for window in (64, 4096) if single and cache == "same" else (0, 64):
        clean = run(q, window)
        bad = q.clone()
        bad[0, 3] = float("nan")
        bad[cu[1], 6, 5] = float("nan")
        out = run(bad, window)
        hit = torch.zeros_like(out, dtype=torch.bool)
        hit[0, 3] = hit[cu[1], 6] = True
        assert torch.isnan(out[hit]).all()
        # each within half a step of the output's type and of the weights' of sums of at most max |v|
        assert (out - clean)[~hit].abs().max() <= 4 * 2.0**-8 * float(max(v.abs().max() for v in vs[:2]))
    # the newest key of sequence 0, kv head 1: only its last query sees it
    slot = lens[0] - 1
    block = int(pool.block_tables[0, slot // 16])
    if cache == "e4m3":
        pool.k.view(torch.uint8)[0, block, 1, slot % 16, 7] = 0x7F
    else:
        pool.k[0, block, 1, slot % 16, 7] = float("nan")
    out = run(q, 64)
    hit = torch.zeros_like(out, dtype=torch.bool)
    hit[cu[1] - 1, 4:] = True
    assert torch.isnan(out[hit]).all()
    assert torch.isfinite(out[~hit]).all()
    pool.check()


@pytest.mark.parametrize("cache,d,single,generic", KERNELS)
def test_positions_past_the_table_do_not_count(cuda_device, cache, d, single, generic):
    """A length of 89 over a table row of 80 positions: the newest tokens see those 80 (under a
    window of 30, the ones of them within it), and the pool's error word tells."""
    pool, ks, vs = make_pool(torch.bfloat16, [80], 2, d, 16, 45, cache)
    row = pool.block_tables[:, :5].contiguous()
    pool.block_tables, pool.max_blocks_per_seq = row, 5
    pool.seq_lens[0] = 89
    t = 1 if single else 3
    q = torch.randn((t, 8, d), device="cuda").bfloat16()
    cu = torch.tensor([0, t], dtype=torch.int32, device="cuda")
    for window in (30,) if single and cache == "same" else (0, 30):
        if single:
            out = pool.decode(0, q, window=window, force_generic=generic)
        else:
            out = pool.attend_chunk(0, q, cu, window=window, force_generic=generic)
        for i in range(t):
            lo = max(0, 89 - t + i - window + 1) if window else 0
            check(out[i:i + 1], q[i:i + 1], [0, 1], [ks[0][:, lo:]], [vs[0][:, lo:]], 0, 0, 2.0**-8)
        with pytest.raises(RuntimeError, match="table"):
            pool.check()


def test_counts_and_offsets_of_other_types(cuda_device):
    pool, _, _ = make_pool(torch.bfloat16, [40, 30], 2, 128, 16, 4, spare=4)
    kv = torch.randn((2, 2, 128), device="cuda").bfloat16()
    cu = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
    for bad in ([1.5, 1.0], ["1", "1"]):
        with pytest.raises(ValueError):
            pool.reserve_each(bad)
    for bad in (cu[0], cu.long(), cu.cpu(), cu[:0]):
        with pytest.raises(ValueError):
            pool.append_packed(0, kv, kv, bad)
    assert pool.host_lens.tolist() == [40, 30]
    pool.reserve_each([])
    pool.reserve_each(np.array([1, 0], dtype=np.uint8))
    pool.reserve_each(torch.tensor([0, 1]))
    assert pool.host_lens.tolist() == pool.seq_lens.tolist() == [41, 31]
    pool.check()


@pytest.mark.parametrize("d", [64, 128, 40, 256])
@pytest.mark.parametrize("src,dst", [("bf16", "bf16"), ("f32", "f32"), ("f16", "f16"), ("f32", "bf16"), ("bf16", "f32")])
def test_packed_rows_are_stored(cuda_device, src, dst, d):
    """append_packed puts every row where it belongs and nothing elsewhere: aligned rows, rows off
    every boundary, rows outside every sequence, an empty sequence, one layer of several."""
    from snapmind_b200 import PagedKVPool

    pool = PagedKVPool(3, 2, d, 40, 4, 20, block_size=8, dtype=DT[dst])
    new = [37, 0, 1, 90]
    pool.reserve_each([5, 3, 0, 2])
    pool.reserve_each(new)
    pool.k.fill_(7)
    pool.v.fill_(7)
    total = sum(new) + 3
    cu = torch.tensor([2, 39, 39, 40, 130], dtype=torch.int32, device="cuda")  # rows 0, 1 and 130 are no one's
    for off in (0, 1):
        k, v = (torch.randn((2, total, 2, d + 1), device="cuda").to(DT[src])[..., off:off + d] for _ in range(2))
        if not off:
            k, v = k.contiguous(), v.contiguous()
        pool.append_packed(None, k, v, cu)  # layers 0 and 1
        pool.check()
        for x, p in ((k, pool.k), (v, pool.v)):
            want = torch.full_like(p, 7)
            for b, n in enumerate(new):
                for i in range(n):
                    slot = int(pool.host_lens[b]) - n + i
                    want[:2, int(pool.block_tables[b, slot // 8]), :, slot % 8] = x[:, int(cu[b]) + i].to(DT[dst])
            assert torch.equal(p, want)
