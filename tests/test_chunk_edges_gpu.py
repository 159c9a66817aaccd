"""The chunk operators and the 8-bit cache at the ends of their ranges: counts from device memory,
exponents far apart, masked infinities, bad block ids."""
import math

import numpy as np
import pytest
import torch

import snapmind_b200._lib as lib
from test_chunk_gpu import CASES, DECODE, DT, HALF, KERNELS, check, make_pool, quantise64, visible

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


def set_exponents(pool, lens, k_exp, v_exp):
    """Gives the rows of an 8-bit pool these exponents ([blocks, heads, slots]); the sequences' K and V in f64."""
    _, _, heads, bs, d = pool.k.shape
    kv = []
    for i, (codes, e) in enumerate(((pool.k, k_exp), (pool.v, v_exp))):
        keep = pool.scales[0, :, :, i] == 255  # slots without a token
        pool.scales[0, :, :, i] = torch.where(keep, pool.scales[0, :, :, i], (e + 127).to(torch.uint8))
        val = codes[0].double() * torch.exp2(e.double()).unsqueeze(-1)
        kv.append([val[pool.block_tables[b, :(n + bs - 1) // bs].long()].permute(1, 0, 2, 3).reshape(heads, -1, d)[:, :n]
                   for b, n in enumerate(lens)])
    return kv


def pick(g, values, shape):
    return torch.tensor(values, device="cuda")[torch.randint(0, len(values), shape, generator=g, device="cuda")]


@pytest.mark.parametrize("window,sinks", [(0, 0), (700, 5)])
@pytest.mark.parametrize("exps", [(-100, 40), (-99, 40), (-100, -60, -20, 20, 60, 100), tuple(range(-100, 101, 7))],
                         ids=lambda e: f"{e[0]}..{e[-1]}x{len(e)}")
@pytest.mark.parametrize("lens", [[2], [5000, 33, 1], [40000]], ids=str)
def test_values_of_far_apart_scales(cuda_device, lens, exps, window, sinks):
    """8-bit decode: every seen row counts in the softmax sum by its score alone, whatever the scale of its
    values; in one tile, over a CTA's warps, and over many CTAs."""
    pool, _, _ = make_pool(torch.bfloat16, lens, 2, 128, 16, 50, "e4m3")
    g = torch.Generator(device="cuda").manual_seed(4)
    shape = pool.scales.shape[1:3] + (16,)
    v_exp = pick(g, exps, shape)
    pool.v.view(torch.uint8)[0].masked_fill_((v_exp == -100).unsqueeze(-1) & (pool.scales[0, :, :, 1] != 255).unsqueeze(-1), 0)
    ks, vs = set_exponents(pool, lens, pick(g, (-9, -8, -7), shape), v_exp)
    q = torch.randn((len(lens), 8, 128), generator=g, device="cuda").bfloat16()
    out = pool.decode(0, q, window=window, sinks=sinks)
    pool.check()
    check(out, q, list(range(len(lens) + 1)), ks, vs, window, sinks, HALF[torch.float16])


def test_a_row_of_zeros_counts(cuda_device):
    """Two keys of equal score, one with V = 0 (stored with the smallest exponent), one with V = 2^40: 2^39."""
    from snapmind_b200 import QuantizedKVPool

    pool = QuantizedKVPool(1, 1, 128, 4, 1, 2, dtype=torch.bfloat16)
    pool.reserve(2, batch=1)
    k = torch.zeros((1, 1, 2, 128), device="cuda").bfloat16()
    v = k.clone()
    v[0, 0, 1] = 2.0**40
    pool.append(0, k, v)
    out = pool.decode(0, torch.ones((1, 4, 128), device="cuda").bfloat16())
    pool.check()
    assert (out == 2.0**39).all()


@pytest.mark.parametrize("k_exp,size,scale", [
    (126, 2.0**-109, 2.0**-20), (126, 2.0**-90, 2.0**-39), (112, 2.0**-109, None), (100, 2.0**-99, 40.0),
    (-92, 2.0**97, None), (-92, 2.0**115, 2.0**-22), (90, 2.0**-92, 2.0**-10),
])
@pytest.mark.parametrize("generic", [False, True])
def test_keys_of_far_scales(cuda_device, k_exp, size, scale, generic):
    """8-bit decode of keys near the ends of the range and queries near the other end: scores of ordinary size."""
    lens = [300, 65]
    pool, _, _ = make_pool(torch.bfloat16, lens, 2, 128, 16, 51, "e4m3")
    g = torch.Generator(device="cuda").manual_seed(5)
    shape = pool.scales.shape[1:3] + (16,)
    ks, vs = set_exponents(pool, lens, pick(g, (k_exp - 8, k_exp - 7), shape), pick(g, (-9, -8), shape))
    q = (size * torch.randn((2, 8, 128), generator=g, device="cuda")).bfloat16()
    out = pool.decode(0, q, scale=scale, force_generic=generic)
    pool.check()
    check(out, q, [0, 1, 2], ks, vs, 0, 0, 0.0 if generic else HALF[torch.float16], scale)


@pytest.mark.parametrize("dtype,cache,single,generic", [
    ("f16", "same", True, False), ("f16", "same", False, False), ("bf16", "same", True, False), ("bf16", "same", False, False),
    ("f16", "e4m3", True, False), ("f16", "e4m3", False, False), ("bf16", "e4m3", True, False), ("bf16", "e4m3", False, False),
    ("f16", "same", False, True),
])
@pytest.mark.parametrize("n,drop", [(16384, 26), (5000, 24), (60000, 28)])
def test_many_small_weights_behind_a_sink(cuda_device, dtype, cache, single, generic, n, drop):
    """The first key has 2^drop times the weight of each other one, and V = 0: the others' sum is all there is.

    want = (n - 1) 2^-drop / (1 + (n - 1) 2^-drop).  A weight is off by half a step of its type (2^-11 of it, bf16
    2^-8) or, below f16's normal range, by 2^-32 of the largest weight; the score 2^8 scale by two roundings of
    24 bits, 2^-18 of the result with 2^x; the output by half a step."""
    from snapmind_b200 import PagedKVPool, QuantizedKVPool

    dtype = DT[dtype]
    t, nseq, hkv, blocks = 1 if single else 3, 40, 8, (n + 15) // 16
    # 320 (sequence, kv head) pairs over one set of blocks: nearly every CTA goes through whole sequences
    pool = (QuantizedKVPool if cache == "e4m3" else PagedKVPool)(1, hkv, 128, blocks, nseq, blocks, dtype=dtype)
    pool.set_state(np.arange(blocks)[None].repeat(nseq, 0), np.full(nseq, n), np.arange(0))
    k = torch.zeros((1, hkv, n, 128), device="cuda", dtype=dtype)
    v = torch.ones_like(k)
    k[:, :, 0, 3], v[:, :, 0] = 16.0, 0.0
    pool.append(0, k, v)
    q = torch.zeros((nseq * t, 2 * hkv, 128), device="cuda", dtype=dtype)
    q[:, :, 3] = 16.0
    scale = drop * math.log(2) / 256
    if single:
        out = pool.decode(0, q, scale=scale, window=1 << 20, force_generic=generic)
    else:
        cu = torch.arange(nseq + 1, dtype=torch.int32, device="cuda") * t
        out = pool.attend_chunk(0, q, cu, scale=scale, force_generic=generic)
    pool.check()
    for i in range(t):
        others = (n - t + i) * 2.0**-drop
        want = others / (1 + others)
        weights = HALF[torch.float16] if cache == "e4m3" and single else 0.0 if generic else HALF[dtype]
        tol = want * (weights + HALF[dtype] * 1.01 + 2.0**-18) + (0 if generic else n * 2.0**-32)
        assert (out[i::t].double() - want).abs().max() <= tol


@pytest.mark.parametrize("generic", [False, True])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("k_exps,v_exps,size", [
    ((-20, -8, 2), (-15, -3, 7), 1.0),            # what f16 holds
    ((-9, -8, -21), (-9,), 2.0**13),              # K below it, queries that bring it back
    ((-40, -39), (-9,), 2.0**13),
    ((-100, 3, 8), (-9, -100), 2.0**-14),         # K above it
    ((-9, -8), (-60, -24, -9), 1.0),              # V below it: lost in an f16 output too
    ((-9, -8), (-9, 8), 1.0),                     # V above it in one row, outputs that f16 holds
    ((-9, -8), (-9, 15), 1.0),
], ids=str)
def test_f16_queries_over_any_exponent(cuda_device, d, k_exps, v_exps, size, generic):
    """Chunks of f16 queries over 8-bit rows that f16 does not hold, one such row among a thousand too: the rows'
    values count as they are stored."""
    lens, new = [900, 130, 40], [70, 130, 0]
    pool, _, _ = make_pool(torch.float16, lens, 2, d, 16, 52, "e4m3")
    g = torch.Generator(device="cuda").manual_seed(7)
    shape = pool.scales.shape[1:3] + (16,)
    cu = [0, 70, 200, 200]
    cud = torch.tensor(cu, dtype=torch.int32, device="cuda")
    for rare in (False, True) if max(v_exps) < 8 else (True,):
        k_exp, v_exp = pick(g, k_exps, shape), pick(g, v_exps, shape)
        if rare:  # ordinary rows, but for one
            one = torch.zeros(shape, dtype=torch.bool, device="cuda")
            one[int(pool.block_tables[0, 20]), 1, 7] = True
            k_exp, v_exp = torch.where(one, k_exps[-1], -9), torch.where(one, v_exps[-1], -9)
        ks, vs = set_exponents(pool, lens, k_exp, v_exp)
        q = (size * torch.randn((200, 8, d), generator=g, device="cuda")).half()
        scale = 0.1 / (size * float(max(k.abs().max() for k in ks)))
        out = pool.attend_chunk(0, q, cud, scale=scale, force_generic=generic)
        pool.check()
        check(out, q, cu, ks, vs, 0, 0, 0.0 if generic else HALF[torch.float16], scale)
        # a token each, as a decode step
        out = pool.decode(0, q[:3], scale=scale, force_generic=generic)
        check(out, q[:3], [0, 1, 2, 3], ks, vs, 0, 0, HALF[torch.float16], scale)
    pool.check()


@pytest.mark.parametrize("cache", ["same", "e4m3"])
def test_decode_stores_tokens_of_its_own_batch_only(cuda_device, cache):
    """decode(append=, window=): rows of another number of sequences or another shape are refused, as without a
    window, and so is the whole call when its queries are; nothing is stored then."""
    pool, _, _ = make_pool(torch.bfloat16, [70, 31, 50], 2, 128, 16, 42, cache, spare=4)
    pool.reserve(1, batch=2)
    kept = [pool.k.view(torch.uint8).clone(), pool.v.view(torch.uint8).clone()]
    kv = torch.randn((3, 2, 128), device="cuda").bfloat16()
    q = torch.randn((3, 8, 128), device="cuda").bfloat16()
    for bad in ((kv, kv), (kv[:2], kv), (kv[:2], kv[:1]), (kv[:2, :1], kv[:2, :1])):
        with pytest.raises(ValueError):
            pool.decode(0, q, append=bad, window=40, batch=2)
    with pytest.raises(ValueError):
        pool.decode(0, q[:2], append=(kv, kv), window=40)
    with pytest.raises(TypeError):
        pool.decode(0, q.half(), append=(kv[:2], kv[:2]), window=40, batch=2)
    pool.check()
    assert torch.equal(kept[0], pool.k.view(torch.uint8)) and torch.equal(kept[1], pool.v.view(torch.uint8))


@pytest.mark.parametrize("cache", ["same", "e4m3"])
def test_decode_of_the_first_sequences(cuda_device, cache):
    """batch= with queries and an output buffer for the whole pool, as without a window: the rows behind stay."""
    lens = [70, 31, 50]
    pool, ks, vs = make_pool(torch.bfloat16, lens, 2, 128, 16, 42, cache)
    q = torch.randn((3, 8, 128), device="cuda").bfloat16()
    out = torch.full_like(q, 7.0)
    assert pool.decode(0, q, out=out, window=40, sinks=1, batch=2) is out
    pool.check()
    check(out[:2], q[:2], [0, 1, 2], ks[:2], vs[:2], 40, 1, 2.0**-8)
    assert (out[2] == 7.0).all()
    assert pool.decode(0, q, window=40, batch=0).shape == (0, 8, 128)
    for batch in (4, -1):
        with pytest.raises(ValueError):
            pool.decode(0, q, window=40, batch=batch)
    with pytest.raises(ValueError):
        pool.decode(0, q, out=out[:1], window=40, batch=2)


@pytest.mark.parametrize("cache", ["same", "e4m3"])
def test_windows_past_32_bits(cuda_device, cache):
    """Windows and sinks of 2^31 and more are what they say, not their lowest bits; negative ones are refused."""
    lens = [70, 31]
    pool, ks, vs = make_pool(torch.bfloat16, lens, 2, 128, 16, 42, cache)
    q = torch.randn((2, 8, 128), device="cuda").bfloat16()
    cu = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
    for window, sinks in ((2**31, 0), (2**32 + 5, 2), (2**64 + 5, 2**40), (5, 2**32 + 1)):
        for out in (pool.decode(0, q, window=window, sinks=sinks), pool.attend_chunk(0, q, cu, window=window, sinks=sinks)):
            check(out, q, [0, 1, 2], ks, vs, 0, 0, 2.0**-8)
    for window, sinks in ((-(2**32) + 5, 0), (5, -(2**32) + 1), (-(2**31), 0)):
        with pytest.raises(ValueError, match="negative"):
            pool.attend_chunk(0, q, cu, window=window, sinks=sinks)
        with pytest.raises(ValueError, match="negative"):
            pool.decode(0, q, window=window, sinks=sinks)
    pool.check()


def test_attend_causal_of_any_sequence_and_length(cuda_device):
    """QuantizedKVPool.attend_causal: a sequence past the 8192nd, and n_b below the length."""
    from snapmind_b200 import QuantizedKVPool

    pool = QuantizedKVPool(1, 2, 128, 8, 8200, 6, dtype=torch.bfloat16)
    tables = np.zeros((8200, 6), np.int64)
    tables[8197], tables[3] = [5, 1, 0, 7, 2, 4], [3, 6, 0, 0, 0, 0]
    lens = np.zeros(8200, np.int64)
    lens[8197], lens[3] = 77, 20
    pool.set_state(tables, lens, np.arange(0))
    codes = (64 * torch.randn((2, 77, 128), device="cuda")).clamp(-448, 448).to(torch.float8_e4m3fn)
    pool.scales.fill_(127 - 6)
    for t in range(77):
        for p in (pool.k, pool.v):
            p.view(torch.uint8)[0, tables[8197, t // 16], :, t % 16] = codes.view(torch.uint8)[:, t]
    held = codes.double() / 64
    q = torch.randn((8, 9, 128), device="cuda").bfloat16()
    for n_b in (77, 41, 9):
        out = torch.empty_like(q)
        assert pool.attend_causal(0, 8197, q, out, n_b) is out
        pool.check()
        check(out.transpose(0, 1), q.transpose(0, 1), [0, 9], [held[:, :n_b]], [held[:, :n_b]], 0, 0, 2.0**-8)


def attention64(q, k, v, see, weight_half, scale=None):
    """(o, tolerance) of one sequence in f64 under any mask see [t, n]: test_chunk_gpu's reference and its bounds."""
    t, hq, d = q.shape
    hkv, n, _ = k.shape
    scale = d ** -0.5 if scale is None else scale
    o = torch.zeros((t, hq, d), dtype=torch.float64, device="cuda")
    tol = torch.zeros_like(o)
    for h in range(hq):
        kh, vh = (x[h * hkv // hq] for x in (k, v))
        s = (q[:, h].double() @ kh.T * scale).masked_fill(~see, -torch.inf)
        sa = (q[:, h].double().abs() @ kh.abs().T).masked_fill(~see, 0).amax(-1, keepdim=True) * scale
        m = s.amax(-1, keepdim=True)
        p = torch.exp(s - torch.where(torch.isfinite(m), m, 0.0))
        z = p.sum(-1, keepdim=True)
        p = torch.where(z > 0, p / z, 0.0)
        u = 2.0**-24
        w = 2.0**-21 + 2 * (d + 4) * u * sa
        o[:, h] = p @ vh
        top = torch.where(z > 0, 1 / z, 0.0) * (see.double() @ vh.abs())
        tol[:, h] = p @ vh.abs() * (2 * w + 2 * n * u + weight_half) + 2.0**-25 * top * (weight_half > 0)
    return o, tol


def check_seen(out, q, k, v, see, weight_half, but=None):
    o, tol = attention64(q, k, v, see, weight_half)
    if but is not None:
        o = o.masked_fill(but, 0)
    tol = tol + HALF[out.dtype] * o.abs() * (1 + 2.0**-6) + 1e-30
    err = (out.double() - o).abs()
    assert torch.isfinite(out).all()
    assert not (err > tol).any(), f"worst {float((err / tol).max()):.2f} x the tolerance"


@pytest.mark.parametrize("bs", [8, 16, 32, 64, 256])
@pytest.mark.parametrize("cache,d,single,generic", KERNELS)
def test_blocks_that_are_none(cuda_device, cache, d, single, generic, bs):
    """A table entry outside the pool: its keys are seen by nobody, whatever lay where they would have been
    staged, and the error word tells."""
    lens, new = ([3000, 700], [1, 1]) if single else ([3000, 700], [40, 300])
    pool, ks, vs = make_pool(torch.bfloat16, lens, 2, d, bs, 53, cache)
    q = torch.randn((sum(new), 8, d), device="cuda").bfloat16()
    cu = torch.tensor([0, new[0], sum(new)], dtype=torch.int32, device="cuda")
    bad = [{0, 1, 900 // bs, 2900 // bs}, {300 // bs, 699 // bs}]  # 699: the newest tokens' own block
    lost = [torch.zeros(n, dtype=torch.bool, device="cuda") for n in lens]
    for b in range(2):
        for i in bad[b]:
            pool.block_tables[b, i] = -1 if i % 2 else 10**6
            lost[b][i * bs:(i + 1) * bs] = True
    window = 2900 if single and cache == "same" else 0
    if single:
        out = pool.decode(0, q, window=window, force_generic=generic)
    else:
        out = pool.attend_chunk(0, q, cu, window=window, force_generic=generic)
    with pytest.raises(RuntimeError, match="block id"):
        pool.check()
    for b in range(2):
        see = visible(lens[b], new[b], window, 0) & ~lost[b]
        check_seen(out[cu[b]:cu[b + 1]], q[cu[b]:cu[b + 1]], ks[b], vs[b], see, HALF[torch.bfloat16])


@pytest.mark.parametrize("window,sinks", [(0, 0), (50, 3), (16, 100)])
@pytest.mark.parametrize("hq", [8, 1])
@pytest.mark.parametrize("cache,dtype,d,generic", [
    ("same", "bf16", 128, False), ("same", "f16", 64, False), ("e4m3", "bf16", 128, False), ("e4m3", "bf16", 64, False),
    ("e4m3", "f16", 128, False), ("same", "bf16", 64, True), ("same", "f32", 128, True), ("same", "bf16", 256, True),
    ("e4m3", "bf16", 128, True),
])
def test_odd_values_reach_those_that_see_them(cuda_device, cache, dtype, d, generic, hq, window, sinks):
    """Infinities and NaN in V of tokens that some queries of a chunk see and others do not: an output is not finite
    exactly where its query sees one in that dim, and the others have their values.  Whole units, units cut
    into pieces, and chunks that start the sequence."""
    dtype = DT[dtype]
    lens, new = [9000, 300, 200, 40], [150, 300, 9, 0]
    hkv = min(hq, 2)
    pool, ks, vs = make_pool(dtype, lens, hkv, d, 16, 54, cache)
    cu = [0, 150, 450, 459, 459]
    odd = [[8999, 8900, 8851, 8840, 8803, 5000], [0, 17, 130, 299], [199, 192, 150], []]
    hit = []
    for b, n in enumerate(lens):
        h = torch.zeros((hkv, n, d), dtype=torch.bool, device="cuda")
        for i, pos in enumerate(odd[b]):
            head, dims, blk = i % hkv, [(7 * i) % d, (7 * i + 33) % d], int(pool.block_tables[b, pos // 16])
            for dim in dims:
                if cache == "e4m3":
                    pool.v.view(torch.uint8)[0, blk, head, pos % 16, dim] = 0xFF if i % 2 else 0x7F
                else:
                    pool.v[0, blk, head, pos % 16, dim] = float(("inf", "-inf", "nan")[i % 3])
            h[head, pos, dims] = True
            vs[b][head, pos, dims] = 0
        hit.append(h)
    q = torch.randn((cu[-1], hq, d), device="cuda").to(dtype)
    cud = torch.tensor(cu, dtype=torch.int32, device="cuda")
    out = pool.attend_chunk(0, q, cud, window=window, sinks=sinks, force_generic=generic)
    pool.check()
    for b, (n, t) in enumerate(zip(lens, new)):
        if t == 0:
            continue
        see = visible(n, t, window, sinks)
        want = torch.stack([see.double() @ hit[b][h * hkv // hq].double() for h in range(hq)], 1) > 0
        rows = out[cu[b]:cu[b + 1]]
        assert torch.equal(~torch.isfinite(rows), want)
        check_seen(rows.masked_fill(want, 0), q[cu[b]:cu[b + 1]], ks[b], vs[b], see, 0.0 if generic else HALF[dtype], want)


def weight_rounding(dtype, cache, hq, hkv, d, bs, single, generic):
    """Half a step of the type that the kernel which takes the call rounds a weight to; 0 for the CUDA-core kernel."""
    if generic or dtype == torch.float32 or d not in (64, 128) or (bs not in (8, 16, 32, 64) and bs % 128):
        return 0.0
    narrow = single and d == 128 and hq // hkv <= 8 and (bs in (16, 32) or bs % 64 == 0)
    return HALF[torch.float16] if narrow and cache == "e4m3" else HALF[dtype]


@pytest.mark.parametrize("generic", [False, True])
@pytest.mark.parametrize("case", CASES + [(*c[:7], None, *c[7:]) for c in DECODE], ids=lambda c: "-".join(str(x) for x in c[:8]))
def test_weights_are_rounded_once(cuda_device, case, generic):
    """Every kernel within the bound of the one rounding of a weight that it makes: none on the CUDA cores, f16's
    in 8-bit decodes of head dim 128, whatever the query's type."""
    dtype, cache, hq, hkv, d, bs, lens, new, window, sinks = case
    dtype, single = DT[dtype], new is None
    new = [1] * len(lens) if single else new
    pool, ks, vs = make_pool(dtype, lens, hkv, d, bs, 61, cache)
    cu = [0, *np.cumsum(new).tolist()]
    g = torch.Generator(device="cuda").manual_seed(8)
    q = (1.5 * torch.randn((cu[-1], hq, d), generator=g, device="cuda")).to(dtype)
    if single and (window or cache == "e4m3"):
        out = pool.decode(0, q, window=window, sinks=sinks, force_generic=generic)
    else:
        out = pool.attend_chunk(0, q, torch.tensor(cu, dtype=torch.int32, device="cuda"), window=window, sinks=sinks,
                                force_generic=generic)
    pool.check()
    check(out, q, cu, ks, vs, window, sinks, weight_rounding(dtype, cache, hq, hkv, d, bs, single, generic))


def test_quantised_pool_refuses_what_it_does_not_hold(cuda_device):
    """Sequences past the pool's (their tables and lengths would be read from whatever lies behind), a length shorter
    than its queries."""
    pool, _, _ = make_pool(torch.bfloat16, [40, 30], 2, 128, 16, 4, "e4m3")
    for batch in (3, 10**6, -1):
        with pytest.raises(ValueError, match="sequences"):
            pool.gather(batch=batch)
    q = torch.randn((8, 5, 128), device="cuda").bfloat16()
    for n_b in (4, 0, -3):
        with pytest.raises(ValueError, match="queries"):
            pool.attend_causal(0, 1, q, torch.empty_like(q), n_b)
    pool.check()


@pytest.mark.parametrize("cache", ["same", "e4m3"])
def test_decode_stores_rows_of_any_layout(cuda_device, cache):
    """decode(append=, window=): rows whose head dim is not contiguous are stored as they are; K and V of two types,
    or from another device, are refused."""
    lens = [70, 31]
    pool, ks, vs = make_pool(torch.bfloat16, lens, 2, 128, 16, 42, cache, spare=4)
    pool.reserve(1, batch=2)
    kn, vn = (torch.randn((2, 128, 2), device="cuda").bfloat16().transpose(1, 2) for _ in range(2))
    q = torch.randn((2, 8, 128), device="cuda").bfloat16()
    for bad in ((kn, vn.float()), (kn.cpu(), vn.cpu()), (kn, vn.cpu())):
        with pytest.raises(ValueError):
            pool.decode(0, q, append=bad, window=40)
    out = pool.decode(0, q, append=(kn, vn), window=40)
    pool.check()
    for b in range(2):
        for hist, x in ((ks, kn), (vs, vn)):
            val = quantise64(x[b])[0] if cache == "e4m3" else x[b].double()
            hist[b] = torch.cat([hist[b], val.unsqueeze(1)], 1)
    check(out, q, [0, 1, 2], ks, vs, 40, 0, 2.0**-8)


@pytest.mark.parametrize("single", [False, True])
@pytest.mark.parametrize("cache,dtype,v_exp", [("same", "bf16", 0), ("e4m3", "bf16", 8), ("e4m3", "f16", -8), ("e4m3", "f16", 9)])
def test_output_over_the_queries(cuda_device, cache, dtype, v_exp, single):
    """out=q: the queries' rows become the outputs', also where a call is done over (V of exponent 9 in f16)."""
    lens, d = [900, 130, 40], 64
    pool, ks, vs = make_pool(DT[dtype], lens, 2, d, 16, 55, cache)
    cu = [0, 1, 2, 3] if single else [0, 70, 200, 203]
    g = torch.Generator(device="cuda").manual_seed(9)
    if cache == "e4m3":
        shape = pool.scales.shape[1:3] + (16,)
        one = torch.zeros(shape, dtype=torch.bool, device="cuda")
        one[int(pool.block_tables[0, 20]), 1, 7] = True
        ks, vs = set_exponents(pool, lens, pick(g, (-9, -8), shape), torch.where(one, v_exp, -9))
    q = torch.randn((cu[-1], 8, d), generator=g, device="cuda").to(DT[dtype])
    out = q.clone()
    if single:
        got = pool.decode(0, out, out=out, window=0 if cache == "e4m3" else 1000)
    else:
        got = pool.attend_chunk(0, out, torch.tensor(cu, dtype=torch.int32, device="cuda"), out=out)
    pool.check()
    assert got is out
    check(out, q, cu, ks, vs, 0, 0, HALF[DT[dtype]])


def test_a_captured_call_that_is_done_over_at_times(cuda_device):
    """A captured f16 chunk over 8 bits, replayed over rows that f16 holds, over one that it does not, and back;
    a second graph over the same pool in between."""
    lens, new = [700, 90], [40, 90]
    pool, _, _ = make_pool(torch.float16, lens, 2, 128, 16, 56, "e4m3")
    g = torch.Generator(device="cuda").manual_seed(10)
    shape = pool.scales.shape[1:3] + (16,)
    exps = pick(g, (-9, -8), shape)
    one = torch.zeros(shape, dtype=torch.bool, device="cuda")
    one[int(pool.block_tables[0, 20]), 1, 7] = True
    q = torch.randn((130, 8, 128), generator=g, device="cuda").half()
    cu = [0, 40, 130]
    cud = torch.tensor(cu, dtype=torch.int32, device="cuda")
    pool.attend_chunk(0, q, cud)
    graphs = []
    for window in (0, 500):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = pool.attend_chunk(0, q, cud, window=window)
        graphs.append((graph, out, window))
    for v_exp in (-9, 12, -9, 9, -9):
        ks, vs = set_exponents(pool, lens, exps, torch.where(one, v_exp, -9))
        for graph, out, window in graphs:
            graph.replay()
            check(out, q, cu, ks, vs, window, 0, HALF[torch.float16])
    pool.check()


@pytest.mark.parametrize("cache,dtype", [("same", "bf16"), ("e4m3", "bf16"), ("e4m3", "f16"), ("same", "f32")])
def test_the_largest_batch(cuda_device, cache, dtype):
    """8192 sequences; one more is refused."""
    dtype, n = DT[dtype], 8192
    rng = np.random.RandomState(3)
    lens = rng.randint(0, 40, n)
    pool, ks, vs = make_pool(dtype, lens.tolist(), 1, 128, 16, 57, cache)
    new = np.minimum(lens, rng.randint(0, 4, n))
    cu = np.concatenate([[0], np.cumsum(new)])
    q = torch.randn((max(int(cu[-1]), n), 2, 128), device="cuda").to(dtype)
    out = pool.attend_chunk(0, q[:int(cu[-1])], torch.tensor(cu, dtype=torch.int32, device="cuda"))
    one = pool.decode(0, q[:n], window=25, sinks=2)
    pool.check()
    for b in [0, 1, n - 1, *rng.randint(0, n, 100).tolist()]:
        a, e = int(cu[b]), int(cu[b + 1])
        check(out[a:e], q[a:e], [0, e - a], ks[b:b + 1], vs[b:b + 1], 0, 0, HALF[dtype])
        check(one[b:b + 1], q[b:b + 1], [0, 1], ks[b:b + 1], vs[b:b + 1], 25, 2, HALF[dtype])
    more = type(pool)(1, 1, 128, 4, n + 1, 1, dtype=dtype)
    with pytest.raises(ValueError, match="8192"):
        more.decode(0, torch.zeros((n + 1, 2, 128), dtype=dtype, device="cuda"), window=25)


@pytest.mark.parametrize("cache,d,single,generic", KERNELS)
def test_a_million_tokens(cuda_device, cache, d, single, generic):
    """One sequence past 2^20 tokens, the whole of it and a window with sinks: half of the keys have a V of 1, the
    others 0, and a far stronger score, so that the sum over all of them is known."""
    from snapmind_b200 import PagedKVPool, QuantizedKVPool

    n, t = 2**20 + 777, 1 if single else 5
    blocks = (n + 15) // 16
    pool = (QuantizedKVPool if cache == "e4m3" else PagedKVPool)(1, 1, d, blocks, 1, blocks, dtype=torch.bfloat16)
    pool.reserve(n, batch=1)
    k = torch.zeros((1, 1, n, d), device="cuda", dtype=torch.bfloat16)
    v = torch.zeros_like(k)
    k[:, :, ::2, 3], v[:, :, 1::2] = 4.0, 1.0
    pool.append(0, k, v)
    q = torch.zeros((t, 4, d), device="cuda").bfloat16()
    q[:, :, 3] = 4.0
    scale = math.log(3) / 16  # even positions weigh 3, odd ones 1
    cu = torch.tensor([0, t], dtype=torch.int32, device="cuda")
    for window, sinks in ((0, 0), (2**19 + 1, 9)):
        if single and cache == "same" and not window:
            window = 2**30
        if single:
            out = pool.decode(0, q, scale=scale, window=window, sinks=sinks, force_generic=generic)
        else:
            out = pool.attend_chunk(0, q, cu, scale=scale, window=window, sinks=sinks, force_generic=generic)
        for i in range(t):
            pos = np.arange(n - t + i + 1)
            pos = pos[(pos > n - t + i - window) | (pos < sinks)] if window else pos
            odd, even = int((pos % 2).sum()), int((pos % 2 == 0).sum())
            want = odd / (odd + 3 * even)
            # the output's rounding, the weights' (all odd ones alike), the sums' and the scores' as in the other file
            assert abs(float(out[i].double().mean()) - want) <= want * (2 * 2.0**-8 + 2.0**-12)
            assert (out[i] == out[i, 0, 0]).all()
    pool.check()
