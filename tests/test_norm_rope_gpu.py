"""Norm, rotation and store in one pass, against the formula in 64 bits.

Tolerances (before any run).  With u = 2^-24: a sum of D squares in f32 is off by at most D u of itself, its root's
inverse by half that and three roundings, y by two more, and z = y cos + y' sin by three roundings of
|y cos| + |y' sin|: e = (D / 2 + 9) u (|y cos| + |y' sin|).  A value stored in a type adds half a step of it; in an 8-bit row
of exponent x half a step of e4m3: 2^-4 |z| or 2^(x - 10)."""
import numpy as np
import pytest
import torch

from test_chunk_gpu import DT, HALF

pytestmark = pytest.mark.gpu

U = 2.0**-24


def tables(n_pos, rot, device="cuda"):
    inv = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / max(rot, 1))
    a = torch.outer(torch.arange(n_pos, dtype=torch.float64), inv).repeat(1, 2)
    return a.cos().float().to(device).contiguous(), a.sin().float().to(device).contiguous()


def reference(x, w, cos, sin, pos, eps):
    """(z, f32 tolerance): x [T, heads, D]."""
    d, rot = x.shape[-1], cos.shape[1]
    y = x.double()
    if w is not None:
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps) * w.double()
    z, a = y.clone(), y.abs()
    c, s = cos.double()[pos].unsqueeze(1), sin.double()[pos].unsqueeze(1)
    h = rot // 2
    y0, y1 = y[..., :h], y[..., h:rot]
    z[..., :h] = y0 * c[..., :h] - y1 * s[..., :h]
    z[..., h:rot] = y1 * c[..., h:] + y0 * s[..., h:]
    a[..., :h] = (y0 * c[..., :h]).abs() + (y1 * s[..., :h]).abs()
    a[..., h:rot] = (y1 * c[..., h:]).abs() + (y0 * s[..., h:]).abs()
    return z, (d / 2 + 9) * U * a


def close(got, z, tol, what):
    t = tol + HALF[got.dtype] * (z.abs() + tol) + (2.0**-25 if got.dtype == torch.float16 else 1e-38)
    err = (got.double() - z).abs()
    assert (err <= t).all(), f"{what}: {float((err / t).max()):.2f} x the tolerance"


CASES = [
    # dtype, pool dtype, hq, hkv, d, rot, bs, lens, new (None: one each), norms: None, "d" or "hd"
    ("bf16", "bf16", 32, 8, 128, 128, 16, [40, 700, 5], [3, 513, 0], "d"),
    ("bf16", "bf16", 32, 8, 128, 128, 16, [1, 700, 16, 17], None, "hd"),
    ("f16", "e4m3", 32, 8, 128, 128, 16, [40, 700, 5], [40, 13, 1], "d"),
    ("f32", "f32", 32, 4, 64, 64, 32, [33, 70], [33, 2], "d"),
    ("f32", "e4m3", 6, 2, 64, 32, 16, [33, 70], None, None),
    ("bf16", "f32", 3, 3, 256, 256, 16, [33], [33], "hd"),
    ("bf16", "f16", 4, 1, 80, 48, 16, [33, 1], [9, 1], "d"),
    ("f16", "bf16", 71, 1, 96, 96, 12, [33, 9], [9, 9], "d"),
    ("bf16", "e4m3", 5, 5, 72, 40, 16, [33, 9], [9, 9], "d"),
    ("f32", "f32", 2, 2, 9, 6, 5, [33, 9], [9, 9], "hd"),
    ("bf16", "bf16", 2, 1, 10, 0, 5, [33, 9], [9, 9], "d"),
    ("f16", "e4m3", 2, 1, 10, 10, 5, [33, 9], [9, 9], "d"),
    ("bf16", "bf16", 2, 1, 320, 320, 16, [33, 9], [9, 9], "d"),
]


def build(case, seed=2, spread=False):
    from snapmind_b200 import PagedKVPool, QuantizedKVPool

    dtype, pool_dtype, hq, hkv, d, rot, bs, lens, new, norms = case
    cls = QuantizedKVPool if pool_dtype == "e4m3" else PagedKVPool
    blocks = [(n + bs - 1) // bs for n in lens]
    nb = sum(blocks) + 4
    perm = np.random.RandomState(seed).permutation(nb)
    tab = np.zeros((len(lens), max(blocks) + 1), np.int64)
    at = 0
    for b, n in enumerate(blocks):
        tab[b, :n] = perm[at:at + n]
        at += n
    pool = cls(2, hkv, d, nb, max_seqs=len(lens), max_blocks_per_seq=tab.shape[1], block_size=bs,
               dtype=DT[dtype] if pool_dtype == "e4m3" else DT[pool_dtype])
    pool.set_state(tab, np.array(lens), perm[at:])
    pool.k.view(torch.uint8).fill_(0x55), pool.v.view(torch.uint8).fill_(0x55)
    g = torch.Generator(device="cuda").manual_seed(seed)
    counts = [1] * len(lens) if new is None else new
    total, t = sum(counts), DT[dtype]
    randn = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    x = {"q": (3 * randn(total, hq, d)).to(t), "k": randn(total, hkv, d).to(t), "v": randn(total, hkv, d).to(t)}
    w = [None, None] if norms is None else [(1 + 0.3 * randn(*((h, d) if norms == "hd" else (d,)))).to(t) for h in (hq, hkv)]
    cos, sin = tables(3000, rot)
    pos = torch.randint(0, 3000, (total,), generator=g, device="cuda")
    cu = None if new is None else torch.tensor([0] + list(np.cumsum(new)), dtype=torch.int32, device="cuda")
    return pool, x, w, cos, sin, pos, cu, counts


def stored(pool, layer, which, b, first, n):
    """(values [n, heads, D] f64, exponents [n, heads] or None) of indexes first .. first + n - 1."""
    bs = pool.block_size
    j = torch.arange(first, first + n, device="cuda")
    blocks, slots = pool.block_tables[b].long()[j // bs], j % bs
    x = (pool.k, pool.v)[which][layer][blocks, :, slots].double()
    if not pool.quantised:
        return x, None
    e = pool.scales[layer, :, :, which][blocks, :, slots].double() - 127
    return x * torch.exp2(e).unsqueeze(-1), e


def check_stored(pool, layer, z, tol, v, counts):
    lens = [int(n) for n in pool.host_lens]
    at = 0
    for b, t in enumerate(counts):
        for which, (want, off) in enumerate(((z, tol), (v.double(), torch.zeros_like(v, dtype=torch.float64)))):
            got, e = stored(pool, layer, which, b, lens[b] - t, t)
            w, o = want[at:at + t], off[at:at + t]
            if e is None:
                h = HALF[pool.dtype]
                lim = o + h * (w.abs() + o) + (2.0**-25 if pool.dtype == torch.float16 else 1e-38)
            else:
                lim = o + torch.maximum(2.0**-4 * (w.abs() + o), torch.exp2(e - 10).unsqueeze(-1))
                top = w.abs().amax(-1)
                slack = o.amax(-1)
                assert ((top - slack <= 448 * torch.exp2(e)) & ((top + slack > 448 * torch.exp2(e - 1)) | (e == -100))).all()
            err = (got - w).abs()
            assert (err <= lim).all(), f"sequence {b}, {'KV'[which]}: {float((err / lim).max()):.2f} x the tolerance"
        at += t


@pytest.mark.parametrize("case", CASES, ids=[f"{i}" for i in range(len(CASES))])
def test_append_rope(case):
    pool, x, w, cos, sin, pos, cu, counts = build(case)
    before = [t.clone() for t in (pool.k, pool.v)]
    out = pool.append_rope(1, x["q"], x["k"], x["v"], cos, sin, pos, cu_new=cu, q_norm=w[0], k_norm=w[1], eps=1e-5)
    pool.check()
    close(out, *reference(x["q"], w[0], cos, sin, pos, 1e-5), "q")
    z, tol = reference(x["k"], w[1], cos, sin, pos, 1e-5)
    check_stored(pool, 1, z, tol, x["v"], counts)
    # nothing else was written
    bs = pool.block_size
    for t, old in zip((pool.k, pool.v), before):
        same = torch.ones(t.shape[1:4], dtype=torch.bool, device="cuda")
        for b, n in enumerate(counts):
            j = torch.arange(int(pool.host_lens[b]) - n, int(pool.host_lens[b]), device="cuda")
            same[pool.block_tables[b].long()[j // bs], :, j % bs] = False
        assert torch.equal(t[0].view(torch.uint8), old[0].view(torch.uint8))
        assert torch.equal(t[1].view(torch.uint8)[same], old[1].view(torch.uint8)[same])


@pytest.mark.parametrize("case", CASES, ids=[f"{i}" for i in range(len(CASES))])
def test_without_norm_and_turn_it_is_an_append(case):
    """cos = 1, sin = 0 and no norms: the bits that append_packed stores, 8-bit codes and scales among them."""
    pool, x, _, cos, sin, pos, cu, counts = build(case)
    cu = torch.tensor([0] + list(np.cumsum(counts)), dtype=torch.int32, device="cuda") if cu is None else cu
    x["k"][0, 0, 1], x["v"][0, 0, 0] = float("inf"), float("nan")
    x["k"][-1, -1] = 0
    out = pool.append_rope(0, x["q"], x["k"], x["v"], torch.ones_like(cos), torch.zeros_like(sin), pos, cu_new=cu)
    pool.append_packed(1, x["k"], x["v"], cu)
    assert torch.equal(out, x["q"])
    lens = [int(n) for n in pool.host_lens]
    for b, t in enumerate(counts):
        for which in range(2):
            a, z = (stored(pool, layer, which, b, lens[b] - t, t) for layer in (0, 1))
            # inf x 0 in the rotation: NaN where a plain store keeps an infinity's neighbours
            fine = torch.isfinite(a[0])
            assert torch.equal(a[0][fine], z[0][fine]) and int((~fine).sum()) <= 2 * pool.head_dim
            if a[1] is not None:
                assert torch.equal(a[1], z[1])


@pytest.mark.parametrize("case", [CASES[0], CASES[3], CASES[7]], ids=["bf16", "f32", "f16"])
def test_strides_and_places(case):
    """Rows cut from one projection's output, in place, and from a layout of heads first: the same bits."""
    pool, x, w, cos, sin, pos, cu, counts = build(case)
    kw = dict(cu_new=cu, q_norm=w[0], k_norm=w[1])
    want = pool.append_rope(0, x["q"], x["k"], x["v"], cos, sin, pos, **kw)
    first = [t[0].clone() for t in (pool.k, pool.v)]

    def same(out):
        assert torch.equal(out, want)
        for t, f in zip((pool.k, pool.v), first):
            assert torch.equal(t[1].view(torch.uint8), f.view(torch.uint8))
            t[1].view(torch.uint8).fill_(0x55)

    hq, hkv = x["q"].shape[1], x["k"].shape[1]
    joint = torch.cat([x["q"], x["k"], x["v"]], 1)
    parts = joint.split([hq, hkv, hkv], 1)
    same(pool.append_rope(1, *parts, cos, sin, pos, **kw))
    into = parts[0]
    got = pool.append_rope(1, *parts, cos, sin, pos, out=into, **kw)
    assert got is into
    same(got)
    turned = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (x["q"], x["k"], x["v"])]
    same(pool.append_rope(1, *turned, cos, sin, pos, **kw))
    odd = [torch.cat([t, t[..., :1]], -1)[..., :-1] for t in (x["q"], x["k"], x["v"])]  # rows off 16-byte boundaries
    got = pool.append_rope(1, *odd, cos, sin, pos, **kw)
    z, tol = reference(x["q"], w[0], cos, sin, pos, 1e-6)
    close(got, z, tol, "odd rows")
    last = [torch.stack([t, t], -1)[..., 0] for t in (x["q"], x["k"], x["v"])]  # head dim not contiguous
    pool.k[1].view(torch.uint8).fill_(0x55), pool.v[1].view(torch.uint8).fill_(0x55)
    same(pool.append_rope(1, *last, cos, sin, pos, **kw))


def test_tokens_outside():
    """Rows of no sequence are rotated and not stored; positions outside the tables leave their token out."""
    pool, x, w, cos, sin, pos, cu, counts = build(CASES[0])
    total = pos.numel()
    before = pool.k.clone()
    cu[1:] = cu[1].item()  # only the first sequence's rows belong to one
    out = pool.append_rope(0, x["q"], x["k"], x["v"], cos, sin, pos, cu_new=cu, q_norm=w[0], k_norm=w[1])
    pool.check()
    close(out, *reference(x["q"], w[0], cos, sin, pos, 1e-6), "q")
    assert int((pool.k[0] != before[0]).any(-1).sum()) == 3 * 8
    pos[0], pos[1] = 3000, -1
    got = torch.full_like(x["q"], 7.0)
    pool.append_rope(1, x["q"], x["k"], x["v"], cos, sin, pos, cu_new=cu, q_norm=w[0], k_norm=w[1], out=got)
    assert (got[:2] == 7).all() and torch.equal(got[2:], out[2:])
    assert int((pool.k[1] != before[1]).any(-1).sum()) == 1 * 8 and total > 3
    with pytest.raises(RuntimeError, match="rotary position"):
        pool.check()


def test_refusals():
    pool, x, w, cos, sin, pos, cu, _ = build(CASES[0])
    q, k, v = x["q"], x["k"], x["v"]
    ok = dict(layer=0, q=q, k=k, v=v, cos=cos, sin=sin, positions=pos, cu_new=cu, q_norm=w[0], k_norm=w[1])
    for bad in (dict(layer=2), dict(layer=-1), dict(q=q[..., :64]), dict(k=k[:, :4]), dict(v=v[1:]), dict(cos=cos[:, :3].contiguous()),
                dict(cos=cos[:, :126].contiguous()), dict(cos=cos.double()), dict(cos=cos.t()), dict(positions=pos.int()),
                dict(positions=pos[1:]), dict(cu_new=cu.long()), dict(cu_new=None), dict(q_norm=w[0][:64]), dict(k_norm=w[1].float()),
                dict(eps=-1.0), dict(eps=float("nan")), dict(out=torch.empty_like(q[:1])), dict(out=q.float()),
                dict(cos=cos.cpu()), dict(positions=pos.cpu())):
        with pytest.raises(ValueError):
            pool.append_rope(**{**ok, **bad})
    with pytest.raises(TypeError):
        pool.append_rope(**{**ok, "k": k.float()})
    pool.append_rope(**{**ok, "q": q[:0], "k": k[:0], "v": v[:0], "positions": pos[:0], "cu_new": cu * 0})
