"""Cases of the paged-cache operators for chunks, windows and 8-bit caches, and their plain forms.

* ``chunk``: attention of a ragged batch of new tokens over a paged cache
  (``PagedKVPool.attend_chunk``, ``QuantizedKVPool.attend_chunk``): query i of the
  n new tokens of a sequence of L cached tokens stands at position L - n + i and
  sees the positions p up to its own, with a window w only p > its own - w or
  p < sinks.
* ``decode``: one token per sequence with a window and sinks
  (``PagedKVPool.decode(window=, sinks=)``), or over an 8-bit cache
  (``QuantizedKVPool.decode``).
* ``quant``: rows quantised as they are written and read back
  (``QuantizedKVPool.append`` and ``gather``): a row x of one token and head is
  held as e4m3 values c = x / 2^e, rounded to nearest even, with the smallest
  exponent e in [-100, 120] for which max |x| <= 448 * 2^e.

Sizes are those of the cache shapes that this repository measures and tests: 32 query
heads over 8 kv heads of 128 (blocks of 16, contexts of 1024 to 8192 and of 32768
tokens, sinks of 4, windows of 1024 and 4096) and 32 over 4 of 64.
"""
import math
import random

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
E_MIN, E_MAX = -100, 120


def _case(name, op, **kw):
    c = dict(op=op, dtype="bf16", cache="same", hq=32, hkv=8, d=128, bs=16, layers=1, nseq=1, ctx_lo=1024,
             ctx_hi=8192, new_lo=1, new_hi=1, window=0, sinks=0, mix=1)
    c.update(kw)
    if name:
        c["name"] = name
    return c


def listed():
    return [
        # a few drafted tokens of every running sequence, checked at once
        _case("chunk_verify", "chunk", nseq=16, new_lo=5, new_hi=5),
        # a serving step that mixes pieces of prompts with single tokens
        _case("chunk_mixed", "chunk", nseq=9, new_lo=1, new_hi=513, ctx_lo=600, ctx_hi=8192, mix=2),
        # a piece of a long document
        _case("chunk_long", "chunk", new_lo=2048, new_hi=2048, ctx_lo=32768, ctx_hi=32768),
        # whole prompts of a small model held in 32 bits
        _case("chunk_prompt_f32", "chunk", dtype="f32", hkv=4, d=64, nseq=4, new_lo=256, new_hi=256, ctx_lo=256,
              ctx_hi=256),
        # a long prompt under a sliding window whose first tokens stay visible
        _case("chunk_window", "chunk", dtype="f16", nseq=2, new_lo=1001, new_hi=1024, ctx_lo=12000, ctx_hi=16384,
              window=4096, sinks=4, mix=3),
        # prompt pieces over an 8-bit cache
        _case("chunk_quant", "chunk", cache="e4m3", nseq=4, new_lo=130, new_hi=512, ctx_lo=1024, ctx_hi=8192, mix=4),
        # one user far into a text, with a window and sinks: latency
        _case("decode_window_one", "decode", ctx_lo=32700, ctx_hi=32768, window=1024, sinks=4, mix=5),
        # a full serving batch with a window and sinks
        _case("decode_window_batch", "decode", nseq=128, window=4096, sinks=4, mix=6),
        # a handful of users on an 8-bit cache: latency
        _case("decode_quant_few", "decode", cache="e4m3", nseq=4, mix=7),
        # a full serving batch on an 8-bit cache
        _case("decode_quant_batch", "decode", cache="e4m3", nseq=128, mix=8),
        # a few tokens of a few sequences written into an 8-bit cache and read back
        _case("quant_few", "quant", cache="e4m3", nseq=3, hkv=4, d=64, new_lo=7, new_hi=7),
        # prompts written into an 8-bit cache, several layers at once, and read back
        _case("quant_prompts", "quant", cache="e4m3", nseq=16, layers=4, new_lo=2049, new_hi=2049),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["chunk", "chunk", "decode", "decode", "quant"])
    mix = rng.randrange(1 << 30)
    hkv, group = rng.choice([(8, 4), (4, 8), (8, 1), (2, 6), (5, 3), (8, 4)])
    d = rng.choice([64, 128, 128])
    bs = rng.choice([16, 16, 32, 64])
    if op == "quant":
        return _case(None, op, dtype=rng.choice(["bf16", "bf16", "f16", "f32"]), cache="e4m3", hkv=hkv, hq=hkv, d=d,
                     bs=bs, nseq=_spread(rng, 1, 24), layers=rng.randint(1, 3), new_lo=(t := _spread(rng, 1, 1600)),
                     new_hi=t, mix=mix)
    window = rng.choice([0, 0, _spread(rng, 16, 4096)])
    sinks = rng.choice([0, 4, rng.randint(1, 40)]) if window else 0
    cache = rng.choice(["same", "e4m3"])
    if op == "decode":
        if cache == "same" and not window:
            window, sinks = _spread(rng, 16, 4096), 4
        hi = _spread(rng, 40, 8192)
        return _case(None, op, dtype=rng.choice(["bf16", "bf16", "f16"]), cache=cache, hkv=hkv, hq=hkv * group, d=d,
                     bs=bs, nseq=_spread(rng, 1, 100), ctx_lo=max(1, hi // 8), ctx_hi=hi, window=window, sinks=sinks,
                     mix=mix)
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    hi = _spread(rng, 40, 1024 if dtype == "f32" else 8192)
    new_hi = min(hi, _spread(rng, 1, 200 if dtype == "f32" else 700))
    return _case(None, op, dtype=dtype, cache="same" if dtype == "f32" else cache, hkv=hkv, hq=hkv * group, d=d,
                 bs=bs, nseq=_spread(rng, 1, 4 if dtype == "f32" else 12), ctx_lo=max(new_hi, hi // 4), ctx_hi=hi,
                 new_lo=max(1, new_hi // 3), new_hi=new_hi, window=window, sinks=sinks, mix=mix)


def _lengths(case):
    """Cached tokens (the new ones among them) and new tokens of every sequence; the case alone decides them."""
    r = random.Random(case["mix"])
    new = [r.randint(case["new_lo"], case["new_hi"]) for _ in range(case["nseq"])]
    if case["op"] == "quant":
        return list(new), new
    return [max(n, r.randint(case["ctx_lo"], case["ctx_hi"])) for n in new], new


def _quantise(x):
    """e4m3 values and exponents of rows: exact steps (a power-of-two scale), so 32 bits are enough."""
    x = x.float()
    a = x.abs().amax(-1)
    m, k = torch.frexp(a)  # a = m 2^k, m in [1/2, 1): a <= 448 2^e = 0.875 2^(e + 9)
    e = torch.where(m <= 0.875, k - 9, k - 8).clamp(E_MIN, E_MAX)
    e = torch.where(a > 0, e, torch.full_like(e, E_MIN))
    return torch.ldexp(x, -e.unsqueeze(-1)).to(torch.float8_e4m3fn), e


def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    lens, new = _lengths(case)
    h, d, bs = case["hkv"], case["d"], case["bs"]
    # channels of unequal size, as projections give them
    chan = torch.exp(0.5 * torch.randn((2, 1, h, 1, d), generator=g, device="cuda"))
    s = {"lens": lens, "new": new}
    if case["op"] == "quant":
        shape = (case["layers"], case["nseq"], h, new[0], d)
        for i, n in enumerate(("k_new", "v_new")):
            x = torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)
            s[n] = x.mul_(chan[i].unsqueeze(0)).to(dt)
        return s
    blocks = [(n + bs - 1) // bs for n in lens]
    total = sum(blocks)
    nb = total + total // 10 + 1
    perm = torch.randperm(nb, generator=g, device="cuda").cpu().numpy()
    tables = np.zeros((len(lens), max(blocks)), dtype=np.int64)
    at = 0
    for b, n in enumerate(blocks):
        tables[b, :n] = perm[at:at + n]
        at += n
    s["tables"], s["free"], s["nb"] = tables, perm[at:].copy(), nb
    holds = torch.zeros((nb, bs), dtype=torch.bool, device="cuda")  # slots that hold a token
    for b, n in enumerate(lens):
        row = torch.zeros(blocks[b] * bs, dtype=torch.bool)
        row[:n] = True
        holds[torch.from_numpy(tables[b, :blocks[b]]).cuda()] = row.view(blocks[b], bs).cuda()
    empty = ~holds.view(nb, 1, bs, 1)
    for i, n in enumerate(("k", "v")):
        x = torch.randn((nb, h, bs, d), generator=g, device="cuda", dtype=torch.float32).mul_(chan[i])
        if case["cache"] == "e4m3":
            c, e = _quantise(x)
            c.view(torch.uint8).masked_fill_(empty, 0x7F)  # whatever an unused slot holds
            s[n], s[n + "_exp"] = c, e.to(torch.int16)
        else:
            s[n] = x.masked_fill_(empty, float("nan")).to(dt)
        del x
    s["q"] = (1.5 * torch.randn((sum(new), case["hq"], d), generator=g, device="cuda")).to(dt)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if not own:
        return s
    from snapmind_b200 import PagedKVPool, QuantizedKVPool

    lens, nseq, bs = s["lens"], case["nseq"], case["bs"]
    quantised = case["cache"] == "e4m3"
    nb = s.get("nb", sum((n + bs - 1) // bs for n in lens))
    width = max((n + bs - 1) // bs for n in lens)
    pool = (QuantizedKVPool if quantised else PagedKVPool)(
        case["layers"], case["hkv"], case["d"], nb, max_seqs=nseq, max_blocks_per_seq=width, block_size=bs,
        dtype=DTYPES[case["dtype"]])
    s["pool"] = pool
    if case["op"] == "quant":
        pool.reserve(s["new"][0], batch=nseq)
        return s
    pool.set_state(s.pop("tables"), np.array(lens), s.pop("free"))
    if quantised:
        for i, n in enumerate(("k", "v")):
            getattr(pool, n)[0].view(torch.uint8).copy_(s.pop(n).view(torch.uint8))
            pool.scales[0, :, :, i].copy_((s.pop(n + "_exp") + 127).to(torch.uint8))
    else:
        for n in ("k", "v"):
            getattr(pool, n)[0].copy_(s.pop(n))
    if case["op"] == "chunk":
        s["cu"] = torch.tensor([0] + list(np.cumsum(s["new"])), dtype=torch.int32, device="cuda")
    return s


def _rows(s, name, b, dtype):
    """K or V of sequence b as [heads, tokens, dim], in `dtype`."""
    case, n = s["case"], s["lens"][b]
    ids = torch.from_numpy(s["tables"][b, :(n + case["bs"] - 1) // case["bs"]]).cuda()
    x = s[name][ids].to(dtype)
    if case["cache"] == "e4m3":
        x = torch.ldexp(x, s[name + "_exp"][ids].to(torch.int32).unsqueeze(-1))
    return x.permute(1, 0, 2, 3).reshape(case["hkv"], -1, case["d"])[:, :n]


def _attention(s):
    case = s["case"]
    group = case["hq"] // case["hkv"]
    out = torch.empty_like(s["q"])
    at = 0
    for b, (n, t) in enumerate(zip(s["lens"], s["new"])):
        k, v = _rows(s, "k", b, torch.float32), _rows(s, "v", b, torch.float32)
        q = s["q"][at:at + t].float().view(t, case["hkv"], group, case["d"])
        i = torch.arange(n - t, n, device="cuda").view(t, 1, 1)
        j = torch.arange(n, device="cuda").view(1, 1, n)
        sees = j <= i
        if case["window"]:
            sees = sees & ((j > i - case["window"]) | (j < case["sinks"]))
        step = case["hkv"] if t * group * n * case["hkv"] <= 1 << 27 else 1  # heads at once, by memory
        for h in range(0, case["hkv"], step):
            w = torch.matmul(q[:, h:h + step].permute(1, 0, 2, 3).reshape(step, t * group, -1),
                             k[h:h + step].transpose(1, 2)).view(step, t, group, n)
            w = (w * case["d"] ** -0.5).masked_fill_(~sees, float("-inf"))
            w = torch.exp(w - w.amax(-1, keepdim=True))
            o = torch.matmul(w.view(step, t * group, n), v[h:h + step]).view(step, t, group, -1)
            o = o / w.sum(-1, keepdim=True)
            out.view(-1, case["hkv"], group, case["d"])[at:at + t, h:h + step] = o.permute(1, 0, 2, 3).to(out.dtype)
        at += t
    return out


def run(state):
    case = state["case"]
    if own:
        pool = state["pool"]
        if case["op"] == "quant":
            pool.append(None, state["k_new"], state["v_new"])
            return pool.gather(batch=case["nseq"])
        if case["op"] == "decode":
            return pool.decode(0, state["q"], window=case["window"], sinks=case["sinks"])
        return pool.attend_chunk(0, state["q"], state["cu"], window=case["window"], sinks=case["sinks"])
    if case["op"] == "quant":
        got = []
        for n in ("k_new", "v_new"):
            c, e = _quantise(state[n])
            top = torch.finfo(state[n].dtype).max
            x = torch.ldexp(c.float(), e.unsqueeze(-1)).clamp_(-top, top)
            got.append(x.to(state[n].dtype).view(case["layers"], -1))
        return tuple(got)
    return _attention(state)


def _exact_quant(x, dtype):
    x = x.double()
    a = x.abs().amax(-1, keepdim=True)
    e = torch.full_like(a, E_MIN)
    for step in (128, 64, 32, 16, 8, 4, 2, 1):  # the smallest e with a <= 448 2^e, by bisection from below
        up = e + step
        e = torch.where((a > 448.0 * torch.exp2(up - 1)) & (up <= E_MAX), up, e)
    y = x / torch.exp2(e)
    # the spacing of e4m3 around |y|: 2^(floor(log2 |y|) - 3), and 2^-9 below 2^-6
    _, k = torch.frexp(y)
    grid = torch.exp2((k - 4).clamp(min=-9).double())
    y = torch.round(y / grid) * grid  # torch.round takes ties to even
    top = torch.finfo(dtype).max
    return (y * torch.exp2(e)).clamp(-top, top)


def exact(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if case["op"] == "quant":
        return tuple(torch.stack([_exact_quant(x, x.dtype).reshape(-1) for x in s[n]]) for n in ("k_new", "v_new"))
    group, w = case["hq"] // case["hkv"], case["window"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    at = 0
    for b, (n, t) in enumerate(zip(s["lens"], s["new"])):
        k, v = _rows(s, "k", b, torch.float64), _rows(s, "v", b, torch.float64)
        step = max(1, min(t, (1 << 26) // (n * case["hq"])))  # queries at once, by memory
        for t0 in range(0, t, step):
            pos = torch.arange(n - t + t0, n - t + min(t, t0 + step), device="cuda")
            hides = torch.arange(n, device="cuda")[None, :] > pos[:, None]
            if w:
                far = torch.arange(n, device="cuda")[None, :] <= pos[:, None] - w
                far[:, :case["sinks"]] = False
                hides = hides | far
            q = s["q"][at + t0:at + t0 + len(pos)].double()
            for h in range(case["hkv"]):
                z = torch.einsum("tgd,nd->gtn", q[:, h * group:(h + 1) * group], k[h]) / math.sqrt(case["d"])
                p = torch.softmax(z.masked_fill(hides, -math.inf), dim=-1)
                out[at + t0:at + t0 + len(pos), h * group:(h + 1) * group] = torch.einsum("gtn,nd->tgd", p, v[h])
        at += t
    return out


def _seen(n, t, window, sinks):
    """(tokens that some query sees, query and key pairs) of a sequence with n tokens, t of them new."""
    pairs = 0
    for i in range(n - t, n):
        lo = max(0, i - window + 1) if window else 0
        pairs += i - lo + 1 + min(sinks, lo)
    lo = max(0, n - t - window + 1) if window else 0
    return n - lo + min(sinks, lo), pairs


def work(case):
    esz = DTYPES[case["dtype"]].itemsize
    lens, new = _lengths(case)
    d = case["d"]
    row = d + 1 if case["cache"] == "e4m3" else d * esz  # one token and head of K, or of V
    if case["op"] == "quant":
        rows = 2 * case["layers"] * sum(new) * case["hkv"]
        return {"bytes": rows * (2 * d * esz + row), "flops": rows * d * 4}
    tokens = pairs = 0
    for n, t in zip(lens, new):
        a, b = _seen(n, t, case["window"], case["sinks"])
        tokens, pairs = tokens + a, pairs + b
    return {"bytes": 2 * tokens * case["hkv"] * row + 2 * sum(new) * case["hq"] * d * esz,
            "flops": 4 * pairs * case["hq"] * d}
