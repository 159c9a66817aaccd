"""Cases of the operators of a paged cache that stays within a budget, and their plain forms.

* ``rope``: queries and keys normalised per head (y = x / sqrt(mean x^2 + eps) * w), rotated
  (z = y cos + rotate_half(y) sin at each token's own position) and stored with the values
  (``append_rope`` of ``PagedKVPool`` and ``QuantizedKVPool``).
* ``attend``: attention of the newest tokens over the cache (one per sequence: ``decode``, a ragged
  batch: ``attend_chunk``), which also adds to each cached token the weight that the call's queries gave
  it, summed over the queries and the query heads that share its kv head (``accumulate=True``).
* ``evict``: per layer, sequence and kv head the first ``sinks`` tokens, the newest ``recent`` and those with
  most accumulated weight (ties: the lowest index) stay, ``budget`` in all, in their order
  (``evict``): in place after new tokens came (``roll``), or as a copy beside the whole (``copy``).

Sizes are those of the cache shapes that this repository measures and tests: 32 query heads over 8 kv
heads of 128 (blocks of 16, contexts of 1024 to 8192 and of 32768 tokens) and 32 over 4 of 64.
"""
import math
import random

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
E_MIN, E_MAX = -100, 120
EPS = 1e-6
N_POS = 40960


def _case(name, op, **kw):
    c = dict(op=op, dtype="bf16", cache="same", hq=32, hkv=8, d=128, bs=16, layers=1, nseq=1, ctx_lo=1024,
             ctx_hi=8192, new_lo=1, new_hi=1, mix=1)
    if op == "attend":
        c.update(window=0, sinks=0)
    if op == "evict":
        c.update(form="copy", budget=1024, recent=64, sinks=4)
    c.update(kw)
    if name:
        c["name"] = name
    return c


def listed():
    return [
        # one user's next token, far into a text: latency
        _case("rope_one", "rope", ctx_lo=32700, ctx_hi=32768),
        # whole prompts of a few users
        _case("rope_prompts", "rope", nseq=4, ctx_lo=4096, ctx_hi=4096, new_lo=1537, new_hi=2560, mix=2),
        # short prompts of many users into an 8-bit cache, read back
        _case("rope_quant", "rope", dtype="f16", cache="e4m3", nseq=16, ctx_lo=1, ctx_hi=1, new_lo=129, new_hi=513, mix=3),
        # one user's next token over a long cache: latency
        _case("decode_one", "attend", ctx_lo=32700, ctx_hi=32768, mix=4),
        # a full serving batch
        _case("decode_batch", "attend", nseq=128, mix=5),
        # a serving batch on an 8-bit cache
        _case("decode_quant", "attend", dtype="f16", cache="e4m3", nseq=64, mix=6),
        # a few drafted tokens of every running sequence
        _case("chunk_verify", "attend", nseq=16, new_lo=5, new_hi=5, mix=7),
        # a piece of a long document
        _case("chunk_long", "attend", new_lo=2048, new_hi=2048, ctx_lo=32768, ctx_hi=32768),
        # whole prompts of a small model held in 32 bits
        _case("chunk_prompt_f32", "attend", dtype="f32", hkv=4, d=64, nseq=4, new_lo=256, new_hi=256, ctx_lo=256, ctx_hi=256),
        # running sequences that took 64 more tokens go back to their budget
        _case("evict_roll", "evict", form="roll", layers=4, nseq=32, new_lo=64, new_hi=64, budget=2048, recent=256, mix=8),
        # a long document's cache, all layers of a small model, thinned to an eighth beside the whole
        _case("evict_document", "evict", layers=16, ctx_lo=32768, ctx_hi=32768, budget=4096, recent=512, mix=9),
        # prompts of many users in an 8-bit cache, read back
        _case("evict_quant", "evict", cache="e4m3", layers=8, nseq=16, budget=1000, recent=100, mix=10),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rope", "attend", "attend", "attend", "evict"])
    mix = rng.randrange(1 << 30)
    hkv, group = rng.choice([(8, 4), (4, 8), (8, 1), (2, 6), (5, 3), (8, 4)])
    dtype, cache = rng.choice(["bf16", "bf16", "f16", "f32"]), rng.choice(["same", "same", "e4m3"])
    c = dict(dtype=dtype, cache=cache, hkv=hkv, hq=hkv * group, d=rng.choice([64, 128, 128]),
             bs=rng.choice([16, 16, 32, 64]), mix=mix)
    if op == "rope":
        new = _spread(rng, 1, 2000)
        ctx = (1, 1) if cache == "e4m3" else (new, new + _spread(rng, 1, 4096))  # 8-bit: whole prompts, read back
        return _case(None, op, nseq=_spread(rng, 1, 8), ctx_lo=ctx[0], ctx_hi=ctx[1],
                     new_lo=max(1, new // 2), new_hi=new, **c)
    hi = _spread(rng, 40, 8192)
    if op == "evict":
        budget = _spread(rng, 17, 2048)
        roll = rng.random() < 0.5
        recent = rng.randint(0, budget // 2)
        c["cache"] = "same" if roll else cache
        return _case(None, op, form="roll" if roll else "copy", layers=rng.randint(1, 4), nseq=_spread(rng, 1, 24),
                     ctx_lo=max(1, hi // 8), ctx_hi=hi, new_lo=(t := _spread(rng, 1, 300)), new_hi=t, budget=budget,
                     recent=recent, sinks=rng.choice([0, 4]) if recent + 4 <= budget else 0, **c)
    window = rng.choice([0, 0, 0, _spread(rng, 16, 4096)])
    sinks = rng.choice([0, 4, rng.randint(1, 40)]) if window else 0
    if rng.random() < 0.5:  # one token of each sequence
        top = hi // 4 + 1 if dtype == "f32" else hi
        return _case(None, op, nseq=_spread(rng, 1, 48), ctx_lo=max(1, top // 8), ctx_hi=top, window=window, sinks=sinks, **c)
    hi = min(hi, 1024) if dtype == "f32" else hi
    new = min(hi, _spread(rng, 1, 200 if dtype == "f32" else 700))
    return _case(None, op, nseq=_spread(rng, 1, 4 if dtype == "f32" else 8), ctx_lo=max(new, hi // 4), ctx_hi=hi,
                 new_lo=max(1, new // 3), new_hi=new, window=window, sinks=sinks, **c)


# ------------------------------------------------------------------ the case's lengths
def _lengths(case):
    """Cached tokens (the new ones among them) and new tokens of every sequence; the case alone decides them."""
    r = random.Random(case["mix"])
    new = [r.randint(case["new_lo"], case["new_hi"]) for _ in range(case["nseq"])]
    if case["op"] == "evict" and case["form"] == "roll":
        return [case["budget"] + t for t in new], new
    return [max(n if case["op"] != "evict" else 1, r.randint(case["ctx_lo"], case["ctx_hi"])) for n in new], new


def _blocks(n, bs):
    return (n + bs - 1) // bs


# ------------------------------------------------------------------ 8-bit rows
def _exponents(a):
    """The smallest e in [-100, 120] with a <= 448 2^e."""
    m, k = torch.frexp(a)  # a = m 2^k, m in [1/2, 1): a <= 448 2^e = 0.875 2^(e + 9)
    e = torch.where(m <= 0.875, k - 9, k - 8).clamp(E_MIN, E_MAX)
    return torch.where(a > 0, e, torch.full_like(e, E_MIN))


def _quantise(x):
    """e4m3 values and exponents of rows."""
    e = _exponents(x.abs().amax(-1))
    return torch.ldexp(x, -e.unsqueeze(-1)).to(torch.float8_e4m3fn), e


# ------------------------------------------------------------------ inputs
def _channels(case, g):
    """Channels of unequal size, as projections give them: [K and V][head][dim]."""
    return torch.exp(0.5 * torch.randn((2, case["hkv"], case["d"]), generator=g, device="cuda"))


def _cache(case, g, s, nb):
    """Blocks of K and V (and their exponents) of every layer, whatever the tables are."""
    chan = _channels(case, g)
    for i, n in enumerate(("k", "v")):
        parts = []
        for _ in range(case["layers"]):
            x = torch.randn((nb, case["hkv"], case["bs"], case["d"]), generator=g, device="cuda").mul_(chan[i].unsqueeze(1))
            parts.append(_quantise(x) if case["cache"] == "e4m3" else x.to(DTYPES[case["dtype"]]))
            del x
        if case["cache"] == "e4m3":
            s[n], s[n + "_exp"] = torch.stack([c for c, _ in parts]), torch.stack([e.to(torch.int32) for _, e in parts])
        else:
            s[n] = torch.stack(parts)


def _shuffled_tables(counts, nb, g):
    perm = torch.randperm(nb, generator=g, device="cuda").cpu().numpy()
    tables = np.zeros((len(counts), max(counts)), dtype=np.int64)
    at = 0
    for b, n in enumerate(counts):
        tables[b, :n] = perm[at:at + n]
        at += n
    return tables, perm[at:].copy()


def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt, h, d, bs, n = DTYPES[case["dtype"]], case["hkv"], case["d"], case["bs"], case["nseq"]
    lens, new = _lengths(case)
    s = {"case": case, "lens": lens, "new": new}
    randn = lambda *shape: torch.randn(shape, generator=g, device="cuda")  # noqa: E731
    if case["op"] == "evict":
        _evict_inputs(case, g, s)
    else:
        counts = [_blocks(x, bs) for x in lens]
        s["nb"] = sum(counts) + sum(counts) // 10 + 1
        s["tables"], s["free"] = _shuffled_tables(counts, s["nb"], g)
    total = sum(new)
    if case["op"] == "rope":
        chan = _channels(case, g)
        s["q_new"] = randn(total, case["hq"], d).to(dt)
        s["k_new"] = randn(total, h, d).mul_(chan[0]).to(dt)
        s["v_new"] = randn(total, h, d).mul_(chan[1]).to(dt)
        s["q_norm"], s["k_norm"] = (1 + 0.2 * randn(d)).to(dt), (1 + 0.2 * randn(d)).to(dt)
        inv = 10000.0 ** (-torch.arange(0, d, 2, device="cuda", dtype=torch.float64) / d)
        angles = torch.outer(torch.arange(N_POS, device="cuda", dtype=torch.float64), inv).repeat(1, 2)
        s["cos"], s["sin"] = angles.cos().float(), angles.sin().float()
        # tokens that were evicted before lie between a token's index in the cache and its position
        lost = torch.randint(0, 4096, (n,), generator=g, device="cuda").repeat_interleave(torch.tensor(new, device="cuda"))
        s["positions"] = torch.cat([torch.arange(a - t, a, device="cuda") for a, t in zip(lens, new)]) + lost
    if case["op"] == "attend":
        _cache(case, g, s, s["nb"])
        s["q"] = (1.5 * randn(total, case["hq"], d)).to(dt)
        # weight that a few such steps left
        s["mass"] = torch.empty((1, s["nb"], h, bs), device="cuda").exponential_(generator=g).square_()
        s["mass"].mul_(case["hq"] // h * total / sum(lens))
    s["seq"] = torch.repeat_interleave(torch.arange(n), torch.tensor(new)).cuda()
    s["step"] = torch.cat([torch.arange(t) for t in new]).cuda()  # a row's place among its sequence's new tokens
    s["cu"] = torch.tensor([0] + list(np.cumsum(new)), dtype=torch.int32, device="cuda")
    return s


def _evict_inputs(case, g, s):
    bs, h, n, L = case["bs"], case["hkv"], case["nseq"], case["layers"]
    lens, new, budget = s["lens"], s["new"], case["budget"]
    if case["form"] == "roll":
        # budget tokens each now; the blocks that the new ones take come next off the free stack
        held, extra = _blocks(budget, bs), [_blocks(x, bs) - _blocks(budget, bs) for x in lens]
        s["nb"] = n * held + sum(extra) + 3
        order = torch.randperm(s["nb"], generator=g, device="cuda").cpu().numpy()
        tables = np.zeros((n, held + max(extra)), dtype=np.int64)
        tables[:, :held] = order[:n * held].reshape(n, held)
        rest, at = order[n * held:], 0
        for b, x in enumerate(extra):
            tables[b, held:held + x] = rest[at:at + x]
            at += x
        s["tables"], s["free"] = tables, rest[::-1].copy()  # popped from the end
        s["k_new"] = torch.randn((L, n, h, new[0], case["d"]), generator=g, device="cuda").to(DTYPES[case["dtype"]])
        s["v_new"] = torch.randn((L, n, h, new[0], case["d"]), generator=g, device="cuda").to(DTYPES[case["dtype"]])
    else:
        # sequences 0 .. n - 1 are the copies (blocks 0, 1, ...), n .. 2 n - 1 the whole
        kept = [_blocks(min(x, budget), bs) for x in lens]
        s["nb"] = sum(kept) + sum(_blocks(x, bs) for x in lens) + 3
        whole, free = _shuffled_tables([_blocks(x, bs) for x in lens], s["nb"] - sum(kept), g)
        s["tables"] = np.zeros((2 * n, max(whole.shape[1], max(kept))), dtype=np.int64)
        at = 0
        for b, x in enumerate(kept):
            s["tables"][b, :x] = np.arange(at, at + x)
            at += x
        s["tables"][n:, :whole.shape[1]] = whole + at
        s["free"], s["copied"] = free + at, at
    _cache(case, g, s, s["nb"])
    s["mass"] = torch.empty((L, s["nb"], h, bs), device="cuda").exponential_(generator=g).square_()
    s["mass"].masked_fill_(torch.rand(s["mass"].shape, generator=g, device="cuda") < 0.1, 0.0)  # tokens that nobody looked at


def prepare(case, seed):
    s = _inputs(case, seed)
    # where the tokens of a sequence lie: block and slot of index j in its cache
    s["tab"] = torch.from_numpy(s["tables"]).cuda()
    s["len"] = torch.tensor(s["lens"], device="cuda")
    s["count"] = torch.tensor(s["new"], device="cuda")
    if case["op"] == "rope" and not own:
        s["k"] = torch.zeros((s["nb"], case["hkv"], case["bs"], case["d"]), dtype=DTYPES[case["dtype"]], device="cuda")
        s["v"] = torch.zeros_like(s["k"])
    if not own:
        return s
    from snapmind_b200 import PagedKVPool, QuantizedKVPool

    tables = s["tables"]
    quantised = case["cache"] == "e4m3"
    pool = (QuantizedKVPool if quantised else PagedKVPool)(
        case["layers"], case["hkv"], case["d"], s["nb"], max_seqs=len(tables), max_blocks_per_seq=tables.shape[1],
        block_size=case["bs"], dtype=DTYPES[case["dtype"]], mass=case["op"] != "rope")
    lens = s["lens"]
    if case["op"] == "evict":
        kept = [min(x, case["budget"]) for x in lens]
        lens = kept if case["form"] == "roll" else kept + lens
    pool.set_state(tables, np.array(lens), s["free"])
    if case["op"] == "rope":
        pool.k.view(torch.uint8).zero_(), pool.v.view(torch.uint8).zero_()
    else:
        for i, n in enumerate(("k", "v")):
            getattr(pool, n).view(torch.uint8).copy_(s.pop(n).view(torch.uint8))
            if quantised:
                pool.scales[:, :, :, i].copy_((s.pop(n + "_exp") + 127).to(torch.uint8))
        pool.mass.copy_(s.pop("mass"))
    s["pool"] = pool
    if case["op"] == "evict" and case["form"] == "copy":
        s["whole"], s["copies"] = list(range(case["nseq"], 2 * case["nseq"])), list(range(case["nseq"]))
    return s


# ------------------------------------------------------------------ plain forms
def _values(s, name, blocks, dtype):
    """K or V of the given blocks of layer 0, as values."""
    x = s[name][0][blocks].to(dtype)
    if s["case"]["cache"] == "e4m3":
        x = torch.ldexp(x, s[name + "_exp"][0][blocks].unsqueeze(-1))
    return x


def _place(s, seq, index):
    bs = s["case"]["bs"]
    return s["tab"][seq, index // bs], index % bs


def _packed(s, lens):
    """Sequence, head and index of the rows of a packed read of that many tokens."""
    h = s["case"]["hkv"]
    there = torch.arange(int(max(s["lens"])), device="cuda") < lens.view(-1, 1, 1).expand(-1, h, 1)
    return torch.nonzero(there, as_tuple=True)


def _plain_rope(s):
    case = s["case"]
    cos, sin = s["cos"][s["positions"]].unsqueeze(1), s["sin"][s["positions"]].unsqueeze(1)
    got = []
    for x, w in ((s["q_new"], s["q_norm"]), (s["k_new"], s["k_norm"])):
        x = x.float()
        y = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w.float()
        a, b = y.chunk(2, -1)
        got.append(y * cos + torch.cat((-b, a), -1) * sin)
    q, k = got
    q, dtype = q.to(s["q_new"].dtype), s["q_new"].dtype
    if case["cache"] == "e4m3":  # what a packed read gives: for each sequence (heads, tokens, dims)
        seq, head, i = _packed(s, s["count"])
        out = [q]
        for x in (k, s["v_new"].float()):
            c, e = _quantise(x)
            x = torch.ldexp(c.float(), e.unsqueeze(-1)).clamp_(-torch.finfo(dtype).max, torch.finfo(dtype).max)
            out.append(x.to(dtype)[s["cu"][seq] + i, head].view(1, -1))
        return tuple(out)
    index = (s["len"] - s["count"])[s["seq"]] + s["step"]
    blocks, slots = _place(s, s["seq"], index)
    s["k"][blocks, :, slots] = k.to(dtype)
    s["v"][blocks, :, slots] = s["v_new"]
    return q, s["k"], s["v"]


def _plain_attend(s):
    case = s["case"]
    n, h, d, group, w = case["nseq"], case["hkv"], case["d"], case["hq"] // case["hkv"], case["window"]
    t, size = max(s["new"]), s["tab"].shape[1] * case["bs"]
    k, v = (_values(s, x, s["tab"], torch.float32).transpose(1, 2).reshape(n, h, size, d) for x in ("k", "v"))
    q = torch.zeros((n, t, case["hq"], d), device="cuda")
    q[s["seq"], s["step"]] = s["q"].float()
    q = q.view(n, t, h, group, d).permute(0, 2, 1, 3, 4).reshape(n, h, t * group, d)
    z = torch.matmul(q, k.transpose(2, 3)).view(n, h, t, group, size)
    i = torch.arange(t, device="cuda").view(1, t, 1)
    at = (s["len"] - s["count"]).view(n, 1, 1) + i
    j = torch.arange(size, device="cuda").view(1, 1, size)
    sees = (j <= at) & (i < s["count"].view(n, 1, 1))
    if w:
        sees = sees & ((j > at - w) | (j < case["sinks"]))
    z.mul_(d ** -0.5).masked_fill_(~sees.view(n, 1, t, 1, size), float("-inf"))
    del k
    z.sub_(z.amax(-1, keepdim=True).clamp_(min=-1e30)).exp_()  # rows of no query: all zeros
    z.div_(z.sum(-1, keepdim=True).clamp_(min=1e-30))
    v = v.masked_fill_(~sees.any(1).view(n, 1, size, 1), 0.0)
    o = torch.matmul(z.view(n, h, t * group, size), v).view(n, h, t, group, d)
    out = o.permute(0, 2, 1, 3, 4).reshape(n, t, case["hq"], d)[s["seq"], s["step"]].to(s["q"].dtype)
    weight = z.sum((2, 3))  # [n, h, size]
    seq, index = torch.nonzero(j.view(1, size) < s["len"].view(n, 1), as_tuple=True)
    blocks, slots = _place(s, seq, index)
    mass = s["mass"][0]
    mass[blocks, :, slots] = mass[blocks, :, slots] + weight[seq, :, index]
    return out, mass


def _keep(mass, length, budget, recent, sinks):
    """Indexes that stay of weights [..., n], ascending, -1 behind the last; length broadcasts to mass[..., :1]."""
    n = mass.shape[-1]
    j = torch.arange(n, device=mass.device)
    key = torch.where((j < sinks) | (j >= length - recent), math.inf, mass).masked_fill(j >= length, -math.inf)
    first = torch.sort(key, dim=-1, descending=True, stable=True)[1][..., :budget]
    first = torch.sort(first.masked_fill(first >= length, n), dim=-1)[0]
    first = torch.nn.functional.pad(first, (0, budget - first.shape[-1]), value=n)
    return first.masked_fill(first == n, -1).to(torch.int32)


def _plain_evict(s):
    case = s["case"]
    n, L, bs, h = case["nseq"], case["layers"], case["bs"], case["hkv"]
    roll = case["form"] == "roll"
    if roll:
        index = (s["len"] - s["count"]).unsqueeze(1) + torch.arange(s["new"][0], device="cuda")
        blocks, slots = _place(s, torch.arange(n, device="cuda").unsqueeze(1), index)
        for x in ("k", "v"):
            s[x][:, blocks, :, slots] = s[x + "_new"].permute(1, 3, 0, 2, 4)
        s["mass"][:, blocks, :, slots] = 0.0
    src = s["tab"][-n:]
    mass = s["mass"][:, src].transpose(2, 3).reshape(L, n, h, -1)
    kept = _keep(mass, s["len"].view(1, n, 1, 1), case["budget"], case["recent"], case["sinks"])
    layer, seq, head, i = torch.nonzero(kept >= 0, as_tuple=True)
    j = kept[layer, seq, head, i].long()
    a = layer, src[seq, j // bs], head, j % bs
    b = layer, s["tab"][seq, i // bs], head, i % bs
    for x in [x for x in ("k", "v", "k_exp", "v_exp", "mass") if x in s]:
        # (8-bit codes move as bytes)
        y = s[x].view(torch.uint8) if s[x].dtype == torch.float8_e4m3fn else s[x]
        y[b] = y[a]
    if roll:
        return kept, s["k"], s["v"], s["mass"]
    m = s["mass"][:, :s["copied"]]
    if case["cache"] == "same":
        return kept, s["k"][:, :s["copied"]], s["v"][:, :s["copied"]], m
    # what a packed read of the copies gives: per layer, for each sequence (heads, tokens, dims)
    seq, head, i = _packed(s, torch.clamp(s["len"], max=case["budget"]))
    at = s["tab"][seq, i // bs], head, i % bs
    got = []
    for x in ("k", "v"):
        c, e = s[x][:, at[0], at[1], at[2]], s[x + "_exp"][:, at[0], at[1], at[2]]
        got.append(torch.ldexp(c.float(), e.unsqueeze(-1)).to(DTYPES[case["dtype"]]).reshape(L, -1))
    return kept, got[0], got[1], m


def run(state):
    case = state["case"]
    if not own:
        return {"rope": _plain_rope, "attend": _plain_attend, "evict": _plain_evict}[case["op"]](state)
    pool = state["pool"]
    one = max(state["new"]) == 1  # a token of each sequence
    if case["op"] == "rope":
        q = pool.append_rope(0, state["q_new"], state["k_new"], state["v_new"], state["cos"], state["sin"], state["positions"],
                             cu_new=None if one else state["cu"], q_norm=state["q_norm"], k_norm=state["k_norm"], eps=EPS)
        return (q, pool.k[0], pool.v[0]) if case["cache"] == "same" else (q, *pool.gather())
    if case["op"] == "attend":
        if one:
            out = pool.decode(0, state["q"], window=case["window"], sinks=case["sinks"], accumulate=True)
        else:
            out = pool.attend_chunk(0, state["q"], state["cu"], window=case["window"], sinks=case["sinks"], accumulate=True)
        return out, pool.mass[0]
    n = case["nseq"]
    if case["form"] == "roll":
        pool.reserve(state["new"][0], batch=n)
        pool.append(None, state["k_new"], state["v_new"])
        kept = pool.evict(case["budget"], recent=case["recent"], sinks=case["sinks"])
        return kept, pool.k, pool.v, pool.mass
    kept = pool.evict(case["budget"], recent=case["recent"], sinks=case["sinks"], seqs=state["whole"], into=state["copies"])
    m = pool.mass[:, :state["copied"]]
    if case["cache"] == "same":
        return kept, pool.k[:, :state["copied"]], pool.v[:, :state["copied"]], m
    k, v = pool.gather(batch=n)
    return kept, k, v, m


# ------------------------------------------------------------------ from the definitions, in 64 bits
def _exact_rope(s):
    case = s["case"]
    d, bs = case["d"], case["bs"]
    cos, sin = s["cos"].double(), s["sin"].double()
    rows = {}
    for name, w in (("q", s["q_norm"]), ("k", s["k_norm"])):
        x = s[name + "_new"].double()
        y = x / torch.sqrt((x * x).sum(-1, keepdim=True) / d + EPS) * w.double()
        z = torch.empty_like(y)
        half = d // 2
        c, sn = cos[s["positions"]][:, None], sin[s["positions"]][:, None]
        z[..., :half] = y[..., :half] * c[..., :half] - y[..., half:] * sn[..., :half]
        z[..., half:] = y[..., half:] * c[..., half:] + y[..., :half] * sn[..., half:]
        rows[name] = z
    rows["v"] = s["v_new"].double()
    got = [rows["q"]]
    for name in ("k", "v"):
        if case["cache"] == "e4m3":  # on the grid of the row's exponent: spacing 2^(floor(log2 |y|) - 3), 2^-9 at least
            x = rows[name]
            e = _exponents(x.abs().amax(-1)).unsqueeze(-1)
            y = torch.ldexp(x, -e)
            grid = torch.exp2((torch.frexp(y)[1] - 4).clamp(min=-9).double())
            x = torch.ldexp(torch.round(y / grid) * grid, e)
            got.append(torch.cat([x[a - t:a].transpose(0, 1).reshape(-1) for a, t in zip(np.cumsum(s["new"]), s["new"])]).view(1, -1))
            continue
        into = torch.zeros((s["nb"], case["hkv"], bs, d), dtype=torch.float64, device="cuda")
        at = 0
        for b, (n, t) in enumerate(zip(s["lens"], s["new"])):
            j = np.arange(n - t, n)
            into[torch.from_numpy(s["tables"][b, j // bs]).cuda(), :, torch.from_numpy(j % bs).cuda()] = rows[name][at:at + t]
            at += t
        got.append(into)
    return tuple(got)


def _exact_attend(s):
    case = s["case"]
    group, w, d, bs = case["hq"] // case["hkv"], case["window"], case["d"], case["bs"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    mass = s["mass"][0].double()
    at = 0
    for b, (n, t) in enumerate(zip(s["lens"], s["new"])):
        ids = torch.from_numpy(s["tables"][b, :_blocks(n, bs)]).cuda()
        k, v = (_values(s, x, ids, torch.float64).permute(1, 0, 2, 3).reshape(case["hkv"], -1, d)[:, :n] for x in ("k", "v"))
        pos = torch.arange(n - t, n, device="cuda")
        hides = torch.arange(n, device="cuda")[None, :] > pos[:, None]
        if w:
            far = torch.arange(n, device="cuda")[None, :] <= pos[:, None] - w
            far[:, :case["sinks"]] = False
            hides = hides | far
        for h in range(case["hkv"]):
            q = s["q"][at:at + t, h * group:(h + 1) * group].double()
            z = torch.einsum("tgd,nd->gtn", q, k[h]) / math.sqrt(d)
            p = torch.softmax(z.masked_fill(hides, -math.inf), dim=-1)
            out[at:at + t, h * group:(h + 1) * group] = torch.einsum("gtn,nd->tgd", p, v[h])
            gave = torch.zeros(len(ids) * bs, dtype=torch.float64, device="cuda")
            gave[:n] = p.sum((0, 1))
            mass[ids, h] += gave.view(-1, bs)
        at += t
    return out, mass


def _exact_evict(s):
    """One (layer, sequence, head) after the other."""
    case = s["case"]
    n, L, bs, budget = case["nseq"], case["layers"], case["bs"], case["budget"]
    roll = case["form"] == "roll"
    kept = torch.full((L, n, case["hkv"], budget), -1, dtype=torch.int32, device="cuda")
    store = {x: s[x].clone() if x == "mass" else s[x].to(torch.float64) for x in ("k", "v", "mass")}
    if case["cache"] == "e4m3":
        for x in ("k", "v"):
            store[x] = torch.ldexp(store[x], s[x + "_exp"].unsqueeze(-1))
    packed = {"k": [], "v": []}
    for b in range(n):
        size = s["lens"][b]
        j = np.arange(size)
        tab = s["tables"][b if roll else n + b]
        blk, slot = torch.from_numpy(tab[j // bs]).cuda(), torch.from_numpy(j % bs).cuda()
        m = min(size, budget)
        to = np.arange(m)
        tb, ts = torch.from_numpy(s["tables"][b][to // bs]).cuda(), torch.from_numpy(to % bs).cuda()
        if roll:
            t = s["new"][b]
            for x in ("k", "v"):
                store[x][:, blk[-t:], :, slot[-t:]] = s[x + "_new"][:, b].double().permute(2, 0, 1, 3)
            store["mass"][:, blk[-t:], :, slot[-t:]] = 0.0
        for layer in range(L):
            weights = store["mass"][layer, blk, :, slot].t()  # [heads, size]
            must = torch.zeros(size, dtype=torch.bool, device="cuda")
            must[:case["sinks"]] = True
            must[size - min(size, case["recent"]):] = True
            # order: forced first, then by weight, then by index
            order = torch.argsort(-weights.double() - must.double() * 1e30, dim=-1, stable=True)[:, :m]
            order = torch.sort(order, dim=-1)[0]
            kept[layer, b, :, :m] = order.to(torch.int32)
            heads = torch.arange(case["hkv"], device="cuda").unsqueeze(1)
            for x in ("k", "v", "mass"):
                rows = store[x][layer, blk[order], heads, slot[order]]
                store[x][layer, tb, heads, ts] = rows
    if roll:
        return kept, store["k"], store["v"], store["mass"].double()
    m = store["mass"][:, :s["copied"]].double()
    if case["cache"] == "same":
        return kept, store["k"][:, :s["copied"]], store["v"][:, :s["copied"]], m
    for x in ("k", "v"):
        for b in range(n):
            to = np.arange(min(s["lens"][b], budget))
            tb, ts = torch.from_numpy(s["tables"][b][to // bs]).cuda(), torch.from_numpy(to % bs).cuda()
            packed[x].append(store[x][:, tb, :, ts].permute(1, 2, 0, 3).reshape(L, -1))
    return kept, torch.cat(packed["k"], 1), torch.cat(packed["v"], 1), m


def exact(case, seed):
    s = _inputs(case, seed)
    return {"rope": _exact_rope, "attend": _exact_attend, "evict": _exact_evict}[case["op"]](s)


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    esz, d, h, bs = DTYPES[case["dtype"]].itemsize, case["d"], case["hkv"], case["bs"]
    lens, new = _lengths(case)
    row = d + 1 if case["cache"] == "e4m3" else d * esz  # one token and head of K, or of V, in the cache
    if case["op"] == "rope":
        t = sum(new)
        read = t * (case["hq"] + 2 * h) * d * esz + t * 2 * d * 4
        return {"bytes": read + t * (case["hq"] * d * esz + 2 * h * row), "flops": t * (case["hq"] + h) * d * 7}
    if case["op"] == "attend":
        tokens = pairs = 0
        for n, t in zip(lens, new):
            w = case["window"] or n
            lo = max(0, n - t - w + 1)
            tokens += n - lo + min(case["sinks"], lo)
            first = np.maximum(0, np.arange(n - t, n) - w + 1)
            pairs += int((np.arange(n - t, n) - first + 1 + np.minimum(case["sinks"], first)).sum())
        return {"bytes": 2 * tokens * h * row + 2 * sum(new) * case["hq"] * d * esz + tokens * h * 8,
                "flops": 4 * pairs * case["hq"] * d}
    heads = case["layers"] * h
    kept = [min(n, case["budget"]) for n in lens]
    if case["form"] == "roll":  # new rows in and out, all weights, at least the newest rows move up
        moved = sum(min(case["recent"], x) for x in kept)
        return {"bytes": heads * (sum(new) * 4 * row + sum(lens) * 4 + moved * (4 * row + 8) + sum(kept) * 4),
                "flops": heads * sum(lens)}
    back = 2 * d * (1 + esz) * sum(kept) if case["cache"] == "e4m3" else 0
    return {"bytes": heads * (sum(lens) * 4 + sum(kept) * (4 * row + 4 + 4) + back), "flops": heads * sum(lens)}
