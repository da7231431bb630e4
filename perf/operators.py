"""Operators of a key/value cache held in 8 or 4 bits, as a serving step uses them: what is measured of them, their plain forms, and what they give in 64 bits.

* ``write``: queries and keys normed per head and rotated, keys and values quantised into their pages.  The outputs are the queries and what the written rows stand for;
* ``read``: tokens' keys and values out of the pages, in bfloat16;
* ``attend``: attention over the pages, one token of each sequence or several;
* ``prefix``: the same where groups of sequences share their first pages, which are read once for all.

A cache is four tensors, pages of codes and their scales (``kind``):

* ``int8``: k, v int8 [pages, heads, page, dim]; ks, vs float32 [pages, heads, page]: a value is its code times its token's scale, max / 127;
* ``mxfp4``: k, v uint8 [pages, heads, page, dim / 2], two e2m1 codes a byte, the even dimension's in the lower half; ks, vs uint8 [pages, heads, page, dim / 32]:
  powers of two, 2^(byte - 127), the smallest with max <= 7 scales over 32 dimensions.
"""
from __future__ import annotations

import math
import random

import torch

own = False

F64 = torch.float64
E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
LLAMA_8B, LLAMA_70B = dict(hq=32, hkv=8, dim=128), dict(hq=64, hkv=8, dim=128)


def listed():
    return [
        # one stream's next token, 8B heads
        dict(name="write_1", op="write", kind="int8", page=16, seqs=1, new=1, ctx=140, norm=True, rot=128, ragged=False, **LLAMA_8B),
        # a wave of 1024 streams, one token each, heads without norms, as Llama's
        dict(name="write_1024", op="write", kind="mxfp4", page=16, seqs=1024, new=1, ctx=120, norm=False, rot=128, ragged=True, **LLAMA_8B),
        # a prefill chunk of 16k tokens, 70B heads
        dict(name="write_prompt_16k", op="write", kind="int8", page=16, seqs=4, new=4096, ctx=4096, norm=True, rot=128, ragged=False, **LLAMA_70B),
        # cached histories of unequal lengths handed on in bfloat16: a few, and one of 128k tokens
        dict(name="read_5", op="read", kind="int8", page=16, seqs=5, ctx=117, ragged=True, **LLAMA_8B),
        dict(name="read_128k", op="read", kind="mxfp4", page=16, seqs=1, ctx=131071, ragged=False, **LLAMA_70B),
        # one verdict being written; a batch in the middle of its replies, unequal lengths; two investigations over 128k tokens each
        dict(name="attend_1", op="attend", kind="int8", page=16, seqs=1, new=1, ctx=140, ragged=False, **LLAMA_8B),
        dict(name="attend_64", op="attend", kind="int8", page=16, seqs=64, new=1, ctx=2048, ragged=True, **LLAMA_8B),
        dict(name="attend_128k", op="attend", kind="mxfp4", page=16, seqs=2, new=1, ctx=131000, ragged=False, **LLAMA_70B),
        # a prefill chunk behind cached histories
        dict(name="attend_prompt", op="attend", kind="int8", page=16, seqs=4, new=2048, ctx=4096, ragged=True, **LLAMA_8B),
        # a few streams on one template, three tokens each (a forced run of the reply)
        dict(name="prefix_9", op="prefix", kind="mxfp4", page=32, groups=1, seqs=9, new=3, prefix=496, own=45, ragged=True, **LLAMA_8B),
        # streams of one fleet: a common history of 2k tokens; 256 streams on two histories of 16k
        dict(name="prefix_64", op="prefix", kind="int8", page=16, groups=1, seqs=64, new=1, prefix=2048, own=120, ragged=True, **LLAMA_8B),
        dict(name="prefix_2x128", op="prefix", kind="mxfp4", page=16, groups=2, seqs=128, new=1, prefix=16384, own=300, ragged=True, **LLAMA_70B),
    ]


def draw(rng):
    def log(a, b):
        return int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))

    hq, hkv = rng.choice([(32, 8), (64, 8), (8, 1), (8, 2), (16, 16), (12, 4), (4, 2)])
    c = dict(op=rng.choice(["write", "read", "attend", "attend", "prefix", "prefix"]), kind=rng.choice(["int8", "mxfp4"]), page=rng.choice([16, 32, 64]),
             hq=hq, hkv=hkv, dim=rng.choice([64, 128, 128]), ragged=rng.random() < 0.7)
    if c["op"] == "write":
        c.update(seqs=log(1, 1024), norm=rng.random() < 0.5, rot=c["dim"] // rng.choice([1, 1, 2]))
        c.update(new=log(1, max(1, 16384 // c["seqs"])))
        c.update(ctx=c["new"] + log(1, 4096))
    elif c["op"] == "read":
        c.update(seqs=log(1, 64))
        c.update(ctx=log(1, 131071 // c["seqs"]))
    elif c["op"] == "attend":
        c.update(seqs=log(1, 128), new=rng.choice([1, 1, log(1, 16), log(16, 1024)]))
        c.update(ctx=c["new"] + log(1, 4096 if c["seqs"] * c["new"] > 64 else 131000 // c["seqs"]))
        c.update(seqs=max(1, min(c["seqs"], 4096 // c["new"])))
    else:
        c.update(groups=log(1, 4), new=rng.choice([1, 1, 1, log(1, 8)]), prefix=log(16, 16384 * 8 // max(8, hkv)), own=log(8, 500))
        c.update(seqs=log(2, 256 // c["groups"] // c["new"]))
    return c


# ---- inputs -----------------------------------------------------------------------------------------------------------------------------------------------


def sizes(case):
    """(lengths of the contexts, of them shared with others, new tokens) of the case's sequences: the same for every seed."""
    rng, least = random.Random(7919 * case["seqs"] + case.get("ctx", 0)), case.get("new", 1)

    def some(n, most):
        return [rng.randint(min(most, max(least, most // 4)), most) if case["ragged"] else most for _ in range(n)]

    if case["op"] == "prefix":
        whole = max(1, case["prefix"] // case["page"]) * case["page"]
        ctx = [whole + t for t in some(case["groups"] * case["seqs"], max(case["own"], least))]
    else:
        whole, ctx = 0, some(case["seqs"], case["ctx"])
    if case["op"] == "write":
        return ctx, whole, [min(least, c) for c in ctx]
    return ctx, whole, [rng.randint(1, least) if case["ragged"] else least for _ in ctx]


def tables(counts, shared, page, rng):
    """Pages of sequences: `counts` tokens each behind the pages `shared[i]` that it has in common with others; their numbers are in no order."""
    used = sum(-(-c // page) for c in counts) + len({p for s in shared for p in s})
    free = [p for p in range(used + 3)]
    rng.shuffle(free)
    names, rows = {}, []
    for c, s in zip(counts, shared):
        for p in s:
            if p not in names:
                names[p] = free.pop()
        rows.append([names[p] for p in s] + [free.pop() for _ in range(-(-c // page))])
    wide = max(len(r) for r in rows)
    return used + 3, torch.tensor([r + [0] * (wide - len(r)) for r in rows], dtype=torch.int32, device="cuda")


def quantised(x, kind):
    """(codes, scales, what they stand for) of x [.., dim] in float64."""
    if kind == "int8":
        s = (x.abs().amax(-1) / 127).float()
        d = s.double()[..., None]
        code = torch.where(d > 0, torch.round(x / torch.where(d > 0, d, 1.0)), 0.0).clamp(-127, 127)
        return code.to(torch.int8), s, code * d
    b = x.unflatten(-1, (-1, 32))
    m, e = torch.frexp(b.abs().amax(-1))                    # max = m 2^e, m in [.5, 1): 7 scales are .875 2^e' with e' = log2(scale) + 3
    e = torch.where(m > 0, e - 3 + (m > 0.875), -126).clamp(-126, 127)
    s = torch.ldexp(torch.ones_like(m), e)[..., None]
    a = b.abs() / s
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0)).to(F64)
    a = (torch.round(a / step) * step).clamp(max=6)
    code = (torch.searchsorted(torch.tensor(E2M1, dtype=F64, device=x.device), a) + 8 * (b < 0)).flatten(-2)
    return (code[..., ::2] + 16 * code[..., 1::2]).to(torch.uint8), (e + 127).to(torch.uint8), (torch.where(b < 0, -a, a) * s).flatten(-2)


def made(pages, case, g):
    """Pages of a cache that holds keys with a few large channels, and values."""
    shape = (pages, case["hkv"], case["page"], case["dim"])
    loud = 1 + 5 * (torch.rand(case["hkv"], 1, case["dim"], device="cuda", generator=g) < 0.03)
    k, ks, _ = quantised((torch.randn(shape, device="cuda", generator=g) * loud).to(torch.bfloat16).double(), case["kind"])
    v, vs, _ = quantised(torch.randn(shape, device="cuda", generator=g).to(torch.bfloat16).double(), case["kind"])
    return dict(k=k, v=v, ks=ks, vs=vs)


def prepare(case, seed):
    rng, g = random.Random(seed * 7919 + 1), torch.Generator(device="cuda").manual_seed(seed)
    hq, hkv, dim, page = case["hq"], case["hkv"], case["dim"], case["page"]

    def ints(v):
        return torch.tensor(v, dtype=torch.int32, device="cuda")

    ctx, whole, new = sizes(case)
    if case["op"] in ("write", "read"):
        pages, table = tables(ctx, [[]] * len(ctx), page, rng)
        new = ctx if case["op"] == "read" else new
        st = dict(case=case, table=table, pos=torch.cat([torch.arange(c - n, c, dtype=torch.int32) for c, n in zip(ctx, new)]).cuda(),
                  seq=torch.repeat_interleave(torch.arange(len(ctx), dtype=torch.int32), torch.tensor(new)).cuda())
        if case["op"] == "read":
            return dict(st, **made(pages, case, g))
        rot, rows = case["rot"], (pages, hkv, page)
        freq = 500000.0 ** (-torch.arange(0, rot, 2, dtype=F64) / rot)
        angle = torch.outer(torch.arange(max(ctx), dtype=F64), freq)
        st["cos_sin"] = torch.cat([angle.cos(), angle.sin()], 1).float().cuda()
        st["qkv"] = torch.randn(int(st["pos"].numel()), (hq + 2 * hkv) * dim, device="cuda", generator=g).to(torch.bfloat16)
        for w in ("q_norm", "k_norm"):
            st[w] = (1 + 0.2 * torch.randn(dim, device="cuda", generator=g)).to(torch.bfloat16) if case["norm"] else None
        if case["kind"] == "int8":
            st.update({c: torch.zeros(*rows, dim, dtype=torch.int8, device="cuda") for c in "kv"}, **{s: torch.zeros(rows, device="cuda") for s in ("ks", "vs")})
        else:
            st.update({c: torch.zeros(*rows, n, dtype=torch.uint8, device="cuda") for c, n in (("k", dim // 2), ("v", dim // 2), ("ks", dim // 32), ("vs", dim // 32))})
        return st
    shared = [[(i // case["seqs"], j) for j in range(whole // page)] for i in range(len(ctx))]
    pages, table = tables([c - whole for c in ctx], shared, page, rng)
    start = [sum(new[:i]) for i in range(len(new) + 1)]
    st = dict(case=case, table=table, ctx=ints(ctx), start=ints(start) if case["new"] > 1 else None, longest=max(ctx), widest=max(new),
              q=(2 * torch.randn(start[-1], hq, dim, device="cuda", generator=g)).to(torch.bfloat16), **made(pages, case, g))
    if case["op"] == "prefix":
        st["group"] = ints([i * case["seqs"] for i in range(case["groups"] + 1)])
        st["prefix"] = ints([whole] * case["groups"])
    return st


# ---- the operators ----------------------------------------------------------------------------------------------------------------------------------------


def run(st):
    op = st["case"]["op"]
    if own:
        from chronos import ops

        cache = ops.QuantKV(st["k"], st["v"], st["ks"], st["vs"])
        if op == "write":
            q = ops.norm_rope_kv_quant(st["qkv"], st["pos"], st["seq"], st["table"], st["cos_sin"], cache, st["case"]["hq"], st["q_norm"], st["k_norm"], eps=1e-6)
            return (q, *ops.quant_kv_read(cache, st["table"], st["pos"], st["seq"]))
        if op == "read":
            return ops.quant_kv_read(cache, st["table"], st["pos"], st["seq"])
        if op == "attend":
            return ops.quant_attention(st["q"], cache, st["table"], st["ctx"], st["start"])
        return ops.prefix_attention(st["q"], cache, st["table"], st["ctx"], st["group"], st["prefix"], st["start"])
    if op == "write":
        return plain_write(st)
    if op == "read":
        at = places(st)
        return plain_values(st["k"][at], st["ks"][at]).to(torch.bfloat16), plain_values(st["v"][at], st["vs"][at]).to(torch.bfloat16)
    return plain_attention(st)


def places(st):
    """(page, all heads, row) of the tokens in hand, [tokens, heads]."""
    pos, page = st["pos"].long(), st["case"]["page"]
    return st["table"][st["seq"].long(), pos // page].long()[:, None], torch.arange(st["case"]["hkv"], device="cuda")[None], (pos % page)[:, None]


def plain_values(code, scale):
    """What codes [.., row] and their scales stand for, float32."""
    if code.dtype == torch.int8:
        return code.float() * scale[..., None]
    grid = torch.tensor(E2M1 + [-x for x in E2M1], device=code.device)
    x = grid[torch.stack([code & 15, code >> 4], -1).flatten(-2).int()]
    return (x.unflatten(-1, (-1, 32)) * torch.exp2(scale.float() - 127)[..., None]).flatten(-2)


def plain_norm_rotation(x, w, cos_sin, pos):
    if w is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w.to(x.dtype)
    half = cos_sin.shape[1] // 2
    cos, sin = cos_sin[pos, None, :half].to(x.dtype), cos_sin[pos, None, half:].to(x.dtype)
    a, b = x[..., :half], x[..., half:2 * half]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., 2 * half:]], -1)


def plain_write(st):
    """Keys and values in 64 bits: those next to a border between two codes go by what 32 bits would lose."""
    case, pos = st["case"], st["pos"].long()
    x = st["qkv"].unflatten(1, (-1, case["dim"]))
    at, (q, k, v) = places(st), x.split([case["hq"], case["hkv"], case["hkv"]], 1)
    q = plain_norm_rotation(q.float(), st["q_norm"], st["cos_sin"], pos).to(torch.bfloat16)
    st["k"][at], st["ks"][at], k = quantised(plain_norm_rotation(k.double(), st["k_norm"], st["cos_sin"], pos), case["kind"])
    st["v"][at], st["vs"][at], v = quantised(v.double(), case["kind"])
    return q, k.to(torch.bfloat16), v.to(torch.bfloat16)


def plain_attention(st):
    """Every sequence's pages in a row, one product over all of them, exp and sums in float32; sequences of unequal lengths are filled up and masked."""
    case, q, ctx = st["case"], st["q"], st["ctx"].long()
    n, hkv, dim, page = ctx.numel(), case["hkv"], case["dim"], case["page"]
    group, start = case["hq"] // hkv, torch.arange(n + 1, device="cuda") if st["start"] is None else st["start"].long()
    new, wide = start.diff(), st["widest"]
    table = st["table"][:, :-(-st["longest"] // page)].long()
    i = torch.arange(wide, device="cuda")
    rows = (start[:-1, None] + i).clamp(max=q.shape[0] - 1)                                  # [n, wide]
    seen = torch.arange(table.shape[1] * page, device="cuda") <= (ctx - new)[:, None, None] + i[None, :, None]
    qs = q[rows].float().view(n, wide, hkv, group, dim).permute(0, 2, 3, 1, 4).reshape(n, hkv, group * wide, dim)
    s = qs @ plain_values(st["k"][table], st["ks"][table]).transpose(1, 2).reshape(n, hkv, -1, dim).transpose(2, 3) / math.sqrt(dim)
    s = s.view(n, hkv, group, wide, -1).masked_fill(~seen[:, None, None], -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True))
    p = (p / p.sum(-1, keepdim=True)).view(n, hkv, group * wide, -1)
    del s
    o = p @ plain_values(st["v"][table], st["vs"][table]).transpose(1, 2).reshape(n, hkv, -1, dim)
    o = o.view(n, hkv, group, wide, dim).permute(0, 3, 1, 2, 4).reshape(n, wide, hkv * group, dim)
    return o[i < new[:, None]].to(torch.bfloat16)


# ---- what they cannot do without, and what they give in 64 bits ---------------------------------------------------------------------------------------------


def work(case):
    hq, hkv, dim = case["hq"], case["hkv"], case["dim"]
    row = 2 * hkv * (dim + 4 if case["kind"] == "int8" else dim // 2 + dim // 32)             # bytes of a token's keys and values with their scales
    ctx, whole, new = sizes(case)
    if case["op"] == "read":
        return dict(bytes=sum(ctx) * (row + 4 * hkv * dim), flops=2 * hkv * dim * sum(ctx))
    if case["op"] == "write":
        return dict(bytes=sum(new) * (2 * dim * (2 * hq + 2 * hkv) + row + 4 * case["rot"] + 4 * hkv * dim), flops=10 * sum(new) * dim * (hq + 2 * hkv))
    once = sum(ctx) - (len(ctx) - case.get("groups", 0)) * whole
    return dict(bytes=once * row + 4 * sum(new) * hq * dim, flops=4 * hq * dim * sum(m * c - m * (m - 1) // 2 for c, m in zip(ctx, new)))


def exact_values(code, scale):
    if code.dtype == torch.int8:
        return code.double() * scale.double().unsqueeze(-1)
    nib = torch.stack([code.long() % 16, code.long() // 16], -1).reshape(*code.shape[:-1], -1)
    size, sign = nib % 8, 1.0 - 2.0 * (nib // 8)
    size = torch.where(size < 2, size * 0.5, (1 + (size % 2) * 0.5) * 2.0 ** (torch.div(size, 2, rounding_mode="floor") - 1).double())
    return sign * size * (2.0 ** (scale.double() - 127)).repeat_interleave(32, -1)


def exact_held(x, kind):
    """x as the cache holds it: the nearest of the values that its scale allows."""
    if kind == "int8":
        s = (x.abs().amax(-1, keepdim=True) / 127).float().double()
        return torch.where(s > 0, torch.floor(x / s.clamp(min=1e-300) + 0.5), 0.0) * s
    b = x.reshape(*x.shape[:-1], -1, 32)
    s = 2.0 ** torch.ceil(torch.log2((b.abs().amax(-1, keepdim=True) / 7).clamp(min=2.0 ** -126)))
    grid = torch.tensor(E2M1, dtype=F64, device=x.device)
    mid = (grid[1:] + grid[:-1]) / 2
    a = b.abs() / s
    down, up = torch.bucketize(a, mid), torch.bucketize(a, mid, right=True)                   # they differ on a border: the even one
    return (torch.sign(b) * grid[torch.where(down % 2 == 0, down, up)] * s).reshape(x.shape)


def exact(case, seed):
    st = prepare(case, seed)
    dim, page, hq, hkv = case["dim"], case["page"], case["hq"], case["hkv"]
    if case["op"] in ("write", "read"):
        pos, seq = st["pos"].long(), st["seq"].long()
        if case["op"] == "read":
            p = st["table"][seq, pos // page].long()
            return tuple(exact_values(st[c][p, :, pos % page], st[c + "s"][p, :, pos % page]) for c in "kv")
        x = st["qkv"].double().view(pos.numel(), hq + 2 * hkv, dim)
        q, k, v = x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:]
        half = case["rot"] // 2
        turn = torch.complex(st["cos_sin"][pos, :half].double(), st["cos_sin"][pos, half:].double())[:, None]

        def turned(x, w):
            if w is not None:
                x = x / torch.sqrt(x.pow(2).sum(-1, keepdim=True) / dim + 1e-6) * w.double()
            z = torch.complex(x[..., :half], x[..., half:2 * half]) * turn
            return torch.cat([z.real, z.imag, x[..., 2 * half:]], -1)

        return turned(q, st["q_norm"]), exact_held(turned(k, st["k_norm"]), case["kind"]), exact_held(v, case["kind"])
    if st["q"].shape[0] * hq * st["longest"] * dim > 2e12:
        return None
    ctx, out = st["ctx"].tolist(), []
    start = list(range(len(ctx) + 1)) if st["start"] is None else st["start"].tolist()
    for b, c in enumerate(ctx):
        pages = st["table"][b, :-(-c // page)].long()
        k, v = (exact_values(st[x][pages], st[x + "s"][pages]).transpose(0, 1).reshape(hkv, -1, dim)[:, :c] for x in "kv")
        q = st["q"][start[b]:start[b + 1]].double()
        m, heads = q.shape[0], []
        hidden = torch.arange(c, device="cuda")[None] > torch.arange(c - m, c, device="cuda")[:, None]
        for h in range(hq):
            s = (k[h // (hq // hkv)] @ q[:, h].T).T / math.sqrt(dim)
            heads.append(torch.softmax(s.masked_fill(hidden, -math.inf), -1) @ v[h // (hq // hkv)])
        out.append(torch.stack(heads, 1))
    return torch.cat(out)
