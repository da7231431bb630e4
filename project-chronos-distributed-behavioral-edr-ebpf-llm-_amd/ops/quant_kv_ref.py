"""PyTorch references of the operators of a key/value cache in 8 or 4 bits (csrc/kernels/quant_kv.hip, quant_attention.hip): the CPU path, with the
kernels' layouts, roundings and rules for what is not there."""
from __future__ import annotations

import torch

E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def encode(x: torch.Tensor, kind: str):
    """(codes, scales) of rows x [.., D] (float64): layout and rules in csrc/include/chronos_quant_kv.h."""
    whole = torch.isfinite(x).all(-1)
    x = torch.where(whole[..., None], x, 0.0)
    if kind == "int8":
        s = (x.abs().amax(-1) / 127).float()
        d = s.double()[..., None]
        code = torch.where(d > 0, torch.round(x / torch.where(d > 0, d, 1.0)), 0.0).clamp(-127, 127)
        return code.to(torch.int8), torch.where(whole, s, float("nan"))
    b = x.unflatten(-1, (-1, 32))
    m, e = torch.frexp(b.abs().amax(-1))  # the maximum is m 2^e, m in [.5, 1), and at most 7 scales = .875 2^(log2(scale) + 3)
    e = torch.where(m > 0, e - 3 + (m > 0.875), -126).clamp(-126, 125)
    a = b.abs() / torch.ldexp(torch.ones_like(m), e)[..., None]
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0)).to(a.dtype)
    a = (torch.round(a / step) * step).clamp(max=6)
    code = (torch.searchsorted(torch.tensor(E2M1, dtype=a.dtype, device=a.device), a) + 8 * (b < 0)).flatten(-2)
    return (code[..., ::2] + 16 * code[..., 1::2]).to(torch.uint8), torch.where(whole[..., None], e + 127, 255).to(torch.uint8)


def decode(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """float32 of codes [.., row] and their scales."""
    if codes.dtype == torch.int8:
        return codes.float() * scales[..., None]
    grid = torch.tensor(E2M1 + tuple(-x for x in E2M1), device=codes.device)
    x = grid[torch.stack([codes & 15, codes >> 4], -1).flatten(-2).long()].unflatten(-1, (-1, 32))
    s = torch.where(scales > 252, float("nan"), torch.ldexp(torch.ones((), device=codes.device), scales.int() - 127))
    return (x * s[..., None]).flatten(-2)


def places(cache, block_table, pos, tok_seq, positions=None):
    """(whether each token has a place, its page, its row there)."""
    pages, _, page, _ = cache.k.shape
    pos, seq = pos.long(), tok_seq.long()
    ok = (pos >= 0) & (seq >= 0) & (seq < block_table.shape[0]) & (pos // page < block_table.shape[1])
    if positions is not None:
        ok &= pos < positions
    if block_table.numel() == 0:
        return ok, torch.zeros_like(pos), pos % page
    blk = block_table[torch.where(ok, seq, 0), torch.where(ok, pos // page, 0)].long()
    return ok & (blk >= 0) & (blk < pages), blk, pos % page


def norm_rope_kv_quant(qkv, pos, tok_seq, block_table, cos_sin, cache, hq, q_norm, k_norm, eps):
    hkv, D = cache.heads, cache.head_dim
    x = qkv.unflatten(1, (-1, D))
    ok, blk, row = places(cache, block_table, pos, tok_seq, cos_sin.shape[0])
    cs = cos_sin[torch.where(ok, pos.long(), 0)][:, None]
    half = cos_sin.shape[1] // 2

    def turned(x, w):
        if w is not None:
            x = x / torch.sqrt(x.double().pow(2).mean(-1, keepdim=True) + eps).to(x.dtype) * w.to(x.dtype)
        c, s = cs[..., :half].to(x.dtype), cs[..., half:].to(x.dtype)
        a, b = x[..., :half], x[..., half:2 * half]
        return torch.cat([a * c - b * s, b * c + a * s, x[..., 2 * half:]], -1)

    q = torch.where(ok[:, None, None], turned(x[:, :hq].float(), q_norm), 0.0).to(torch.bfloat16)
    for codes, scales, y in ((cache.k, cache.ks, turned(x[:, hq:hq + hkv].double(), k_norm)), (cache.v, cache.vs, x[:, hq + hkv:].double())):
        c, s = encode(y, cache.kind)
        codes[blk[ok], :, row[ok]] = c[ok]
        scales[blk[ok], :, row[ok]] = s[ok]
    return q


def quant_kv_read(cache, block_table, pos, tok_seq):
    ok, blk, row = places(cache, block_table, pos, tok_seq)
    at = torch.where(ok, blk, 0), slice(None), row
    return tuple(torch.where(ok[:, None, None], decode(c[at], s[at]), 0.0).to(torch.bfloat16) for c, s in ((cache.k, cache.ks), (cache.v, cache.vs)))


def quant_attention(q, cache, block_table, ctx_len, q_start, scale):
    """A shared prefix changes nothing of what is computed, so the reference of the attention with groups is this one."""
    T, hq, D = q.shape
    pages, hkv, page, _ = cache.k.shape
    out = torch.zeros_like(q)
    B = ctx_len.numel()
    start = list(range(B + 1)) if q_start is None else [0] + q_start[1:B + 1].tolist()
    for b in range(B):
        n, ctx = start[b + 1] - start[b], min(int(ctx_len[b]), block_table.shape[1] * page)
        if n <= 0 or ctx <= 0:
            continue
        blk = block_table[b, :-(-ctx // page)].long()
        there = ((blk >= 0) & (blk < pages)).repeat_interleave(page)[:ctx]
        at = torch.where((blk >= 0) & (blk < pages), blk, 0)
        k, v = (decode(c[at], s[at]).transpose(0, 1).reshape(hkv, -1, D)[:, :ctx] for c, s in ((cache.k, cache.ks), (cache.v, cache.vs)))
        seen = there & (torch.arange(ctx) <= torch.arange(ctx - n, ctx)[:, None])
        bad = ~torch.isfinite(v).all(-1)                                   # a value of NaN is one for the whole row, and only where it is seen
        v = torch.where(bad[..., None], 0.0, v)
        qq = q[start[b]:start[b + 1]].float().view(n, hkv, -1, D).permute(1, 2, 0, 3)
        s = (qq @ k.transpose(1, 2)[:, None] * scale).masked_fill(~seen, float("-inf"))
        top = s.amax(-1, keepdim=True)
        p = torch.exp(s - torch.where(top == float("-inf"), 0.0, top))
        p = torch.where(seen & bad[:, None, None], float("nan"), p)
        l = p.sum(-1, keepdim=True)
        o = torch.where(l == 0, 0.0, (p / l) @ v[:, None])                 # no sum is larger than the largest value
        out[start[b]:start[b + 1]] = o.permute(2, 0, 1, 3).reshape(n, hq, D).to(q.dtype)
    return out
