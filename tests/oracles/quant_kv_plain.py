"""The operators of a key/value cache in 8 or 4 bits, plain, in float64, token by token and row by row."""
import math

import torch

GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def quantise(x, kind):
    """(codes as whole numbers [.., D], scales) of rows x [.., D]: the nearest code by trying all of them, ties to the even one."""
    flat = x.double().reshape(-1, x.shape[-1])
    if kind == "int8":
        codes, scales = torch.zeros(flat.shape, dtype=torch.int64), torch.zeros(flat.shape[0])
        for i, r in enumerate(flat):
            if not torch.isfinite(r).all():
                scales[i] = float("nan")
                continue
            scales[i] = float(r.abs().max()) / 127
            if scales[i] > 0:
                codes[i] = torch.round(r / scales[i].double()).clamp(-127, 127).long()
        return codes.reshape(x.shape), scales.reshape(x.shape[:-1])
    grid = torch.tensor(GRID, dtype=torch.float64)
    codes, scales = torch.zeros(flat.shape, dtype=torch.int64), torch.zeros(flat.shape[0], flat.shape[1] // 32, dtype=torch.int64)
    for i, r in enumerate(flat):
        if not torch.isfinite(r).all():
            scales[i] = 255
            continue
        for b in range(flat.shape[1] // 32):
            part = r[32 * b:32 * b + 32]
            e = -126
            while e < 125 and float(part.abs().max()) > 7 * 2.0 ** e:
                e += 1
            off = (part.abs()[:, None] / 2.0 ** e - grid).abs()
            best = off.min(1).values
            tied = off == best[:, None]
            even = tied & (torch.arange(8) % 2 == 0)
            code = torch.where(even.any(1), even.int().argmax(1), tied.int().argmax(1))
            codes[i, 32 * b:32 * b + 32] = code + 8 * (part < 0)
            scales[i, b] = e + 127
    return codes.reshape(x.shape), scales.reshape(*x.shape[:-1], -1)


def whole_codes(cache):
    """(k, v) as the whole numbers that :func:`quantise` gives."""
    if cache.k.dtype == torch.int8:
        return cache.k.cpu().long(), cache.v.cpu().long()
    return tuple(torch.stack([c.cpu().long() & 15, c.cpu().long() >> 4], -1).flatten(-2) for c in (cache.k, cache.v))


def values(cache):
    """k, v [pages, heads, page, D] in float64."""
    out = []
    for c, s in zip(whole_codes(cache), (cache.ks.cpu(), cache.vs.cpu())):
        if cache.k.dtype == torch.int8:
            out.append(c.double() * s.double()[..., None])
        else:
            grid = torch.tensor(GRID + tuple(-g for g in GRID), dtype=torch.float64)
            f = torch.where(s == 255, float("nan"), 2.0 ** (s.double() - 127))
            out.append(grid[c] * f.repeat_interleave(32, -1))
    return out


def norm_rotation(x, w, eps, cos_sin, pos):
    """x [T, heads, D] of tokens at pos, in float64."""
    x = x.double()
    if w is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w.double()
    half = cos_sin.shape[1] // 2
    y = x.clone()
    for t, p in enumerate(pos.tolist()):
        if 0 <= p < cos_sin.shape[0]:
            c, s = cos_sin[p, :half].double(), cos_sin[p, half:].double()
            y[t, :, :half] = x[t, :, :half] * c - x[t, :, half:2 * half] * s
            y[t, :, half:2 * half] = x[t, :, half:2 * half] * c + x[t, :, :half] * s
    return y


def attention(q, cache, table, ctx_len, q_start, scale=None):
    """(out, sum_j p_j |v_j|) [T, hq, D] in float64 (the second is what roundings of the probabilities are relative to)."""
    q, table = q.double().cpu(), table.cpu()
    T, hq, D = q.shape
    pages, hkv, page, _ = cache.k.shape
    scale = 1 / math.sqrt(D) if scale is None else scale
    k, v = values(cache)
    out, size = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    ctx = ctx_len.tolist()
    start = list(range(len(ctx) + 1)) if q_start is None else q_start.tolist()
    for b, n in enumerate(ctx):
        keys = [(int(table[b, j // page]), j % page, j) for j in range(min(n, table.shape[1] * page))]
        keys = [(p, o, j) for p, o, j in keys if 0 <= p < pages]
        if not keys:
            continue
        at = torch.tensor(keys)
        kk, vv = k[at[:, 0], :, at[:, 1]], v[at[:, 0], :, at[:, 1]]
        vv = torch.where(torch.isfinite(vv).all(-1, keepdim=True), vv, float("nan"))
        for t in range(start[b], start[b + 1]):
            seen = at[:, 2] <= n - start[b + 1] + t
            if not seen.any():
                continue
            ks, vs = kk[seen].repeat_interleave(hq // hkv, 1), vv[seen].repeat_interleave(hq // hkv, 1)
            p = torch.softmax((ks * q[t]).sum(-1) * scale, 0)[..., None]
            out[t], size[t] = (p * vs).sum(0), (p * vs.abs()).sum(0)
    return out, size
