"""Attention over a key/value cache in 8 or 4 bits in float64, a sequence at a time on the device of the queries: what :mod:`.quant_kv_plain` computes token by token, for more rows."""
import math

import torch

from . import quant_kv_plain as plain


def attention(q, cache, table, ctx_len, q_start=None, scale=None):
    """(out, sum_j p_j |v_j|) [T, hq, D] in float64."""
    dev, (T, hq, D) = q.device, q.shape
    pages, hkv, page, _ = cache.k.shape
    scale = 1 / math.sqrt(D) if scale is None else scale
    k, v = (x.to(dev) for x in plain.values(cache))
    v = torch.where(torch.isfinite(v).all(-1, keepdim=True), v, float("nan"))
    out, size = (torch.zeros(q.shape, dtype=torch.float64, device=dev) for _ in "ab")
    ctx, table = ctx_len.tolist(), table.cpu()
    start = list(range(len(ctx) + 1)) if q_start is None else q_start.tolist()
    for b, c in enumerate(ctx):
        n = start[b + 1] - start[b]
        at = torch.arange(max(0, min(c, table.shape[1] * page)))
        blk = table[b, at // page].long()
        there = (blk >= 0) & (blk < pages)
        at, blk = at[there], blk[there]
        if n == 0 or at.numel() == 0:
            continue
        kk, vv = (x[blk.to(dev), :, (at % page).to(dev)].transpose(0, 1).contiguous() for x in (k, v))      # [hkv, keys, D]
        seen = at.to(dev) <= torch.arange(c - n, c, device=dev)[:, None]                                     # [n, keys]
        rows = q[start[b]:start[b + 1]].double().view(n, hkv, -1, D).permute(1, 2, 0, 3)                     # [hkv, G, n, D]
        s = (rows.reshape(hkv, -1, D) @ kk.transpose(1, 2).contiguous()).view(hkv, -1, n, at.numel()) * scale
        bad = torch.isnan(vv).any(-1)                                                                        # [hkv, keys]
        s = torch.where(bad[:, None, None], float("nan"), s)
        p = torch.softmax(torch.where(seen, s, -math.inf), -1)
        p = torch.where(seen.any(-1, keepdim=True), p, 0.0).reshape(hkv, -1, at.numel())
        vv = torch.where(bad[..., None], 0.0, vv)
        for o, x in ((out, vv), (size, vv.abs())):
            o[start[b]:start[b + 1]] = (p @ x).view(hkv, -1, n, D).permute(2, 0, 1, 3).reshape(n, hq, D)
    return out, size
