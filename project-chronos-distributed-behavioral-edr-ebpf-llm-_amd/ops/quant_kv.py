"""A paged key/value cache in 8 or 4 bits: heads normed, rotated and written in one pass, read back, and attended to, also by groups of sequences
that share their first pages.

Beside the bf16 / e4m3 pages of ``rope_kv_write`` and ``paged_attention``, whose e4m3 form has one scale per layer, :class:`QuantKV` holds a scale for what it scales:

* ``int8``: codes -127 .. 127 and a float32 scale per token and head (max / 127): half the bytes of bf16, errors of 1/254 of a row's largest number;
* ``mxfp4``: e2m1 codes and a power of two per 32 dimensions: a quarter of the bytes (17 for 64), errors of some 11 % of a number's size.

Heads have 64 or 128 dimensions, pages a multiple of 16 tokens, query heads are any multiple of the cache's.  Every function takes GPU tensors (the HIP kernels of
csrc/kernels/quant_kv.hip and quant_attention.hip; current stream, captured into graphs as other launches are) or CPU tensors (:mod:`.quant_kv_ref`).

What is not there is left out: a token whose position is negative or (as it is written) behind the rope table, or whose page the table or the cache does not have, is not
written and reads as zeros (so padded batches need no page of their own); keys on pages outside the cache (say -1) are not seen; a query row that sees no key is zeros.  A head row with an infinity or NaN is
held as NaN as a whole, and makes NaN of the rows that see it, of no others.
"""
from __future__ import annotations

import math
import sys
from dataclasses import dataclass

import torch

from . import quant_kv_ref as ref

_pkg = sys.modules[__package__]
_ops: dict = {}


def _k(name: str):
    """The kernel library's operator: looked up once, a call costs half as much without it."""
    op = _ops.get(name)
    if op is None:
        op = _ops[name] = getattr(_pkg._k(), name).default
    return op


@dataclass(frozen=True)
class QuantKV:
    """One layer's cache.  k, v: [pages, heads, page, D] int8 or [pages, heads, page, D / 2] uint8; ks, vs: [pages, heads, page] float32 or
    [pages, heads, page, D / 32] uint8 (csrc/include/chronos_quant_kv.h)."""
    k: torch.Tensor
    v: torch.Tensor
    ks: torch.Tensor
    vs: torch.Tensor

    @property
    def kind(self) -> str:
        return "int8" if self.k.dtype == torch.int8 else "mxfp4"

    @property
    def heads(self) -> int:
        return self.k.shape[1]

    @property
    def head_dim(self) -> int:
        return self.k.shape[3] * (1 if self.k.dtype == torch.int8 else 2)

    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in (self.k, self.v, self.ks, self.vs))


def quant_kv_cache(num_blocks: int, block_size: int, hkv: int, head_dim: int = 128, kind: str = "int8", device=None) -> QuantKV:
    """An empty cache (zeros)."""
    _need(kind in ("int8", "mxfp4"), f"kind must be 'int8' or 'mxfp4', not {kind!r}")
    rows = (num_blocks, hkv, block_size)
    if kind == "int8":
        cache = QuantKV(*(torch.zeros(*rows, head_dim, dtype=torch.int8, device=device) for _ in "kv"), *(torch.zeros(rows, device=device) for _ in "kv"))
    else:
        cache = QuantKV(*(torch.zeros(*rows, n, dtype=torch.uint8, device=device) for n in (head_dim // 2, head_dim // 2, head_dim // 32, head_dim // 32)))
    _check_cache(cache)
    return cache


def _need(cond: bool, what: str) -> None:
    if not cond:
        raise RuntimeError(f"chronos: {what}")


def _check_cache(c: QuantKV) -> None:
    int8 = c.k.dtype == torch.int8
    _need(int8 or c.k.dtype == torch.uint8, "k must be int8 codes or uint8 pairs of e2m1 codes")
    _need(c.k.dim() == 4 and c.v.shape == c.k.shape and c.v.dtype == c.k.dtype, "k and v must be [pages, heads, page, row] of one type")
    _need(c.head_dim in (64, 128), f"heads of 64 or 128 dimensions, not {c.head_dim}")
    _need(c.k.shape[2] > 0 and c.k.shape[2] % 16 == 0, f"pages of a multiple of 16 tokens, not {c.k.shape[2]}")
    _need(c.k.shape[0] > 0 and c.k.shape[1] > 0, "the cache has no pages or heads, or too many")
    want = tuple(c.k.shape[:3]) if int8 else (*c.k.shape[:3], c.head_dim // 32)
    for s in (c.ks, c.vs):
        _need(s.dtype == (torch.float32 if int8 else torch.uint8), "scales must be float32 (int8 codes) or uint8 (e2m1 codes)")
        _need(tuple(s.shape) == want, "scales must be [pages, heads, page] (int8 codes) or [pages, heads, page, D / 32] (e2m1 codes)")
    for t in (c.k, c.v, c.ks, c.vs):
        _need(t.device == c.k.device, f"k, v, ks and vs must be on {c.k.device}")
        _need(t.is_contiguous(), "k, v, ks and vs must be contiguous, from a multiple of 16 bytes")


def _check_ints(t, like, least: int, what: str) -> None:
    _need(t.device == like.device, f"{what} must be on {like.device}")
    _need(t.dtype == torch.int32 and t.dim() == 1 and t.is_contiguous(), f"{what} must be a contiguous int32 vector")
    _need(t.numel() >= least, f"{what} needs {least} entries, has {t.numel()}")


def _check_table(t, like) -> None:
    _need(t.device == like.device, f"block_table must be on {like.device}")
    _need(t.dtype == torch.int32 and t.dim() == 2, "block_table must be int32 [sequences, pages] with neighbouring pages side by side")


def _check_tokens(pos, tok_seq, n: int, like) -> None:
    _need(pos.dim() == 1 and pos.numel() == n and tok_seq.dim() == 1 and tok_seq.numel() == n, "pos and tok_seq need an entry per token")
    _check_ints(pos, like, n, "pos")
    _check_ints(tok_seq, like, n, "tok_seq")


def norm_rope_kv_quant(qkv: torch.Tensor, pos: torch.Tensor, tok_seq: torch.Tensor, block_table: torch.Tensor, cos_sin: torch.Tensor, cache: QuantKV, hq: int,
                       q_norm: torch.Tensor | None = None, k_norm: torch.Tensor | None = None, eps: float = 1e-6) -> torch.Tensor:
    """A projection's rows qkv [T, (hq + 2 hkv) D] (bfloat16) into queries and cache, in one pass: the RMS norm of every query and key head (weights [D]; None: no
    norm), the rotation of their first R dimensions (cos_sin [positions, R] float32, cosines then sines; R a multiple of 16 up to D), keys and values quantised into
    row ``pos % page`` of page ``block_table[tok_seq, pos // page]``.  Returns the queries [T, hq, D].  Two tokens of one call must not have the same place.  The
    queries of a token without a place are zeros."""
    if _pkg._checking(qkv):
        ok, blk, row = ref.places(cache, block_table.cpu(), pos.cpu(), tok_seq.cpu(), cos_sin.shape[0])      # tokens without a place are left out
        n = (blk * cache.k.shape[2] + row)[ok]
        _pkg._need(torch.unique(n).numel() == n.numel(), "norm_rope_kv_quant: two tokens in one place")
    if qkv.is_cuda:
        return _k("norm_rope_kv_quant")(qkv, pos, tok_seq, block_table, cos_sin, cache.k, cache.v, cache.ks, cache.vs, hq, q_norm, k_norm, eps)
    _check_cache(cache)
    D, R = cache.head_dim, cos_sin.shape[1] if cos_sin.dim() == 2 else -1
    _need(qkv.device == cache.k.device, f"qkv must be on {cache.k.device}")
    _need(qkv.dtype == torch.bfloat16 and qkv.dim() == 2, "qkv must be bfloat16 [T, (hq + 2 hkv) D]")
    _need(hq >= 0 and qkv.shape[1] == (hq + 2 * cache.heads) * D, f"qkv must be [T, (hq + 2 hkv) D] = [T, {(hq + 2 * cache.heads) * D}], has rows of {qkv.shape[1]}")
    _check_tokens(pos, tok_seq, qkv.shape[0], cache.k)
    _check_table(block_table, cache.k)
    _need(cos_sin.dtype == torch.float32 and R >= 16 and R % 16 == 0 and R <= D, "cos_sin must be float32 [positions, R], R a multiple of 16 up to D")
    _need(cos_sin.shape[0] > 0 or qkv.shape[0] == 0, "cos_sin has no positions")
    _need(eps >= 0, "eps must not be negative")
    for w, what in ((q_norm, "q_norm"), (k_norm, "k_norm")):
        _need(w is None or (w.dtype == torch.bfloat16 and w.dim() == 1 and w.numel() == D), f"{what} must be bfloat16 [D]")
    return ref.norm_rope_kv_quant(qkv, pos, tok_seq, block_table, cos_sin, cache, hq, q_norm, k_norm, eps)


def quant_kv_read(cache: QuantKV, block_table: torch.Tensor, pos: torch.Tensor, tok_seq: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Keys and values [T, hkv, D] in bfloat16 of the tokens (tok_seq, pos), addressed as :func:`norm_rope_kv_quant` writes them."""
    if cache.k.is_cuda:
        return _k("quant_kv_read")(cache.k, cache.v, cache.ks, cache.vs, block_table, pos, tok_seq)
    _check_cache(cache)
    _check_tokens(pos, tok_seq, pos.numel(), cache.k)
    _check_table(block_table, cache.k)
    return ref.quant_kv_read(cache, block_table, pos, tok_seq)


def quant_attention(q: torch.Tensor, cache: QuantKV, block_table: torch.Tensor, ctx_len: torch.Tensor, q_start: torch.Tensor | None = None,
                    scale: float | None = None, max_ctx: int | None = None) -> torch.Tensor:
    """Causal attention of q [T, hq, D] over the cache: sequence b has the tokens q_start[b] .. q_start[b + 1] - 1 (q_start[0] = 0; None: token b alone), the last of
    them at position ctx_len[b] - 1, its keys on the pages block_table[b].  One token or whole prompts.  Rows behind the last sequence are zeros.  ``scale``: 1 / sqrt(D) by default.
    ``max_ctx``: a length that no context passes, if the table is much wider than the contexts; it goes into how the work is cut up, and into nothing else (without it a row of 140 keys in a
    table of 131072 gets 64 pieces and a second launch, 11 us in place of 6.5)."""
    return _attention(q, cache, block_table, ctx_len, q_start, None, None, scale, max_ctx)


def prefix_attention(q: torch.Tensor, cache: QuantKV, block_table: torch.Tensor, ctx_len: torch.Tensor, group_start: torch.Tensor, prefix_len: torch.Tensor,
                     q_start: torch.Tensor | None = None, scale: float | None = None, max_ctx: int | None = None) -> torch.Tensor:
    """:func:`quant_attention` where groups of neighbouring sequences share their first pages: sequences group_start[g] .. group_start[g + 1] - 1 have the same pages
    in the first prefix_len[g] tokens (rounded down to whole pages) of their tables.  Those are read once for the whole group, every sequence's own keys behind them by
    itself.  Sequences outside all groups are attended to as well.  The result is that of :func:`quant_attention`, but for the order of its sums.

    This is for decode rows on a long common prefix, with some hundreds of keys of their own: 64 rows on 4096 shared keys 29 us where :func:`quant_attention` takes 67, 16 on 4096 19 and 27, 8 on
    4096 18 and 19, 64 on 1024 21 and 21, 9 x 3 on 480 15 and 10 (int8, 32 query and 8 key heads).  Two launches that wait for each other take 12 us, so below some 16 rows or 2048 shared keys
    :func:`quant_attention` is the faster one.  So it is where own keys are long: in tables of up to 32768 keys they are walked in one piece (two sequences of 18000 own keys behind 2048: 175 us,
    :func:`quant_attention` 22), those of sequences outside the groups too.  The work on the groups is cut up by all rows of the call: prompts are better given to a call of their own."""
    return _attention(q, cache, block_table, ctx_len, q_start, group_start, prefix_len, scale, max_ctx)


def _attention(q, cache, block_table, ctx_len, q_start, group_start, prefix_len, scale, max_ctx):
    if scale is None:
        scale = 1.0 / math.sqrt(q.shape[-1])
    if max_ctx is None:
        max_ctx = -1
    if _pkg._checking(q):
        B = ctx_len.numel()
        _pkg._need(bool((ctx_len.cpu() <= block_table.shape[1] * cache.k.shape[2]).all()), "quant_attention: length exceeds block table")
        if q_start is not None:
            qs = q_start.cpu().long()[:B + 1]
            _pkg._need(bool((qs.diff() >= 0).all()) and int(qs[0]) == 0 and int(qs[-1]) <= q.shape[0], "quant_attention: q_start")
        if group_start is not None:
            gs, bt = group_start.cpu().long()[:prefix_len.numel() + 1], block_table.cpu()
            _pkg._need(bool((gs.diff() >= 0).all()) and int(gs[0]) >= 0 and int(gs[-1]) <= B, "prefix_attention: group_start")
            for g, n in enumerate(prefix_len.tolist()):
                rows = bt[int(gs[g]):int(gs[g + 1]), :max(n, 0) // cache.k.shape[2]]
                _pkg._need(bool((rows == rows[:1]).all()), f"prefix_attention: the pages of group {g} differ")
    if q.is_cuda:
        return _k("quant_attention")(q, cache.k, cache.v, cache.ks, cache.vs, block_table, ctx_len, q_start, group_start, prefix_len, scale, max_ctx)
    _check_cache(cache)
    T, hq, B = q.shape[0], q.shape[1] if q.dim() == 3 else 0, ctx_len.numel()
    _need(q.device == cache.k.device, f"q must be on {cache.k.device}")
    _need(q.dtype == torch.bfloat16 and q.dim() == 3 and q.shape[2] == cache.head_dim, f"q must be bfloat16 [T, hq, {cache.head_dim}]")
    _need(hq > 0 and hq % cache.heads == 0, f"q heads ({hq}) must be a multiple of the cache's ({cache.heads})")
    _check_table(block_table, cache.k)
    _check_ints(ctx_len, cache.k, 0, "ctx_len")
    _need(block_table.shape[0] >= B, "block_table needs a row per sequence")
    if q_start is not None:
        _check_ints(q_start, cache.k, B + 1, "q_start")
    else:
        _need(T >= B, f"without q_start every sequence has a token: q needs {B} rows, has {T}")
    _need((group_start is None) == (prefix_len is None), "group_start and prefix_len go together")
    if group_start is not None:
        _check_ints(prefix_len, cache.k, 0, "prefix_len")
        _check_ints(group_start, cache.k, prefix_len.numel() + 1, "group_start")
    return ref.quant_attention(q, cache, block_table, ctx_len, q_start, scale)
