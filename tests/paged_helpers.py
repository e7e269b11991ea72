"""Inputs, 64-bit definitions and error bounds of the paged KV cache operators' tests.

The bounds count roundings: a value rounded to a type with epsilon e is off by at most e / 2 of itself.  U = 2^-24 is
that of F32."""
from __future__ import annotations

import ctypes as C
import math

import torch

U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def type_id(G, dtype):
    return {torch.float32: G.F32, torch.float16: G.F16, torch.bfloat16: G.BF16}[dtype]


def ptr(t):
    return None if t is None else t.data_ptr()


def ints(v, dtype=torch.int32):
    return torch.tensor(v, dtype=dtype, device="cuda")


def stream():
    return torch.cuda.current_stream().cuda_stream


class Cache:
    """K and V of one layer, every element NaN until it is written.  layout: 'head' contiguous
    [block][head][token][dim], 'token' [block][token][head][dim], 'both' K and V interleaved in one
    [block][2][head][token][dim] allocation."""

    def __init__(self, G, blocks, kv_heads, bs, dim, dtype, layout="head"):
        self.bs, self.blocks = bs, blocks
        full = lambda *shape: torch.full(shape, math.nan, dtype=dtype, device="cuda")  # noqa: E731
        if layout == "token":
            self.k, self.v = (full(blocks, bs, kv_heads, dim).permute(0, 2, 1, 3) for _ in range(2))
        elif layout == "both":
            both = full(blocks, 2, kv_heads, bs, dim)
            self.k, self.v = both[:, 0], both[:, 1]
        else:
            self.k, self.v = full(blocks, kv_heads, bs, dim), full(blocks, kv_heads, bs, dim)
        st = [2 * s for s in self.k.stride()]
        strides = {} if layout == "head" else dict(nb_block=st[0], nb_head=st[1], nb_token=st[2])
        self.rec = G.KvCache(type=type_id(G, dtype), head_dim=dim, kv_heads=kv_heads, block_size=bs, num_blocks=blocks,
                             k=ptr(self.k), v=ptr(self.v), **strides)

    def put(self, blocks, k, v):
        """Keys and values [tokens, heads, dim] of one request into its blocks."""
        at = torch.arange(k.shape[0], device="cuda")
        b = ints(blocks, torch.int64)[at // self.bs]
        self.k[b, :, at % self.bs], self.v[b, :, at % self.bs] = k.to(self.k.dtype), v.to(self.v.dtype)

    def get(self, blocks, n):
        at = torch.arange(n, device="cuda")
        b = ints(blocks, torch.int64)[at // self.bs]
        return self.k[b, :, at % self.bs], self.v[b, :, at % self.bs]


def slopes(heads, max_bias):
    near = 1 << (heads.bit_length() - 1)
    return [2.0 ** (-max_bias * (h + 1) / near) if h < near else 2.0 ** (-max_bias / 2 * (2 * (h - near) + 1) / near)
            for h in range(heads)]


def attention_ref(q, k, v, pos0, scale, cap=0.0, max_bias=0.0, window=0, weight_half=0.0):
    """64-bit attention of q [n, H, D] at positions pos0 .. over k, v [kv, KH, D], and a bound on the kernel's error.

    The bound: a score's D products add up in D / 16 matrix instructions, each off by at most 2 U of the sum of their
    absolute values so far, and F32 queries are split into pieces that carry 22 bits or more: (D / 16 + 4) 2 U S with S
    the scaled sum of absolute products.  The cap (tanh within 4 U, times c), the bias and the exponential add a few U
    of the score itself.  Relative to exp, an error d of a score is a weight off by d; the weighted sum over n keys
    adds n / 16 + 8 roundings, and a weight's own rounding to the cache's type weight_half."""
    n, H, D = q.shape
    kv, KH, _ = k.shape
    q, k, v = q.double(), k.double(), v.double()
    k, v = k.repeat_interleave(H // KH, 1), v.repeat_interleave(H // KH, 1)
    s = torch.einsum("nhd,khd->hnk", q, k) * scale
    size = torch.einsum("nhd,khd->hnk", q.abs(), k.abs()) * abs(scale)
    off = (D / 16 + 4) * 2 * U * size + 4 * U * s.abs()
    if cap:
        s = cap * torch.tanh(s / cap)
        off = off + 6 * U * cap
    p = torch.arange(n, device=q.device)[:, None] + pos0
    j = torch.arange(kv, device=q.device)[None, :]
    if max_bias:
        s = s + torch.tensor(slopes(H, max_bias), dtype=torch.float64, device=q.device)[:, None, None] * (j - p).double()
        off = off + 8 * U * s.abs()
    seen = j <= p
    if window:
        seen = seen & (j > p - window)
    s = s.masked_fill(~seen, -math.inf)
    w = torch.softmax(s, -1)
    w = torch.where(seen.any(-1)[None, :, None], w, torch.zeros_like(w))
    off = torch.where(w > 0, off + 4 * U, torch.zeros_like(off))
    out = torch.einsum("hnk,khd->nhd", w, v)
    mean = (w * off).sum(-1)  # what the normaliser is off by
    bound = torch.einsum("hnk,khd->nhd", w * (off + mean[..., None] + weight_half + (kv / 16 + 8) * 2 * U), v.abs())
    return out, bound


def run_attention(G, q, out, cache, cu, kv, table, scale, cap=0.0, max_bias=0.0, window=0, max_new=None, max_kv=None,
                  nb_q=0, nb_out=0, workspace=None, call=True):
    """One b200_paged_attention call on tensors; returns what has to stay alive for a replay."""
    heads = q.shape[1]
    n = [b - a for a, b in zip(cu.tolist()[:-1], cu.tolist()[1:])]
    p = G.PagedAttention(n_tokens=q.shape[0], n_seqs=kv.numel(), heads=heads, q_type=type_id(G, q.dtype),
                         out_type=type_id(G, out.dtype), q=ptr(q), out=ptr(out), nb_q=nb_q, nb_out=nb_out,
                         cu_new=ptr(cu), kv_lens=ptr(kv), block_table=ptr(table), table_width=table.shape[1],
                         max_new=max(n + [0]) if max_new is None else max_new,
                         max_kv=max(kv.tolist() + [0]) if max_kv is None else max_kv, scale=scale, logit_softcap=cap,
                         max_bias=max_bias, window=window)
    need = G.lib().b200_paged_attention_workspace(C.byref(p), C.byref(cache.rec))
    ws = workspace if workspace is not None else torch.full((need + 16,), 255, dtype=torch.uint8, device="cuda")
    p.workspace, p.workspace_bytes = ptr(ws), ws.numel()
    if call:
        G.check(G.lib().b200_paged_attention(C.byref(p), C.byref(cache.rec), stream()), "paged_attention")
    return p, ws


def spread_tables(lens, bs, spare=3, seed=0):
    """Shuffled blocks for requests of the given key counts: (per-request block lists, table with garbage behind
    each row, number of blocks)."""
    gen = torch.Generator().manual_seed(seed)
    pages = [-(-n // bs) for n in lens]
    total = sum(pages) + spare
    perm = torch.randperm(total, generator=gen).tolist()
    lists, at = [], 0
    for n in pages:
        lists.append(perm[at: at + n])
        at += n
    width = max(pages + [1])
    table = [row + [0x7FFFFFF0 - i if i % 2 else -5 - i for i in range(width - len(row))] for row in lists]
    return lists, ints(table), total
