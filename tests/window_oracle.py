"""Attention of rows that see a sliding window and the first `sinks` keys, in float64 on the CPU. Test support.

Row j of a sequence (position p = seq_len - q_len + j) sees key k < seq_len (and k <= p where causal) if window <= 0,
p - k < window or k < sinks. Only keys that some row sees are read, through the block table; `freed` points every
page without such a key at a block of NaN.
"""
from __future__ import annotations

import math

import numpy as np
import torch

import workload as kvc


def seen_keys(seq_len, q_len, window, sinks):
    k = torch.arange(seq_len)
    return k if window <= 0 else k[(k < sinks) | (k >= max(0, seq_len - q_len - window + 1))]


def freed(case, window, sinks):
    """The case's block table with every page that holds no seen key at a block of NaN (which the cache gains); and how many."""
    c = case.cache
    block = int((~torch.isin(torch.arange(c.num_blocks), case.block_table.flatten())).nonzero()[0])
    kvc.poison_block(c, block)
    bt, n = case.block_table.clone(), 0
    for b, (seq, ql) in enumerate(zip(case.seqs, case.qlens)):
        pages = set((seen_keys(seq, max(ql, 1), window, sinks) // c.block_size).tolist()) if seq > 0 else set()
        for p in range(-(-max(seq, 0) // c.block_size)):
            if p not in pages:
                bt[b, p] = block
                n += 1
    return bt, n


def windowed(case, window, sinks, causal=True, block_table=None, qmax=None):
    """(out [T, Hq, 256], ln of the softmax sums [T, Hq], rows written [T]) in float64."""
    bt = case.block_table if block_table is None else block_table
    c, T, Hq = case.cache, case.num_tokens, case.num_q_heads
    hkv, bs = c.num_kv_heads, c.block_size
    g = Hq // hkv
    out, lse = torch.zeros((T, Hq, 256), dtype=torch.float64), torch.full((T, Hq), -math.inf, dtype=torch.float64)
    written = np.zeros(T, dtype=bool)
    q0 = 0
    for b, (seq, ql) in enumerate(zip(case.seqs, case.qlens)):
        rows = ql if qmax is None else min(ql, qmax)
        if rows > 0 and seq > 0:
            key = seen_keys(seq, ql, window, sinks)
            page, at = bt[b].long()[key // bs], key % bs
            k = c.key_cache[page, at, :, :256].double() * c.k_scale[page, at].double()[..., None]
            v = c.value_cache[page, at, :, :256].double() * c.v_scale[page, at].double()[..., None]
            pos = seq - ql + torch.arange(rows)
            see = torch.ones((rows, key.numel()), dtype=torch.bool)
            if causal:
                see &= key[None, :] <= pos[:, None]
            if window > 0:
                see &= (pos[:, None] - key[None, :] < window) | (key[None, :] < sinks)
            for h in range(hkv):
                x = torch.matmul(case.q[q0:q0 + rows, h * g:(h + 1) * g].double().reshape(rows * g, 256),
                                 k[:, h].t().contiguous()).view(rows, g, -1) * case.scale
                x = x.masked_fill(~see[:, None, :], -math.inf)
                ln = torch.logsumexp(x, -1)
                p = torch.where(ln[..., None] == -math.inf, 0.0, (x - ln[..., None]).exp())
                out[q0:q0 + rows, h * g:(h + 1) * g] = torch.matmul(p.view(rows * g, -1), v[:, h].contiguous()).view(rows, g, 256)
                lse[q0:q0 + rows, h * g:(h + 1) * g] = ln
            written[q0:q0 + rows] = True
        q0 += ql
    return out.numpy(), lse.numpy(), written
