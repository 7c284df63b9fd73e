"""decode_shared over drawn batches against float64 on the GPU: every input dimension at once, prefixes to 24,000 keys, batches of
few and of many rows (one and two row blocks of the prefix's waves), few and many segments. The bounds are those that
tests/test_shared_gpu.py derives: 2^-11 of sum p |v| for the rounding of P' (hi + lo is closer), 2 e for the scores, (n / 16 + 100) U for the
sums, half an fp16 step at the end.
"""
import random

import pytest
import torch

import workload as kvc
from mi50_vllm_lab_amd import pth_dec

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def draw(seed):
    r = random.Random(seed)
    hkv, g = r.choice([(1, 6), (2, 6), (4, 6), (1, 1), (2, 7), (1, 16), (1, 12), (8, 2)])
    qmax = r.randint(1, min(4, 48 // g))
    n = r.choice([1, 2, r.randint(3, 12), r.randint(13, 60), r.randint(60, 200)])
    long = 24000 if n <= 20 else 16000 if n <= 60 else 3000
    prefix = r.choice([r.randint(0, 40), r.randint(0, 1500), r.randint(1000, long), r.randint(1000, long)])
    most = r.choice([1, 60, 700, 5000 if n <= 12 else 700])
    own = [None if n > 1 and r.random() < 0.1 else r.randint(0, most) for _ in range(n)]
    qlens = [r.randint(1, qmax) for _ in range(n)]
    kw = dict(block_size=r.choice([8, 16, 16, 32, 48]), layout=r.choice(["HND", "NHD"]), outlier_frac=r.choice([0.0, 0.0, 0.02]))
    return dict(hkv=hkv, g=g, n=n, prefix=prefix, own=own, qlens=qlens, nseg=r.choice([4, 5, 16, 64, 100]), kw=kw)


@pytest.mark.parametrize("seed", range(32))
def test_drawn_batches(seed):
    x = draw(seed)
    hkv, g, prefix, own, qlens, kw = x["hkv"], x["g"], x["prefix"], x["own"], x["qlens"], x["kw"]
    print({k: v for k, v in x.items() if k not in ("own", "qlens")}, flush=True)
    bs, ctxs = kw["block_size"], [min(40, prefix) if o is None else prefix + o for o in own]
    case = kvc.make_case(ctxs, qlens, num_q_heads=hkv * g, num_kv_heads=hkv, seed=seed, **kw)
    c, holders = case.cache, [b for b, o in enumerate(own) if ctxs[b] >= prefix]
    for b in holders[1:]:
        case.block_table[b, :prefix // bs] = case.block_table[holders[0], :prefix // bs]
        if prefix % bs:
            src, dst = int(case.block_table[holders[0], prefix // bs]), int(case.block_table[b, prefix // bs])
            c.kv[dst, :, :prefix % bs] = c.kv[src, :, :prefix % bs]
    prefix = min(prefix, case.block_table.shape[1] * bs)
    d = case.to("cuda")
    c, T, hq = d.cache, d.num_tokens, hkv * g
    out = torch.full((T, hq, 256), float("nan"), dtype=torch.float16, device="cuda")
    lse = torch.empty((T, hq), device="cuda")
    pth_dec.decode_shared(d.q, c.key_cache, c.value_cache, c.k_scale, c.v_scale, d.block_table, d.seq_lens, d.query_start_loc, out, d.scale,
                          *kvc.partial_buffers(T, hq, x["nseg"], "cuda"), d.num_seqs, max(qlens), prefix, lse=lse)
    torch.cuda.synchronize()
    at = 0
    for b, ql in enumerate(qlens):
        n = ctxs[b] + ql
        pos = torch.arange(n, device="cuda")
        page, off = d.block_table[b].long()[pos // bs], pos % bs
        see = pos[None] <= (n - ql + torch.arange(ql, device="cuda").repeat_interleave(g))[:, None]
        for h in range(hkv):
            k, v = (t[page, off, h, :256].double() for t in (c.key_cache, c.value_cache))
            ks, vs = (t[page, off, h].double() for t in (c.k_scale, c.v_scale))
            q = d.q[at:at + ql, h * g:(h + 1) * g].double().reshape(-1, 256)
            s, a = (q @ k.T) * ks * d.scale, (q.abs() @ k.abs().T) * ks * d.scale
            m = s.masked_fill(~see, -float("inf")).amax(-1, keepdim=True)
            p = torch.exp(s - m).masked_fill(~see, 0)
            tot = p.sum(-1, keepdim=True)
            val = v * vs[:, None]
            e = U * (256 * a.masked_fill(~see, 0).amax(-1) + 8 * s.masked_fill(~see, 0).abs().amax(-1) + 8)[:, None]
            o, w = (p / tot) @ val, (p / tot) @ val.abs()
            sums = (n / 16 + 100) * U
            tol = (2.0 ** -11 + 2 * e + 2 * sums) * w + 2.0 ** -25 / 16 * v.abs().sum(0)[None] / tot
            mag = (o.abs() + tol).clamp(min=2.0 ** -14)
            tol = tol + torch.exp2(torch.floor(torch.log2(mag)) - 11)         # half an fp16 step
            got = out[at:at + ql, h * g:(h + 1) * g].double().reshape(-1, 256)
            bad = ~((got - o).abs() <= tol)
            assert not bool(bad.any()), (b, h, float(((got - o).abs() - tol).max()))
            want = (m + torch.log(tot))[:, 0]
            off_by = (lse[at:at + ql, h * g:(h + 1) * g].double().reshape(-1) - want).abs()
            assert bool((off_by <= e[:, 0] + sums + 8 * U * want.abs()).all()), (b, h, float(off_by.max()))
        at += ql
