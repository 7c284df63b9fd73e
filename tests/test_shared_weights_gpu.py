"""decode_shared keeps the weights' low bits (P' = p v_scale enters P.V as fp16 hi + lo, as decode's does) in every form of its
kernels, against float64: one and two row blocks of the prefix's waves, row counts at the edges of their tiles (128 and 256 rows),
own rows of one wave and of four, 16-key row blocks or not, short and long prefixes.

A query row has one nonzero value, so a score is one exact product and its scaling; a dozen keys of the prefix and some of
each sequence's own carry nearly all of a row. What is left of the error is then far below one fp16 rounding of P'. Each
case first shows on the float64 side that P' rounded once, of the shared keys or of the own ones, would not pass.

Bound. U = 2^-24. A score is scaled, offset by the running max and raised with it: 8 roundings of at most |s| < 28; 200 U for the
exponentials, the factors that join key groups and segments (each its own rounding and one of a difference of maxima) and the
constants: e = U (8 x 28 + 208) relative per weight. hi leaves at most 2^-11 of P' and lo at most 2^-11 of that: 2^-22, or half a
subnormal step of 2^-24 of 16 p v_scale, or all of a smaller one. The sums: at most 18 tiles hold a heavy key, 4 roundings each, 100 for the joins; a
tile without one adds no more error than it adds: S = 172 U + the light keys' share, in numerator and denominator. The output
is rounded to fp16 once.
"""
import numpy as np
import pytest
import torch

import workload as kvc
from mi50_vllm_lab_amd import pth_dec

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
SCALE = 0.0625


def build(n, ql, prefix, g, hkv, bs, layout, seed):
    """A batch on the GPU: `prefix` common keys, then 0 to 60 own ones and ql query tokens per sequence."""
    r = torch.Generator().manual_seed(seed)
    own = torch.randint(0, 61, (n,), generator=r) + ql
    whole = prefix // bs
    per = [-(-(prefix + int(o)) // bs) - whole for o in own]
    blocks = whole + sum(per)
    perm = torch.randperm(blocks, generator=r).to(torch.int32)
    bt = torch.zeros((n, whole + max(per)), dtype=torch.int32)
    bt[:, :whole], at = perm[:whole], whole
    for b, m in enumerate(per):
        bt[b, whole:whole + m] = perm[at:at + m]
        at += m
    c = kvc.allocate_cache(blocks, bs, hkv, layout, "cuda")
    d = torch.Generator(device="cuda").manual_seed(seed)
    shape = (blocks, bs, hkv)
    # the light keys; then the heavy ones
    c.key_cache[..., :256] = -torch.randint(120, 128, (*shape, 256), device="cuda", generator=d).to(torch.int8)
    c.value_cache[..., :256] = torch.randint(-127, 128, (*shape, 256), device="cuda", generator=d).to(torch.int8)
    c.k_scale.copy_(0.1 + 0.005 * torch.rand(shape, device="cuda", generator=d))
    c.v_scale.copy_(0.01 + 0.02 * torch.rand(shape, device="cuda", generator=d))

    def heavy(b, keys):
        pages = bt[b].long()[keys // bs]
        c.key_cache[pages, keys % bs, :, :256] = c.key_cache[pages, keys % bs, :, :256].neg()

    if prefix:
        heavy(0, torch.randperm(prefix, generator=r)[:12])
    if prefix % bs:
        for b in range(1, n):
            c.kv[int(bt[b, whole]), :, :prefix % bs] = c.kv[int(bt[0, whole]), :, :prefix % bs]
    for b in range(n):
        heavy(b, prefix + torch.randperm(int(own[b]), generator=r)[:6])
    T, hq = n * ql, g * hkv
    q = torch.zeros((T, hq, 256))
    at = torch.randint(0, 256, (T, hq, 1), generator=r)
    q.scatter_(2, at, torch.randint(24, 33, (T, hq, 1), generator=r).float())
    lens = (prefix + own).to(torch.int32)
    return c, bt.cuda(), lens, q.half().cuda(), torch.arange(0, T + 1, ql, dtype=torch.int32, device="cuda")


def half_step(x):
    return torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -14))) - 11)


def once(p, vs, x):
    """p v_scale rounded once to fp16, at the scale 2^x that a running max below the row's would give it."""
    return (p * vs * 2.0 ** x).half().double() * 2.0 ** -x / vs


@pytest.mark.parametrize("n,ql,prefix,g,hkv,bs,layout", [
    (4, 1, 100, 1, 2, 16, "HND"),         # few rows
    (3, 1, 0, 6, 1, 16, "HND"),           # nothing shared
    (5, 3, 300, 6, 1, 16, "NHD"),         # own rows on four waves
    (6, 8, 500, 6, 1, 16, "HND"),         # 48 of them
    (128, 1, 97, 1, 1, 16, "HND"),        # a full tile of one row block per wave
    (129, 1, 97, 1, 1, 16, "HND"),        # and a row more
    (256, 1, 97, 1, 1, 32, "NHD"),
    (257, 1, 97, 1, 1, 16, "HND"),
    (300, 1, 160, 1, 2, 16, "HND"),
    (43, 2, 640, 6, 1, 16, "HND"),        # 516 rows
    (65, 2, 400, 2, 1, 8, "NHD"),         # 260 rows without 16-key row blocks
    (128, 1, 12289, 1, 1, 16, "HND"),     # a long prefix
    (385, 1, 16384, 1, 1, 16, "HND"),     # the edge of the two forms
    (129, 1, 12289, 1, 1, 16, "HND"),
    (43, 1, 12289, 6, 1, 16, "NHD"),      # 258 rows
    (384, 1, 16385, 1, 1, 16, "HND"),
    (385, 1, 16385, 1, 1, 16, "HND"),     # two row blocks per wave
    (65, 1, 17000, 6, 2, 16, "NHD"),      # 390 rows
    (43, 2, 20000, 6, 1, 32, "HND"),      # 516 rows
])
def test_low_bits_of_the_weights(n, ql, prefix, g, hkv, bs, layout):
    print(f"shared weights: {n} x {ql} over {prefix}, {g * hkv} / {hkv} heads, blocks of {bs} {layout}", flush=True)
    c, bt, lens, q, qsl = build(n, ql, prefix, g, hkv, bs, layout, seed=n + prefix)
    T, hq = q.shape[:2]
    out = torch.full((T, hq, 256), float("nan"), dtype=torch.float16, device="cuda")
    lse = torch.empty((T, hq), device="cuda")
    pth_dec.decode_shared(q, c.key_cache, c.value_cache, c.k_scale, c.v_scale, bt, lens.cuda(), qsl, out, SCALE,
                          *kvc.partial_buffers(T, hq, 64, "cuda"), n, ql, prefix, lse=lse)
    torch.cuda.synchronize()
    worst = 0.0
    caught = [0, 0]                                  # elements that P' rounded once, of shared keys or of own ones, puts out of bounds
    for b in range(n):
        length = int(lens[b])
        pos = torch.arange(length, device="cuda")
        page, off = bt[b].long()[pos // bs], pos % bs
        see = pos[None] <= (length - ql + torch.arange(ql, device="cuda").repeat_interleave(g))[:, None]
        rows = slice(b * ql, (b + 1) * ql)
        for h in range(hkv):
            k, v = (t[page, off, h, :256].double() for t in (c.key_cache, c.value_cache))
            ks, vs = (t[page, off, h].double() for t in (c.k_scale, c.v_scale))
            x = q[rows, h * g:(h + 1) * g].double().reshape(-1, 256)
            s = ((x @ k.T) * ks * SCALE).masked_fill(~see, -float("inf"))
            m = s.amax(-1, keepdim=True)
            p = torch.exp(s - m)
            tot = p.sum(-1, keepdim=True)
            val = v * vs[:, None]
            o, w = (p / tot) @ val, (p / tot) @ val.abs()
            light = (p / tot).masked_fill(k[None, :, 0] > 0, 0).sum(-1).max()
            e, sums = U * (8 * 28 + 208), 172 * U + float(light)           # |s| <= 32 x 127 x 0.105 / 16 < 28
            tol = (2.0 ** -22 + 2 * e + 2 * sums) * w + ((p * vs).clamp(max=2.0 ** -29) / tot) @ v.abs()
            tol = tol + half_step(o.abs() + tol)
            got = out[rows, h * g:(h + 1) * g].double().reshape(-1, 256)
            err = (got - o).abs()
            assert bool((err <= tol).all()), (b, h, float((err - tol).max()))
            worst = max(worst, float((err / tol).max()))
            want = (m + torch.log(tot))[:, 0]
            off_by = (lse[rows, h * g:(h + 1) * g].double().reshape(-1) - want).abs()
            assert bool((off_by <= e + sums + 8 * U * want.abs()).all()), (b, h, float(off_by.max()))
            for i, part in enumerate((pos < prefix, pos >= prefix)):
                hi = torch.where(part[None], once(p, vs, 4 + (b % 7) / 2), p)
                caught[i] += int(((((hi / tot) @ val).half().double() - o).abs() > tol).sum())
    print(f"worst {worst:.2f} of the bound; rounded once: {caught}", flush=True)
    assert caught[1] > 0 and (prefix == 0 or caught[0] > 0)
