"""norm_rotary_cache_write on the GPU: queries against a float64 norm and rotation within the roundings of the formula, cache bytes
equal to the cache writer's for the key normed and rotated in fp32, the result the same bits for every layout of the rotated dims; the
three input types, weights of the input's type and fp32, in place and into another tensor, heads of zeros, of infinities and of NaN,
skipped tokens, 0 and 1 tokens; another stream and a captured graph.
"""
import numpy as np
import pytest
import torch

import workload as kvc
from mi50_vllm_lab_amd import pth_dec, rotary

pytestmark = pytest.mark.gpu
DT = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
TABLE = 600
EPS = 1e-5


def normed64(x, w, eps=EPS, offset=0.0):
    x, w = x.double().numpy(), w.double().numpy() + offset
    return x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w


def rotated64(y, table, pos, interleaved):
    """(rotated, |x c| + |y s| of each rotated value) of y [T, H, 256]."""
    cs = table.double().numpy()[pos.numpy()]
    rd = cs.shape[1]
    c, s = cs[:, None, :rd // 2], cs[:, None, rd // 2:]
    fi, se = (slice(0, rd, 2), slice(1, rd, 2)) if interleaved else (slice(0, rd // 2), slice(rd // 2, rd))
    out, size = y.copy(), np.abs(y)
    a, b = y[..., fi], y[..., se]
    out[..., fi], out[..., se] = a * c - b * s, b * c + a * s
    size[..., fi], size[..., se] = np.abs(a * c) + np.abs(b * s), np.abs(b * c) + np.abs(a * s)
    return out, size


def make(T, hq, hkv, dtype, rd, seed, weight="same"):
    g = torch.Generator().manual_seed(seed)
    qkv = torch.randn((T, hq + 2 * hkv, 256), generator=g)
    if T > 3:
        qkv[1] = 0.0           # an all-zero token: normed to 0, scale 0
        qkv[2] *= 40
        qkv[3] *= 1e-4         # mean square below eps
    pos = torch.randint(0, TABLE, (T,), generator=g)
    if T > 0:
        pos[0], pos[-1] = 0, TABLE - 1
    wt = torch.float32 if weight == "fp32" else DT[dtype]
    w = [(torch.rand(256, generator=g) + 0.5).to(wt) for _ in range(2)]
    return qkv.to(DT[dtype]), pos, rotary.rotary_table(rd, TABLE, 1e4), w


@pytest.mark.parametrize("T,hq,hkv,dtype,rd,interleaved,out,bs,layout,weight,offset", [
    (1, 24, 4, "fp16", 256, False, "inplace", 16, "HND", "same", 0.0),
    (1, 1, 1, "fp32", 8, True, "inplace", 1, "NHD", "same", 1.0),
    (5, 24, 4, "bf16", 64, False, "fp16", 16, "NHD", "same", 1.0),
    (7, 12, 2, "fp16", 128, True, "same", 1584, "HND", "fp32", 0.0),
    (33, 6, 6, "fp32", 96, False, "fp16", 32, "HND", "same", 0.0),
    (130, 5, 1, "bf16", 200, True, "same", 16, "HND", "fp32", -0.25),
    (64, 24, 4, "fp32", 256, True, "inplace", 16, "NHD", "fp32", 0.0),
    (301, 24, 4, "bf16", 56, False, "inplace", 16, "HND", "same", 0.0),
    (513, 24, 4, "fp16", 8, False, "inplace", 48, "HND", "fp32", 1.0),
    (700, 7, 1, "fp32", 200, False, "same", 1584, "NHD", "same", 0.0),
    (1100, 24, 4, "bf16", 120, False, "fp16", 16, "HND", "same", 0.0),
])
def test_against_float64(T, hq, hkv, dtype, rd, interleaved, out, bs, layout, weight, offset):
    qkv, pos, table, (wq, wk) = make(T, hq, hkv, dtype, rd, T + rd, weight)
    d = qkv.cuda()
    q, k, v = d[:, :hq], d[:, hq:hq + hkv], d[:, hq + hkv:]
    blocks = -(-T // bs) + 2
    slots = torch.randperm(blocks * bs, generator=torch.Generator().manual_seed(5))[:T]
    c = kvc.allocate_cache(blocks, bs, hkv, layout, "cuda")
    c.kv.fill_(77)
    qout = q if out == "inplace" else torch.full((T, hq + 1, 256), 7.0, dtype=DT[dtype] if out == "same" else torch.float16,
                                                 device="cuda")[:, :hq]
    pth_dec.norm_rotary_cache_write(q, k, v, wq.cuda(), wk.cuda(), pos.cuda(), table.cuda(), c.key_cache, c.value_cache, c.k_scale,
                                    c.v_scale, slots.cuda(), eps=EPS, weight_offset=offset, interleaved=interleaved,
                                    query_out=None if out == "inplace" else qout)
    torch.cuda.synchronize()
    # Roundings in fp32, u = 2^-24 each: a square, the three sums of four, six of the tree, * 2^-8 exact, + eps: at most 11 of the
    # (positive) sum, halved by the root; the root itself 1 u and its products with x and w 2 u, the weight's offset 1 u of
    # (|w| + |offset|): 5.5 + 1 + 2 <= 9 u relative; then three of the rotation, of its size; then the output's, eps / 2.
    u = 2.0 ** -24
    w64 = wq.double().numpy() + offset
    wrel = u * (np.abs(wq.double().numpy()) + abs(offset)) / np.maximum(np.abs(w64), 1e-30) if offset else 0.0
    y = normed64(qkv[:, :hq], wq, offset=offset)
    ref, size = rotated64(y, table, pos, interleaved)
    # (a value's own weight rounding reaches both of its pair: bound it by the largest)
    rel = 9 * u + (np.max(wrel) if offset else 0.0)
    fp32 = (rel + 3 * u) * size * (1 + 1e-5)
    t = torch.finfo(qout.dtype)
    bound = fp32 + t.eps / 2 * (np.abs(ref) + fp32) + t.tiny * t.eps / 2
    err = np.abs(qout.double().cpu().numpy() - ref)
    assert (err <= bound).all(), float((err - bound).max())
    assert torch.equal(d[:, hq:].cpu(), qkv[:, hq:])               # key and value stay
    if out != "inplace":
        assert torch.equal(d.cpu(), qkv)
        assert bool((qout.as_strided((T, 1, 256), ((hq + 1) * 256, 256, 1), qout.storage_offset() + hq * 256) == 7.0).all())
    # the cache: int8 within half a step and the bound's own, the scale the largest magnitude / 127
    key, size = rotated64(normed64(qkv[:, hq:hq + hkv], wk, offset=offset), table, pos, interleaved)
    wrel = u * (np.abs(wk.double().numpy()) + abs(offset)) / np.maximum(np.abs(wk.double().numpy() + offset), 1e-30) if offset else 0.0
    tol = (9 * u + (np.max(wrel) if offset else 0.0) + 3 * u) * size * (1 + 1e-5)
    blk, at = slots // bs, slots % bs
    scale = c.k_scale.cpu()[blk, at].double().numpy()
    got = c.key_cache.cpu()[blk, at, :, :256].double().numpy()
    most = np.abs(key).max(-1)
    assert (np.abs(scale - most / 127) <= tol.max(-1) / 127 + 2 * u * most / 127).all()
    # (a division's rounding, at most 2^-24 of 127 steps, on top of the half step)
    step = scale[..., None]
    assert (np.abs(got * step - key) <= tol + step * (0.5 + 2.0 ** -16) + 1e-30).all()
    # the values: the cache writer's bytes
    other = kvc.allocate_cache(blocks, bs, hkv, layout, "cuda")
    other.kv.fill_(77)
    pth_dec.cache_write(v, v, other.key_cache, other.value_cache, other.k_scale, other.v_scale, slots.cuda())
    assert torch.equal(other.value_cache, c.value_cache)


@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
def test_the_norm_does_not_depend_on_the_rotated_dims(dtype):
    """With angles of 0 the rotation leaves every value as it is: all layouts give the same bits, and the same cache rows."""
    T, hq, hkv = 70, 24, 4
    qkv, _, _, (wq, wk) = make(T, hq, hkv, dtype, 8, 3)
    d = qkv.cuda()
    seen = []
    for rd in (8, 24, 64, 200, 256):
        for interleaved in (False, True):
            table = torch.cat([torch.ones((4, rd // 2)), torch.zeros((4, rd // 2))], -1).cuda()
            c = kvc.allocate_cache(6, 16, hkv, "HND", "cuda")
            out = torch.empty((T, hq, 256), dtype=torch.float16 if dtype == "fp16" else DT[dtype], device="cuda")
            pth_dec.norm_rotary_cache_write(d[:, :hq], d[:, hq:hq + hkv], d[:, hq + hkv:], wq.cuda(), wk.cuda(),
                                            torch.zeros(T, dtype=torch.int64, device="cuda"), table, c.key_cache, c.value_cache,
                                            c.k_scale, c.v_scale, torch.arange(T, device="cuda"), interleaved=interleaved, query_out=out)
            seen.append((out, c.kv))
    for out, kv in seen[1:]:
        assert torch.equal(out, seen[0][0]) and torch.equal(kv, seen[0][1])


def test_heads_that_are_not_finite_stay_their_own():
    """A head with an infinity or a NaN becomes what the formula gives (NaN and 0); the heads and tokens beside it do not change."""
    T, hq, hkv, rd = 9, 8, 2, 64
    qkv, pos, table, (wq, wk) = make(T, hq, hkv, "fp32", rd, 4)
    outs = []
    for spoil in (False, True):
        x = qkv.clone()
        if spoil:
            x[4, 3, 17], x[5, 6, 200], x[6, 8, 100] = float("inf"), float("nan"), float("nan")
        d = x.cuda()
        c = kvc.allocate_cache(1, 16, hkv, "HND", "cuda")
        out = torch.empty((T, hq, 256), device="cuda")
        pth_dec.norm_rotary_cache_write(d[:, :hq], d[:, hq:hq + hkv], d[:, hq + hkv:], wq.cuda(), wk.cuda(), pos.cuda(), table.cuda(),
                                        c.key_cache, c.value_cache, c.k_scale, c.v_scale, torch.arange(T, device="cuda"), query_out=out)
        outs.append((out.cpu(), c.kv.cpu()))
    same = torch.ones((T, hq), dtype=torch.bool)
    same[4, 3] = same[5, 6] = False
    assert torch.equal(outs[0][0][same], outs[1][0][same])
    assert bool(outs[1][0][5, 6].isnan().all()) and bool(outs[1][0][4, 3, 17].isnan())
    keep = [t for t in range(T) if t != 6]
    assert torch.equal(outs[0][1][:, :, keep], outs[1][1][:, :, keep])
    assert torch.equal(outs[0][1][:, 1], outs[1][1][:, 1])  # (token 6: only kv head 0's key is spoilt)


def test_skipped_tokens_stay():
    T, hq, hkv, rd = 12, 6, 2, 128
    qkv, pos, table, (wq, wk) = make(T, hq, hkv, "fp16", rd, 6)
    pos[3], pos[4] = -1, TABLE
    slots = torch.arange(T)
    slots[5], slots[6] = -1, 16 * 2
    d = qkv.cuda()
    c = kvc.allocate_cache(2, 16, hkv, "HND", "cuda")
    c.kv.fill_(77)
    out = torch.full((T, hq, 256), 7.0, dtype=torch.float16, device="cuda")
    pth_dec.norm_rotary_cache_write(d[:, :hq], d[:, hq:hq + hkv], d[:, hq + hkv:], wq.cuda(), wk.cuda(), pos.cuda(), table.cuda(),
                                    c.key_cache, c.value_cache, c.k_scale, c.v_scale, slots.cuda(), query_out=out)
    written = c.kv.cpu()[0]  # [Hkv, 16, 520]
    for t in range(16):
        stays = t >= T or t in (3, 4, 5, 6)
        assert bool((written[:, t] == 77).all()) == stays, t
    assert bool((c.kv[1] == 77).all())
    assert bool((out[3:5] == 7).all()) and not bool((out[5:7] == 7).all())


def test_stream_graph_and_no_tokens():
    T, hq, hkv, rd = 50, 24, 4, 64
    qkv, pos, table, (wq, wk) = make(T, hq, hkv, "bf16", rd, 8)
    d, pos, table, wq, wk = qkv.cuda(), pos.cuda(), table.cuda(), wq.cuda(), wk.cuda()
    slots = torch.arange(T, device="cuda")

    def call(x, c, out):
        pth_dec.norm_rotary_cache_write(x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:], wq, wk, pos[:x.shape[0]], table, c.key_cache,
                                        c.value_cache, c.k_scale, c.v_scale, slots[:x.shape[0]], query_out=out)

    caches = [kvc.allocate_cache(4, 16, hkv, "HND", "cuda") for _ in range(3)]
    outs = [torch.zeros((T, hq, 256), dtype=torch.float16, device="cuda") for _ in range(3)]
    call(d[:0], caches[0], outs[0][:0])
    assert not bool(caches[0].kv.any())
    call(d, caches[0], outs[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(d, caches[1], outs[1])
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(outs[0], outs[1]) and torch.equal(caches[0].kv, caches[1].kv)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(d, caches[2], outs[2])
    for i in range(3):
        d.copy_(qkv.cuda() * (i + 1))
        call(d, caches[0], outs[0])
        outs[2].zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], outs[2]) and torch.equal(caches[0].kv, caches[2].kv)
