"""rotary_cache_write on the GPU: queries against a float64 rotation within the roundings of the formula, cache bytes equal to
the cache writer's for the rotated key (bit for bit), both pair layouts, rotary dims from 8 to 256, the three input types, in place and into
another tensor, block sizes 16, 1,584 and 1, skipped tokens, 0 and 1 tokens, either kernel form (one and four heads per
lane group); two streams, and a captured graph.
"""
import numpy as np
import pytest
import torch

import workload as kvc
from mi50_vllm_lab_amd import pth_dec, rotary
from oracle import kvwrite as kvw

pytestmark = pytest.mark.gpu
DT = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
TABLE = 600


def rotate32(x, cos_sin, pos, interleaved):
    """x [T, H, 256] on the CPU in fp32, each product and sum rounded (numpy)."""
    x = x.float().numpy().copy()
    rd = cos_sin.shape[1]
    cs = cos_sin.numpy()[pos.numpy()]
    c, s = cs[:, None, :rd // 2], cs[:, None, rd // 2:]
    first, second = (slice(0, rd, 2), slice(1, rd, 2)) if interleaved else (slice(0, rd // 2), slice(rd // 2, rd))
    a, b = x[..., first].copy(), x[..., second].copy()
    x[..., first], x[..., second] = a * c - b * s, b * c + a * s
    return x


def make(T, hq, hkv, dtype, rd, seed, scaling=None):
    g = torch.Generator().manual_seed(seed)
    qkv = torch.randn((T, hq + 2 * hkv, 256), generator=g)
    if T > 3:
        qkv[1] = 0.0           # an all-zero token: scale 0
        qkv[2] *= 40
        qkv[3, :, rd:] = 0.0   # only the rotated part
    pos = torch.randint(0, TABLE, (T,), generator=g)
    if T > 0:
        pos[0], pos[-1] = 0, TABLE - 1
    return qkv.to(DT[dtype]), pos, rotary.rotary_table(rd, TABLE, 1e4, scaling)


@pytest.mark.parametrize("T,hq,hkv,dtype,rd,interleaved,out,bs,layout", [
    (1, 24, 4, "fp16", 256, False, "inplace", 16, "HND"),
    (1, 1, 1, "fp32", 8, True, "inplace", 1, "NHD"),
    (5, 24, 4, "bf16", 64, False, "fp16", 16, "NHD"),
    (7, 12, 2, "fp16", 128, True, "same", 1584, "HND"),
    (33, 6, 6, "fp32", 96, False, "fp16", 32, "HND"),
    (130, 5, 1, "bf16", 200, True, "same", 16, "HND"),
    (64, 24, 4, "fp32", 256, True, "inplace", 16, "NHD"),
    (301, 24, 4, "bf16", 56, False, "inplace", 16, "HND"),
    (513, 24, 4, "fp16", 64, True, "inplace", 48, "HND"),      # four heads per lane group
    (700, 7, 1, "fp32", 256, False, "same", 1584, "NHD"),      # heads not a multiple of four
    (1100, 24, 4, "bf16", 120, False, "fp16", 16, "HND"),
])
def test_against_float64_and_the_cache_writer(T, hq, hkv, dtype, rd, interleaved, out, bs, layout):
    qkv, pos, table = make(T, hq, hkv, dtype, rd, seed=T + rd)
    d = qkv.cuda()
    q, k, v = d[:, :hq], d[:, hq:hq + hkv], d[:, hq + hkv:]
    before = qkv.clone()
    blocks = -(-T // bs) + 2
    slots = torch.randperm(blocks * bs, generator=torch.Generator().manual_seed(5))[:T]
    caches = [kvc.allocate_cache(blocks, bs, hkv, layout, "cuda") for _ in range(2)]
    for c in caches:
        c.kv.fill_(77)
    qout = q if out == "inplace" else torch.full((T, hq + 1, 256), 7.0, dtype=DT[dtype] if out == "same" else torch.float16,
                                                 device="cuda")[:, :hq]
    c = caches[0]
    pth_dec.rotary_cache_write(q, k, v, pos.cuda(), table.cuda(), c.key_cache, c.value_cache, c.k_scale, c.v_scale, slots.cuda(),
                               interleaved=interleaved, query_out=None if out == "inplace" else qout)
    torch.cuda.synchronize()
    # the query: fp32 with three roundings, each at most 2^-24 of its own result (|x c| + |y s| bounds all three), then
    # one rounding to the output type: eps / 2 of the value, below the normal range half a subnormal step
    x = before[:, :hq].double().numpy()
    cs = table.double().numpy()[pos.numpy()]
    half = rd // 2
    cc, ss = cs[:, None, :half], cs[:, None, half:]
    fi, se = (slice(0, rd, 2), slice(1, rd, 2)) if interleaved else (slice(0, half), slice(half, rd))
    ref, size = x.copy(), np.zeros_like(x)
    a, b = x[..., fi], x[..., se]
    ref[..., fi], ref[..., se] = a * cc - b * ss, b * cc + a * ss
    size[..., fi], size[..., se] = np.abs(a * cc) + np.abs(b * ss), np.abs(b * cc) + np.abs(a * ss)
    fi32 = 2 * 2.0 ** -24 * size
    t = torch.finfo(qout.dtype)
    bound = fi32 + t.eps / 2 * (np.abs(ref) + fi32) + t.tiny * t.eps / 2
    err = np.abs(qout.double().cpu().numpy() - ref)
    assert (err <= bound).all(), float((err - bound).max())
    # the dims behind the rotated ones come over as they are (through the output's rounding)
    assert torch.equal(qout[..., rd:].cpu(), before[:, :hq, rd:].to(qout.dtype))
    assert torch.equal(d[:, hq:].cpu(), before[:, hq:])                    # key and value stay
    if out != "inplace":
        assert torch.equal(d.cpu(), before)
        assert bool((qout.as_strided((T, 1, 256), ((hq + 1) * 256, 256, 1), qout.storage_offset() + hq * 256) == 7.0).all())
    # the cache: the bytes that the writer stores for the key rotated in fp32
    c = caches[1]
    kr = torch.from_numpy(rotate32(before[:, hq:hq + hkv], table, pos, interleaved)).cuda()
    pth_dec.cache_write(kr, v.float(), c.key_cache, c.value_cache, c.k_scale, c.v_scale, slots.cuda())
    assert torch.equal(caches[0].kv, caches[1].kv)


def test_key_scale_and_values_within_half_a_step():
    T, hkv = 40, 4
    qkv, pos, table = make(T, 24, hkv, "fp32", 256, seed=9)
    c = kvc.allocate_cache(4, 16, hkv, "HND", "cuda")
    d = qkv.cuda()
    slots = torch.arange(T)
    pth_dec.rotary_cache_write(d[:, :24], d[:, 24:28], d[:, 28:], pos.cuda(), table.cuda(), c.key_cache, c.value_cache, c.k_scale,
                               c.v_scale, slots.cuda())
    ref = rotate32(qkv[:, 24:28], table, pos, False).astype(np.float64)
    got = c.key_cache[slots // 16, slots % 16, :, :256].double().cpu().numpy()
    scale = c.k_scale[slots // 16, slots % 16].double().cpu().numpy()[..., None]
    assert (np.abs(got * scale - ref) <= scale * (0.5 + 127 * 2.0 ** -22)).all()
    q, s = kvw.quantize_rows(ref.astype(np.float32))
    assert (q == got).all() and (s == scale[..., 0]).all()


def test_skipped_tokens_leave_everything_as_it_was():
    T, hq, hkv = 12, 24, 4
    qkv, pos, table = make(T, hq, hkv, "fp16", 128, seed=11)
    slots = torch.arange(T)
    slots[2], slots[5] = -1, 64                      # padding, and past the cache's 64 slots: no row, the query turns
    pos[7], pos[8], pos[9] = -1, TABLE, 1 << 40      # outside the table: nothing at all
    c = kvc.allocate_cache(4, 16, hkv, "HND", "cuda")
    c.kv.fill_(55)
    d, out = qkv.cuda(), torch.full((T, hq, 256), 3.0, dtype=torch.float16, device="cuda")
    pth_dec.rotary_cache_write(d[:, :hq], d[:, hq:hq + hkv], d[:, hq + hkv:], pos.cuda(), table.cuda(), c.key_cache, c.value_cache,
                               c.k_scale, c.v_scale, slots.cuda(), query_out=out)
    live = pos.clone()
    live[7:10] = 0
    want = torch.from_numpy(rotate32(qkv[:, :hq], table, live, False)).half()
    want[7:10] = 3.0
    assert torch.equal(out.cpu(), want)
    rows = c.kv.cpu().transpose(1, 2).reshape(64, hkv, 520)
    untouched = [s for s in range(64) if s >= T or s in (2, 5, 7, 8, 9)]
    assert bool((rows[untouched] == 55).all())
    assert bool((rows[[0, 1, 3, 4, 6, 10, 11]] != 55).any(-1).all())


def test_no_tokens_and_strided_table():
    c = kvc.allocate_cache(2, 16, 4, "HND", "cuda")
    big = rotary.rotary_table(64, 50, device="cuda")
    table = torch.zeros((50, 128), device="cuda")[:, :64]
    table.copy_(big)
    d = torch.randn((9, 32, 256), device="cuda")
    views = (c.key_cache, c.value_cache, c.k_scale, c.v_scale)
    n = torch.zeros(0, dtype=torch.int64, device="cuda")
    e = d[:0]
    pth_dec.rotary_cache_write(e[:, :24], e[:, 24:28], e[:, 28:], n, table, *views, n)
    assert not bool(c.kv.any())
    pos, slots = torch.arange(9, device="cuda") * 5, torch.arange(9, device="cuda")
    outs = []
    for t in (table, big):
        o = torch.empty((9, 24, 256), device="cuda")
        pth_dec.rotary_cache_write(d[:, :24], d[:, 24:28], d[:, 28:], pos, t, *views, slots, query_out=o)
        outs.append((o, c.kv.clone()))
    assert torch.equal(outs[0][0], outs[1][0]) and torch.equal(outs[0][1], outs[1][1])


def test_tensors_on_different_devices_are_refused():
    c = kvc.allocate_cache(2, 16, 4, "HND", "cuda")
    d = torch.randn((2, 32, 256), device="cuda")
    n = torch.zeros(2, dtype=torch.int64, device="cuda")
    with pytest.raises(RuntimeError, match="one GPU"):
        pth_dec.rotary_cache_write(d[:, :24], d[:, 24:28], d[:, 28:], n, torch.zeros((9, 64)), c.key_cache, c.value_cache, c.k_scale,
                                   c.v_scale, n)


def test_streams_and_graph():
    T, hq, hkv = 300, 24, 4
    qkv, pos, table = make(T, hq, hkv, "bf16", 256, seed=21)
    d, pos, table, slots = qkv.cuda(), pos.cuda(), table.cuda(), torch.arange(T, device="cuda")
    c = kvc.allocate_cache(20, 16, hkv, "HND", "cuda")
    out = torch.zeros((T, hq, 256), dtype=torch.float16, device="cuda")

    def call():
        pth_dec.rotary_cache_write(d[:, :hq], d[:, hq:hq + hkv], d[:, hq + hkv:], pos, table, c.key_cache, c.value_cache, c.k_scale,
                                   c.v_scale, slots, query_out=out)

    call()
    want = (out.clone(), c.kv.clone())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        with torch.cuda.stream(side):
            out.zero_()
            c.kv.zero_()
            call()
        side.synchronize()
        assert torch.equal(out, want[0]) and torch.equal(c.kv, want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for step in range(3):
        pos.copy_((pos * 7 + 3) % TABLE)
        out.zero_()
        c.kv.zero_()
        graph.replay()
        got = (out.clone(), c.kv.clone())
        out.zero_()
        c.kv.zero_()
        call()
        assert torch.equal(out, got[0]) and torch.equal(c.kv, got[1]), step
