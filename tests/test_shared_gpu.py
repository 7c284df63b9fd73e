"""decode_shared on the GPU against float64: batches from 1 to 300 sequences, prefixes of 0, 1, 31 to 33 keys to thousands, ends
inside blocks, own parts of the query tokens alone to long ones, every kernel form (one and two row blocks of the prefix's
waves; own rows of one wave and of four; 16-key row blocks or not), GQA groups of 1 to 48, both layouts, 4 to 128 segments,
sequences that do not hold the prefix, padded sequences and tokens, NaN in masked places, outlier rows, strided
tensors; the rows' logarithms; streams and a captured graph; and a decode step through all of the operators.

Bounds. Scores in fp32 are off by U (256 A + 4 |s| + 8), U = 2^-24, A = sum_d |q_d k_d| scaled (256 partial sums), which is a relative
error of each weight, of the sum of weights as well. P' = p v_scale is rounded once to fp16: half a step, 2^-11 of it,
below 2^-14 / 16 half a subnormal step. The weighted sums of n keys add (n / 16 + 100) U of sum p |v|. With W = sum p |v| / sum p
an output is off by (2^-11 + 2 e + ..) W, and by half an fp16 step at the end.
"""
import numpy as np
import pytest
import torch

import workload as kvc
from mi50_vllm_lab_amd import pth_dec, rotary

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def say(msg):
    print(msg, flush=True)


def make(own, qlens, prefix, *, hq=24, hkv=4, bs=16, layout="HND", seed=0, **kw):
    """A batch whose sequences hold `prefix` common keys, then own[b] keys of their own and their query tokens; own[b] None: a
    sequence without the prefix, of 40 keys."""
    ctxs = [40 if o is None else prefix + o for o in own]
    case = kvc.make_case(ctxs, qlens, num_q_heads=hq, num_kv_heads=hkv, block_size=bs, layout=layout, seed=seed, **kw)
    c, holders = case.cache, [b for b, o in enumerate(own) if o is not None]
    for b in holders[1:]:
        case.block_table[b, :prefix // bs] = case.block_table[holders[0], :prefix // bs]
        if prefix % bs:
            src, dst = int(case.block_table[holders[0], prefix // bs]), int(case.block_table[b, prefix // bs])
            c.kv[dst, :, :prefix % bs] = c.kv[src, :, :prefix % bs]
    return case


def reference(case, prefix):
    """out, its bound, lse, its bound ([T, Hq, ..], NaN where a row is not written)."""
    c, bs, hq = case.cache, case.cache.block_size, case.num_q_heads
    g = hq // c.num_kv_heads
    T = case.num_tokens
    out, tol = np.full((T, hq, 256), np.nan), np.zeros((T, hq, 256))
    lse, lse_tol = np.full((T, hq), np.nan), np.zeros((T, hq))
    at = 0
    for b, (seq, ql) in enumerate(zip(case.seqs, case.qlens)):
        if seq == 0:
            at += ql
            continue
        pos = torch.arange(seq)
        page, off = case.block_table[b].long()[pos // bs], pos % bs
        for h in range(c.num_kv_heads):
            k, v = (x[page, off, h, :256].double().numpy() for x in (c.key_cache, c.value_cache))
            ks, vs = (x[page, off, h].double().numpy() for x in (c.k_scale, c.v_scale))
            q = case.q[at:at + ql, h * g:(h + 1) * g].double().numpy().reshape(-1, 256)
            s, a = (q @ k.T) * ks * case.scale, (np.abs(q) @ np.abs(k).T) * ks * case.scale
            see = np.arange(seq)[None] <= (seq - ql + np.arange(ql).repeat(g))[:, None]
            s, a = np.where(see, s, -np.inf), np.where(see, a, 0)
            m = s.max(-1, keepdims=True)
            p = np.exp(s - m)
            tot = p.sum(-1, keepdims=True)
            val = v * vs[:, None]
            e = U * (256 * a.max(-1) + 8 * np.abs(np.where(see, s, 0)).max(-1) + 8)[:, None]
            w = (p / tot) @ np.abs(val)
            o = (p / tot) @ val
            n = (seq / 16 + 100) * U
            # P' is formed as 16 p v_scale: below 2^-14 its half step is 2^-25
            small = 2.0 ** -25 / 16 * np.abs(v).sum(0)[None] / tot
            err = (2.0 ** -11 + 2 * e + 2 * n) * w + small
            rows = (slice(at, at + ql), slice(h * g, (h + 1) * g))
            out[rows], tol[rows] = (x.reshape(ql, g, 256) for x in (o, err))
            lse[rows] = (m + np.log(tot))[:, 0].reshape(ql, g)
            lse_tol[rows] = (e + n)[:, 0].reshape(ql, g) + U * 8 * np.abs(lse[rows])
        at += ql
    with np.errstate(invalid="ignore"):
        tol += kvc.fp16_half_ulp(np.abs(out) + tol)
    return out, tol, lse, lse_tol


def run(d, prefix, qmax, nseg=64, lse=None, num_seqs=None, out=None, q=None, bufs=None):
    q = d.q if q is None else q
    if out is None:
        out = torch.full((q.shape[0], d.num_q_heads, 256), float("nan"), dtype=torch.float16, device="cuda")
    c = d.cache
    if bufs is None:
        bufs = kvc.partial_buffers(q.shape[0], d.num_q_heads, nseg, "cuda")
    pth_dec.decode_shared(q, c.key_cache, c.value_cache, c.k_scale, c.v_scale, d.block_table, d.seq_lens, d.query_start_loc, out, d.scale,
                          *bufs, d.num_seqs if num_seqs is None else num_seqs, qmax, prefix, lse=lse)
    return out


def compare(case, prefix, out, lse=None):
    want, tol, wl, tl = reference(case, prefix)
    got = out.double().cpu().numpy()
    dead = np.isnan(want)
    assert np.isnan(got[dead]).all()                      # rows of padded sequences were not written
    err = np.abs(got - want)[~dead]
    assert np.isfinite(err).all() and (err <= tol[~dead]).all(), float((err - tol[~dead]).max())
    if lse is not None:
        e = np.abs(lse.double().cpu().numpy() - wl)
        live = ~np.isnan(wl)
        assert (e[live] <= tl[live]).all(), float((e - tl)[live].max())


CASES = [
    # own keys, query tokens, prefix, and what differs from 24 / 4 heads, block size 16, 64 segments
    ([20, 5], [1, 1], 64, {}),
    ([5] * 25 + [300], [1] * 26, 12321, dict(hq=6, hkv=1)),        # 156 rows behind a long prefix: two row blocks per wave
    # few segments over long runs: block tables that do not fit the workgroup's LDS, of the prefix and of own keys
    ([40000, 3], [1, 1], 40000, dict(hq=6, hkv=1, nseg=4)),
    ([40000, 3], [3, 1], 40000, dict(hq=6, hkv=1, nseg=4)),
    ([20000, 3], [1, 3], 20000, dict(hq=6, hkv=1, nseg=4, bs=8, layout="NHD")),
    ([0], [1], 0, {}),                                            # one sequence, nothing shared, one key
    ([0, 0, 0], [1, 1, 1], 1, {}),                                # one shared key
    ([3, 40, 0], [1, 2, 1], 31, {}),
    ([3, 40, 0], [1, 2, 1], 32, {"bs": 32}),
    ([3, 40, 0], [1, 2, 1], 33, {"layout": "NHD"}),
    ([100, 300, 7, 55], [1] * 4, 2048, {}),                       # 24 rows per kv head
    ([100, 300, 7, 55, 12], [1] * 5, 1000, {}),                   # 30 rows
    ([100, 300, 7, 55, 12, 1], [1] * 6, 1000, {}),                # 36 rows: 192-row tiles
    ([9, 900, 30], [4, 4, 4], 500, {"hq": 12, "hkv": 2, "bs": 1584}),
    ([9, 900, 30, 2] * 5, [3] * 20, 1584, {"hq": 12, "hkv": 2, "bs": 1584, "layout": "NHD"}),
    ([50] * 32, [1] * 32, 300, {}),                               # one full row tile
    ([50] * 33, [1] * 33, 300, {}),                               # and one more row
    ([17 * (i % 9) for i in range(80)], [1] * 80, 700, {}),       # more than 64 sequences
    ([11 * (i % 30) for i in range(300)], [1] * 300, 128, {"hq": 4, "hkv": 2}),
    ([40, 0, 200], [8, 8, 8], 350, {}),                           # 48 rows: two slices
    ([40, 0, 200], [8, 3, 6], 350, {}),                           # and sequences without the second
    ([40, 90], [6, 5], 77, {"bs": 1}),                            # 36 rows: the second slice has 4
    ([60, 5], [1, 1], 400, {"hq": 48, "hkv": 1}),                 # 48 query heads on one kv head
    ([60, 5, 8, 3], [1, 2, 1, 1], 400, {"hq": 7, "hkv": 1}),      # 27 tokens per row tile
    ([60, 5] * 20, [2, 1] * 20, 400, {"hq": 7, "hkv": 7}),        # one query head per kv head
    ([70, 3, 20], [1] * 3, 600, {"nseg": 4}),
    ([70, 3, 20] * 4, [1] * 12, 600, {"nseg": 5}),
    ([700, 3, 20] * 4, [1] * 12, 600, {"nseg": 128}),
    ([5000, 3], [1, 1], 4000, {}),                                # one long own part
    ([30, 10] * 10, [4] * 20, 9000, {"hq": 12, "hkv": 2}),
    ([100, 300, 7, 55] * 3, [1] * 12, 800, {"outlier_frac": 0.02}),
    ([4, None, 100, None], [1, 2, 1, 1], 200, {}),                # two sequences without the prefix
    ([None, None, 4, 100] * 4, [1] * 16, 200, {}),                # the first that holds it is the third
    ([None] * 3, [1, 2, 3], 60, {}),                              # nobody holds it
]


@pytest.mark.parametrize("own,qlens,prefix,kw", CASES)
def test_against_float64(own, qlens, prefix, kw):
    kw = dict(kw)
    nseg = kw.pop("nseg", 64)
    say(f"shared: {len(own)} sequences, prefix {prefix}, {kw}")
    case = make(own, qlens, prefix, seed=len(own) + prefix, **kw)
    d = case.to("cuda")
    lse = torch.full((d.num_tokens + 1, d.num_q_heads), 7.0, device="cuda")
    out = run(d, prefix, max(qlens), nseg, lse)
    torch.cuda.synchronize()
    compare(case, prefix, out, lse[:-1])
    assert bool((lse[-1] == 7.0).all())
    # again, without logarithms: the same
    assert torch.equal(run(d, prefix, max(qlens), nseg).view(torch.int16), out.view(torch.int16))


def test_padded_sequences_and_tokens():
    # sequences 1 (no query tokens), 3 (seq_len 0) and 5 are padding, and three tokens lie behind the last sequence
    case = make([30, 5, 80, 9, 12, 33], [1, 0, 2, 1, 1, 0], 150, seed=3)
    case.ctxs[3], case.seq_lens[3] = -1, 0
    assert case.seqs[3] == 0
    for first_dead in (False, True):
        if first_dead:
            case.ctxs[0], case.seq_lens[0] = -1, 0
        d = case.to("cuda")
        T = d.num_tokens
        q = torch.full((T + 3, 24, 256), float("nan"), dtype=torch.float16, device="cuda")
        q[:T] = d.q
        out = run(d, 150, 2, q=q)
        assert bool(torch.isnan(out[T:]).all())
        compare(case, 150, out[:T])
        lone = run(d, 150, 2, q=q, num_seqs=3)          # the first three sequences alone
        assert torch.isnan(lone[3:]).all() and torch.equal(torch.isnan(lone[:3]), torch.isnan(out[:3]))


def test_all_sequences_dead():
    case = make([3, 4], [1, 1], 50, seed=4)
    case.seq_lens.zero_()
    out = run(case.to("cuda"), 50, 1)
    assert bool(torch.isnan(out).all())


def test_query_tokens_beyond_qmax_are_left_alone():
    case = make([30, 50], [4, 2], 100, seed=5)
    d = case.to("cuda")
    out = run(d, 100, 2)
    assert bool(torch.isnan(out[2:4]).all())
    want, tol, _, _ = reference(case, 100)
    got = out.double().cpu().numpy()
    rows = [0, 1, 4, 5]
    assert (np.abs(got - want)[rows] <= tol[rows]).all()


def test_nan_behind_the_last_keys_does_not_leak():
    case = make([30, 5, 61], [1, 1, 1], 120, seed=6)
    c, bs = case.cache, 16
    for b, n in enumerate(case.seqs):
        page = int(case.block_table[b, (n - 1) // bs])
        for x in (c.k_scale, c.v_scale):
            x[page, (n - 1) % bs + 1:] = float("nan")
    d = case.to("cuda")
    compare(case, 120, run(d, 120, 1))


def test_strided_query_and_output():
    case = make([30, 5, 61, 9], [2, 1, 2, 1], 120, seed=7, q_noncontig=True)
    d = case.to("cuda")
    plain = run(d, 120, 2)
    big = torch.full((6, 30, 512), 9.0, dtype=torch.float16, device="cuda")
    view = big[:, 3:27, 128:384]
    view.fill_(float("nan"))
    run(d, 120, 2, out=view)
    assert torch.equal(view, plain)
    rest = big.clone()
    rest[:, 3:27, 128:384] = 9.0
    assert bool((rest == 9.0).all())


def test_agrees_with_decode():
    case = make([30, 500, 61, 9] * 6, [1, 2, 4, 1] * 6, 900, seed=8)
    d = case.to("cuda")
    out, lse, lse2 = run(d, 900, 4), torch.empty((48, 24), device="cuda"), torch.empty((48, 24), device="cuda")
    run(d, 900, 4, lse=lse)
    whole = torch.empty_like(out)
    c = d.cache
    pth_dec.decode(d.q, c.key_cache, c.value_cache, c.k_scale, c.v_scale, d.block_table, d.seq_lens, d.query_start_loc, whole, d.scale,
                   *kvc.partial_buffers(48, 24, 64, "cuda"), 24, 4, 8, lse=lse2)
    _, tol, _, tl = reference(case, 900)
    assert ((out.double() - whole.double()).abs().cpu().numpy() <= 2 * tol).all()
    assert ((lse.double() - lse2.double()).abs().cpu().numpy() <= 2 * tl).all()


def test_two_streams_at_once():
    a, b = make([30, 500, 61, 9] * 3, [1] * 12, 900, seed=9).to("cuda"), make([40, 5], [4, 4], 3000, hq=12, hkv=2, seed=10).to("cuda")
    ra, rb = run(a, 900, 1), run(b, 3000, 4)
    torch.cuda.synchronize()
    s, t = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(3):
        for x in (s, t):
            x.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            xa = run(a, 900, 1)
        with torch.cuda.stream(t):
            xb = run(b, 3000, 4)
        torch.cuda.synchronize()
        assert torch.equal(xa, ra) and torch.equal(xb, rb)


def test_captured_graph():
    case = make([30, 500, 61, 9, 200, 44], [1] * 6, 640, seed=11)
    d = case.to("cuda")
    bufs = kvc.partial_buffers(6, 24, 64, "cuda")
    out = torch.zeros((6, 24, 256), dtype=torch.float16, device="cuda")
    run(d, 640, 1, out=out, bufs=bufs)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run(d, 640, 1, out=out, bufs=bufs)
    for lens in ([671, 1141, 702, 650, 841, 685], [641, 641, 641, 641, 641, 641], [100, 900, 702, 0, 700, 20]):
        d.seq_lens.copy_(torch.tensor(lens, dtype=torch.int32))
        out.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        out.fill_(float("nan"))
        run(d, 640, 1, out=out, bufs=bufs)
        assert torch.equal(got.view(torch.int16), out.view(torch.int16))
        case.seq_lens = torch.tensor(lens, dtype=torch.int32)
        case.ctxs = [n - 1 for n in lens]
        compare(case, 640, got)


def test_a_step_through_all_operators():
    """Rotary cache write, shared-prefix decode with its logarithms, key weights, eviction, and a decode over what was kept."""
    n, prefix, hq, hkv, keep, recent = 6, 320, 24, 4, 100, 10
    case = make([31 * i for i in range(n)], [1] * n, prefix, seed=12, spare_blocks=3 + n * 8)
    used = set(case.block_table.flatten().tolist())
    free = [p for p in range(case.cache.num_blocks) if p not in used]
    d = case.to("cuda")
    c = d.cache
    views = (c.key_cache, c.value_cache, c.k_scale, c.v_scale)
    g = torch.Generator().manual_seed(13)
    qkv = torch.randn((n, hq + 2 * hkv, 256), generator=g).bfloat16().cuda()
    lens = case.seq_lens.long()
    pos = (lens - 1).cuda()
    slots = torch.stack([case.block_table[b].long()[(lens[b] - 1) // 16] * 16 + (lens[b] - 1) % 16 for b in range(n)]).cuda()
    q = torch.empty((n, hq, 256), dtype=torch.float16, device="cuda")
    pth_dec.rotary_cache_write(qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:], pos, rotary.rotary_table(128, 600, device="cuda"),
                               *views, slots, query_out=q)
    lse = torch.empty((n, hq), device="cuda")
    out = run(d, prefix, 1, lse=lse, q=q)
    w = torch.zeros((n, hkv, int(lens.max())), device="cuda")
    pth_dec.key_weights(q, *views, d.block_table, d.seq_lens, d.query_start_loc, lse, w, d.scale, n, 1)
    nbt = torch.tensor(free[:n * 7], dtype=torch.int32, device="cuda").view(n, 7)
    nlens, nw = torch.zeros(n, dtype=torch.int32, device="cuda"), torch.zeros((n, hkv, keep + 50), device="cuda")
    kept = torch.zeros((n, hkv, keep), dtype=torch.int32, device="cuda")
    pth_dec.evict(w, *views, d.block_table, d.seq_lens, nbt, nlens, nw, kept, n, keep, recent)
    less = torch.empty_like(out)
    pth_dec.decode(q, *views, nbt, nlens, d.query_start_loc, less, d.scale, *kvc.partial_buffers(n, hq, 64, "cuda"), n, 1, 4)
    torch.cuda.synchronize()
    # what was written is what the float64 reference reads, so the first attention is checked as any other
    case.q = q.cpu()
    case.cache = kvc.clone_cache(c, "cpu")
    compare(case, prefix, out, lse)
    # weights of a row sum to 1 (see the key weights' test for the bound)
    assert (w.double().sum(-1).cpu() - hq // hkv).abs().max() < 6 * 3e-4
    assert nlens.tolist() == [keep] * n
    for b in range(n):
        for h in range(hkv):
            mine = w[b, h, :int(lens[b])].tolist()
            old = int(lens[b]) - recent
            stay = sorted(sorted(range(old), key=lambda t: (-mine[t], t))[:keep - recent] + list(range(old, int(lens[b]))))
            assert kept[b, h].tolist() == stay and nw[b, h, :keep].tolist() == [mine[t] for t in stay]
    # the second attention: the same rows over the kept keys
    case.block_table, case.seq_lens, case.ctxs = nbt.cpu(), nlens.cpu(), [keep - 1] * n
    compare(case, prefix, less)
