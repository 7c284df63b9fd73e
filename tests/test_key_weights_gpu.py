"""decode(..., lse=) and key_weights against float64: the rows' logarithms and every key's accumulated weight within bounds
that count the fp32 roundings, over GQA groups of 1 to 48 rows, one key to long contexts, block sizes 1, 16 and 1,584, both layouts,
padded sequences and tokens, keys past the weights' columns, rows without a logarithm; sums that go on over
several steps, strided weights, streams and a captured graph.

Bounds. A score is s = (sum_d q_d k_d) * (k_scale * scale): the 256 products are exact in fp32 and their sum is off by at
most 256 roundings of partial sums, each 2^-24 of at most A = sum_d |q_d k_d|, the scaling by three roundings of s. In
2^(s log2(e) - lse log2(e)) that is an absolute error of the exponent, so a relative one of the weight: e = 2^-24 (256 A' + 4
|s| + 4 |lse| + 8) with A' = A k_scale scale, the 8 for the exponential itself and for what e^e - 1 is above e. Sums add 2^-24 of the
total per addition.
"""
import numpy as np
import pytest
import torch

import workload as kvc
from mi50_vllm_lab_amd import pth_dec

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def dequant(case, b):
    c, bs = case.cache, case.cache.block_size
    pos = torch.arange(case.seqs[b])
    page, at = case.block_table[b].long()[pos // bs], pos % bs
    return c.key_cache[page, at, :, :256].double().numpy(), c.k_scale[page, at].double().numpy()   # [S, Hkv, 256], [S, Hkv]


def reference(case):
    """lse [T, Hq] and its bound, and per sequence the weights [Hkv, S] for those logarithms (rounded to fp32) with theirs."""
    T, hq = case.num_tokens, case.num_q_heads
    hkv = case.cache.num_kv_heads
    g = hq // hkv
    lse, bound, at, scores = np.full((T, hq), -np.inf), np.zeros((T, hq)), 0, []
    for b, (seq, ql) in enumerate(zip(case.seqs, case.qlens)):
        if seq == 0 or ql == 0:
            scores.append(None)
            at += ql
            continue
        k, ks = dequant(case, b)
        x, size = np.full((ql, hq, seq), -np.inf), np.zeros((ql, hq, seq))
        for j in range(ql):
            see = seq - ql + j + 1
            for h in range(hq):
                q = case.q[at + j, h].double().numpy()
                f = ks[:see, h // g] * case.scale
                x[j, h, :see] = (k[:see, h // g] @ q) * f
                size[j, h, :see] = (np.abs(k[:see, h // g]) @ np.abs(q)) * f
        m = x.max(-1, keepdims=True)
        lse[at:at + ql] = (m + np.log(np.exp(x - m).sum(-1, keepdims=True)))[..., 0]
        fin = np.where(np.isfinite(x), np.abs(x), 0)
        # the sum's relative error is at most its terms' largest, plus a rounding per addition (a lane's keys, the
        # lanes, waves and splits), then the logarithm and the products with ln 2 and log2(e)
        bound[at:at + ql] = U * (256 * size.max(-1) + 8 * fin.max(-1) + seq / 16 + 100 + 8 * np.abs(lse[at:at + ql]))
        scores.append((x, size, at))
        at += ql
    rounded = lse.astype(np.float32).astype(np.float64)
    weights = []
    for b, sc in enumerate(scores):
        if sc is None:
            weights.append(None)
            continue
        x, size, at = sc
        ql, _, seq = x.shape
        r = rounded[at:at + ql, :, None]
        p = np.exp(x - r)
        e = U * (256 * size + 4 * np.where(np.isfinite(x), np.abs(x), 0) + 4 * np.abs(r) + 8)
        w, err = (y.reshape(ql, hkv, g, seq).sum((0, 2)) for y in (p, p * e))
        weights.append((w, err + U * (ql * g + 2) * w))
    return lse, bound, rounded, weights


def run_decode(d, nseg, nsplit, qmax, lse):
    hq = d.num_q_heads
    out = torch.full((d.num_tokens, hq, 256), float("nan"), dtype=torch.float16, device="cuda")
    pth_dec.decode(d.q, d.cache.key_cache, d.cache.value_cache, d.cache.k_scale, d.cache.v_scale, d.block_table, d.seq_lens,
                   d.query_start_loc, out, d.scale, *kvc.partial_buffers(d.num_tokens, hq, nseg, "cuda"), d.num_seqs, qmax, nsplit, lse=lse)
    return out


def add(d, lse, weights, qmax):
    pth_dec.key_weights(d.q, d.cache.key_cache, d.cache.value_cache, d.cache.k_scale, d.cache.v_scale, d.block_table, d.seq_lens,
                        d.query_start_loc, lse, weights, d.scale, d.num_seqs, qmax)


CASES = [
    ([0], [1], 24, 4, 16, "HND", 1),              # one key
    ([40], [1], 1, 1, 1, "NHD", 3),               # one head, one-key blocks
    ([300, 37, 1000], [4, 4, 4], 24, 4, 16, "HND", 8),
    ([700, 16, 31], [8, 2, 5], 12, 2, 1584, "NHD", 4),   # 48 rows per kv head, fewer in some sequences
    ([64, 0, 500, 20], [1, 1, 0, 3], 32, 2, 16, "HND", 4),  # a graph slot without query tokens
    ([257, 90], [2, 1], 21, 7, 48, "HND", 2),
    ([5000], [3], 48, 8, 16, "NHD", 64),
    ([600] * 20, [1] * 20, 24, 4, 16, "HND", 32),  # dealt over the GPU
]


@pytest.mark.parametrize("ctxs,qlens,hq,hkv,bs,layout,nsplit", CASES)
def test_logarithms_and_weights_against_float64(ctxs, qlens, hq, hkv, bs, layout, nsplit):
    case = kvc.make_case(ctxs, qlens, num_q_heads=hq, num_kv_heads=hkv, block_size=bs, layout=layout, seed=len(ctxs) + hq)
    lse, bound, rounded, weights = reference(case)
    d = case.to("cuda")
    qmax = max(qlens)
    got = torch.full((d.num_tokens + 2, hq), 5.0, device="cuda")
    out = run_decode(d, 64, nsplit, qmax, got)
    plain = torch.full_like(out, float("nan"))
    pth_dec.decode(d.q, d.cache.key_cache, d.cache.value_cache, d.cache.k_scale, d.cache.v_scale, d.block_table, d.seq_lens,
                   d.query_start_loc, plain, d.scale, *kvc.partial_buffers(d.num_tokens, hq, 64, "cuda"), d.num_seqs, qmax, nsplit)
    assert torch.equal(out, plain)                                  # the outputs are decode's
    assert bool((got[d.num_tokens:] == 5.0).all())
    err = np.abs(got[:d.num_tokens].double().cpu().numpy() - lse)
    assert (err <= bound).all(), (err - bound).max()
    cols = max(case.seqs) + 3
    big = torch.rand((d.num_seqs + 1, hkv, cols + 5), generator=torch.Generator().manual_seed(4))
    before = big[:, :, :cols].clone().double().numpy()
    w = big.cuda()[:, :, :cols]
    add(d, torch.from_numpy(rounded).float().cuda(), w, qmax)
    after = w.double().cpu().numpy()
    for b, x in enumerate(weights):
        n = 0 if x is None else x[0].shape[1]
        assert (after[b, :, n:] == before[b, :, n:]).all()
        if n:
            want = before[b, :, :n] + x[0]
            off = np.abs(after[b, :, :n] - want)
            assert (off <= x[1] + U * 2 * want).all(), (b, (off - x[1]).max())
    assert (after[len(weights):] == before[len(weights):]).all()


def test_weights_of_a_step_sum_to_its_rows():
    # each row's weights sum to 1: over three steps on one context, to rows x steps per kv head, and a column bound cuts keys off
    case = kvc.make_case([3000], [4], num_q_heads=24, num_kv_heads=4, seed=5)
    d = case.to("cuda")
    w, cut = torch.zeros((1, 4, 3004), device="cuda"), torch.zeros((1, 4, 1000), device="cuda")
    for _ in range(3):
        lse = torch.empty((4, 24), device="cuda")
        run_decode(d, 64, 16, 4, lse)
        add(d, lse, w, 4)
        add(d, lse, cut, 4)
    # each term within 2^-24 (256 A' + ..) < 3e-4 of itself (A' < 20 here), the sums' additions far less
    assert (w.double().sum(-1).cpu() - 72).abs().max() < 72 * 3e-4
    assert torch.equal(cut, w[:, :, :1000])


def test_rows_without_a_logarithm_weigh_nothing_and_masked_keys_do_not_leak():
    case = kvc.make_case([50, 20], [2, 2], num_q_heads=12, num_kv_heads=2, block_size=16, seed=8)
    d = case.to("cuda")
    # the slots behind the last key of the second sequence's block hold NaN scales
    page = int(case.block_table[1, 1])
    d.cache.k_scale[page, 22 - 16:] = float("nan")
    lse = torch.zeros((4, 12), device="cuda")
    lse[1] = float("-inf")
    w = torch.zeros((2, 2, 60), device="cuda")
    add(d, lse, w, 2)
    assert bool(torch.isfinite(w).all())
    lone = torch.zeros((2, 2, 60), device="cuda")
    lse[0] = float("-inf")
    add(d, lse, lone, 2)
    assert not bool(lone[0].any()) and bool((lone[1, :, :22] > 0).all()) and not bool(lone[1, :, 22:].any())
    assert bool((w[0, :, :51] > 0).all()) and not bool(w[0, :, 51:].any())     # row 0 does not see the last key


def test_streams_and_graph():
    case = kvc.make_case([900, 2000], [1, 1], num_q_heads=24, num_kv_heads=4, seed=12)
    d = case.to("cuda")
    lse, w = torch.empty((2, 24), device="cuda"), torch.zeros((2, 4, 2100), device="cuda")
    bufs = kvc.partial_buffers(2, 24, 64, "cuda")
    out = torch.zeros((2, 24, 256), dtype=torch.float16, device="cuda")

    def step():
        pth_dec.decode(d.q, d.cache.key_cache, d.cache.value_cache, d.cache.k_scale, d.cache.v_scale, d.block_table, d.seq_lens,
                       d.query_start_loc, out, d.scale, *bufs, 2, 1, 16, lse=lse)
        add(d, lse, w, 1)

    step()
    one = w.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        w.zero_()
        step()
    side.synchronize()
    assert torch.equal(w, one)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for length in (901, 333, 40):
        d.seq_lens[0] = length
        w.zero_()
        graph.replay()
        got = w.clone()
        w.zero_()
        step()
        assert torch.equal(got, w)
        torch.cuda.synchronize()
