"""decode with a window and sink keys on the GPU against float64: windows and sinks that overlap, touch, lie far apart or hold
every key, more sinks than a tile or the sequence has, causal and non-causal rows, 1 to 48 rows per kv head, block sizes 1 to 1,584,
pages between the sinks and the window at a block of NaN, split, sliced and dealt launches, outlier rows (sinks often are), the
rows' logarithms, padded slots; as before without sinks; on two streams and in a captured graph.

Tolerance: workload.fp16_output_errors, the bar of every decode test (2e-3 and 2e-4 before the output's rounding to fp16);
logarithms as in the key weights' tests: scores carry fp32 products of exact fp16 and int8 operands, 1e-5 covers 256 of them.
"""
import random

import numpy as np
import pytest
import torch

import window_oracle
import workload as kvc
from mi50_vllm_lab_amd import pth_dec, vllm_shim

pytestmark = pytest.mark.gpu


def run(case, bt, window, sinks, causal, nsplit, nseg=None, lse=False, qmax=None):
    d = case.to("cuda")
    out = torch.full((case.num_tokens, case.num_q_heads, 256), 7.0, dtype=torch.float16, device="cuda")
    po, pm, pl = kvc.partial_buffers(case.num_tokens, case.num_q_heads, nseg or max(nsplit, 1), "cuda")
    for x in (po, pm, pl):
        x.fill_(float("nan"))
    ln = torch.full((case.num_tokens, case.num_q_heads), 7.0, device="cuda") if lse else None
    pth_dec.decode(d.q, d.cache.key_cache, d.cache.value_cache, d.cache.k_scale, d.cache.v_scale, bt.cuda(), d.seq_lens,
                   d.query_start_loc, out, case.scale, po, pm, pl, case.num_seqs, qmax or case.qmax, nsplit, window=window,
                   causal=causal, lse=ln, sinks=sinks)
    torch.cuda.synchronize()
    return out.cpu(), None if ln is None else ln.cpu()


def check(case, window, sinks, causal=True, nsplit=4, nseg=None, lse=False, qmax=None):
    bt, _ = window_oracle.freed(case, window, sinks) if window > 0 else (case.block_table, 0)
    ref, ln, written = window_oracle.windowed(case, window, sinks, causal, bt, qmax)
    out, got = run(case, bt, window, sinks, causal, nsplit, nseg, lse, qmax)
    assert bool((out[~written] == 7.0).all())
    _, _, worst, mean = kvc.fp16_output_errors(out.double().numpy()[written], ref[written])
    assert worst <= 0 and mean <= 2e-4, (worst, mean)
    if lse:
        assert np.abs(got.double().numpy()[written] - ln[written]).max() <= 1e-5 + 1e-6 * np.abs(ln[written]).max()
        assert bool((got[~written] == 7.0).all())


@pytest.mark.parametrize("ctx,qlen,window,sinks,causal,bs,layout,hq,hkv,nsplit", [
    (1000, 1, 100, 4, True, 16, "HND", 24, 4, 4),        # far apart
    (1000, 1, 100, 33, True, 16, "HND", 24, 4, 1),       # more sinks than a tile
    (1000, 4, 100, 64, True, 16, "NHD", 24, 4, 8),       # whole tiles
    (500, 4, 460, 37, True, 16, "HND", 24, 4, 8),        # the window begins two keys behind the last sink
    (500, 4, 464, 37, True, 16, "HND", 24, 4, 8),        # touching, by the row
    (500, 4, 480, 37, True, 16, "HND", 24, 4, 8),        # overlapping
    (500, 4, 505, 37, True, 16, "HND", 24, 4, 8),        # rows that see everything
    (500, 8, 33, 1, False, 16, "HND", 24, 4, 3),         # 48 rows, non-causal
    (500, 3, 1, 16, True, 16, "HND", 12, 2, 2),          # a window of the row itself
    (500, 1, 64, 600, True, 16, "HND", 24, 4, 4),        # more sinks than keys
    (0, 3, 2, 1, True, 16, "HND", 24, 4, 4),             # the first tokens
    (0, 1, 1, 1, True, 16, "HND", 6, 6, 4),
    (31, 1, 1, 31, True, 16, "HND", 24, 4, 4),           # sinks and the row itself, in one tile
    (70, 2, 5, 40, True, 8, "HND", 24, 4, 4),            # pages inside a 16-key block, given back one by one
    (70, 2, 5, 3, False, 1, "NHD", 5, 1, 4),
    (900, 4, 200, 50, True, 24, "HND", 24, 4, 8),        # pages that no 16-key block divides
    (4000, 4, 700, 37, True, 1584, "NHD", 12, 2, 8),
    (9000, 4, 2048, 4, True, 16, "HND", 24, 4, 16),      # waves interleaved over the gap
    (20000, 2, 8192, 128, True, 32, "HND", 24, 4, 64),
    (30000, 1, 14000, 20, True, 16, "HND", 24, 4, 1),    # more blocks than a wave keeps in LDS
    (30000, 1, 9000, 20, True, 3, "HND", 6, 1, 2),
])
def test_one_sequence(ctx, qlen, window, sinks, causal, bs, layout, hq, hkv, nsplit):
    case = kvc.make_case([ctx], [qlen], num_q_heads=hq, num_kv_heads=hkv, block_size=bs, layout=layout, seed=ctx + window + sinks)
    check(case, window, sinks, causal, nsplit, lse=sinks % 2 == 0)


@pytest.mark.parametrize("seed", range(24))
def test_random_batches(seed):
    rng = random.Random(seed)
    hq, hkv = rng.choice([(24, 4), (12, 2), (6, 6), (5, 1), (16, 1)])
    g = hq // hkv
    qmost = rng.choice([1, 2, 4, 8])
    qmost = max(1, min(qmost, 48 // g))
    n = rng.choice([1, 3, 7, 40])
    qlens = [rng.choice([0, 1, qmost]) for _ in range(n)]
    qlens[-1] = qmost
    ctxs = [rng.choice([0, 1, rng.randint(0, 100), rng.randint(0, 3500 if n < 10 else 900)]) for _ in range(n)]
    case = kvc.make_case(ctxs, qlens, num_q_heads=hq, num_kv_heads=hkv, block_size=rng.choice([1, 8, 16, 16, 32, 48, 1584]),
                         layout=rng.choice(["HND", "NHD"]), seed=seed, q_noncontig=rng.random() < 0.3,
                         outlier_frac=rng.choice([0.0, 0.02]))
    check(case, rng.choice([1, 7, 100, 1000, 2048]), rng.choice([1, 4, 16, 37, 128, 1000]), rng.random() < 0.7,
          rng.choice([1, 2, 5, 16, 64]), nseg=64, lse=rng.random() < 0.5)


@pytest.mark.parametrize("n,qlen,window,sinks", [(48, 1, 512, 4), (40, 4, 300, 37), (90, 1, 64, 64)])
def test_dealt_batches(n, qlen, window, sinks):
    """Batches that pd_sinks_balanced_kernel takes: more splits than CUs."""
    ctxs = [17 * i % 1500 for i in range(n)]
    case = kvc.make_case(ctxs, [qlen] * n, seed=n)
    check(case, window, sinks, True, 64, lse=True)


def test_sliced_rows_count_the_sinks():
    """4 sequences of 8 rows (48 per kv head) over 1,024 keys and sinks run sliced, over 4,096 not: both against float64."""
    case = kvc.make_case([3000, 2000, 5000, 4500], [8] * 4, seed=2)
    check(case, 1024, 64, False, 5)
    check(case, 4096, 64, True, 5)


def test_outlier_sinks():
    """Sinks whose values are large, behind a window of ordinary ones: the weights enter P.V as hi + lo."""
    case = kvc.make_case([6000, 900], [4, 4], seed=5)
    for b in range(2):
        kvc.write_tokens(case.cache, case.block_table[b], torch.arange(4), *kvc.quantize_per_token_head(torch.randn(4, 4, 256)),
                         *kvc.quantize_per_token_head(60 * torch.randn(4, 4, 256)))
    check(case, 512, 4, True, 8)


def test_without_a_window_or_sinks_nothing_changes():
    case = kvc.make_case([700, 300], [4, 1], seed=6)
    plain = [run(case, case.block_table, w, 0, True, 4)[0] for w in (-1, 200)]
    assert torch.equal(run(case, case.block_table, -1, 5, True, 4)[0], plain[0])
    assert torch.equal(run(case, case.block_table, 0, 5, True, 4)[0], plain[0])
    ref, _, written = window_oracle.windowed(case, 200, 0)
    assert kvc.fp16_output_errors(plain[1].double().numpy()[written], ref[written])[2] <= 0


@pytest.mark.parametrize("window,sinks", [((1 << 31) - 1, 5), (1 << 30, (1 << 31) - 1), (40, (1 << 31) - 1)])
def test_the_largest_windows_and_sinks(window, sinks):
    """Every key is seen; the first sequence has fewer keys than rows."""
    case = kvc.make_case([0, 300], [4, 4], seed=13)
    d = case.to("cuda")
    lens = torch.tensor([2, 304], dtype=torch.int32)
    out = torch.full((8, 24, 256), 7.0, dtype=torch.float16, device="cuda")
    pth_dec.decode(d.q, d.cache.key_cache, d.cache.value_cache, d.cache.k_scale, d.cache.v_scale, d.block_table, lens.cuda(), d.query_start_loc,
                   out, d.scale, *kvc.partial_buffers(8, 24, 4, "cuda"), 2, 4, 4, window=window, sinks=sinks)
    assert bool((out[:2] == 0).all())  # positions -2 and -1
    tail = kvc.DecodeCase(case.q[2:], case.cache, case.block_table, lens, torch.tensor([0, 2, 6], dtype=torch.int32), [0, 300], [2, 4], 24,
                          case.scale)
    ref, _, _ = window_oracle.windowed(tail, -1, 0)
    assert kvc.fp16_output_errors(out[2:].double().cpu().numpy(), ref)[2] <= 0


def test_rows_beyond_qmax_and_padding_stay():
    case = kvc.make_case([700, 300, 40], [4, 0, 3], seed=7)
    check(case, 100, 4, True, 4, qmax=2, lse=True)


def test_streams_and_a_captured_graph():
    cases = [kvc.make_case([2000 + 100 * i, 37], [2, 2], seed=i) for i in range(2)]
    window, sinks = 300, 20
    devs = [c.to("cuda") for c in cases]
    outs = [torch.zeros((4, 24, 256), dtype=torch.float16, device="cuda") for _ in cases]
    bufs = [kvc.partial_buffers(4, 24, 8, "cuda") for _ in cases]

    def call(i):
        d = devs[i]
        pth_dec.decode(d.q, d.cache.key_cache, d.cache.value_cache, d.cache.k_scale, d.cache.v_scale, d.block_table, d.seq_lens,
                       d.query_start_loc, outs[i], d.scale, *bufs[i], 2, 2, 8, window=window, sinks=sinks)

    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                call(i)
    torch.cuda.synchronize()
    refs = [window_oracle.windowed(c, window, sinks)[0] for c in cases]
    for o, r in zip(outs, refs):
        assert kvc.fp16_output_errors(o.double().cpu().numpy(), r)[2] <= 0
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(0)
    for lens in ([2002, 39], [400, 39], [30, 2], [2002, 39]):  # the lengths are read on the device
        devs[0].seq_lens.copy_(torch.tensor(lens, dtype=torch.int32))
        outs[0].zero_()
        graph.replay()
        torch.cuda.synchronize()
        got = outs[0].clone()
        call(0)
        torch.cuda.synchronize()
        assert torch.equal(got, outs[0])
    assert kvc.fp16_output_errors(outs[0].double().cpu().numpy(), refs[0])[2] <= 0


def test_the_planned_split_counts():
    """The shim's counts for a windowed batch, which the sinks lengthen by a tile or two."""
    case = kvc.make_case([5000, 100, 9000, 30], [2] * 4, seed=11)
    batch = (64, 1000 + 37, 4, 4, torch.device("cuda"), case.seq_lens, 2, 24)
    n = vllm_shim.launched_splits(vllm_shim.decode_splits(*batch), *batch)
    check(case, 1000, 37, True, n, nseg=64)
