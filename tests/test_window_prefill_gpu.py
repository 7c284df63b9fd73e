"""forward_window on the GPU against float64: windows and sinks that overlap, touch, lie far apart or hold every key, chunks of one
token to several workgroups, fresh prompts and turns of long conversations, ragged batches with empty sequences, group sizes that no tile
divides, block sizes 1 to 1,584, pages that no row sees at a block of NaN, unsplit and split, both numerics, outlier rows; rows that
belong to no sequence, views with gaps, two streams and a captured graph; against forward_rows and decode where those take the call.

Tolerance: workload.fp16_output_errors, 2e-3 and 2e-4 before the output's rounding to fp16, as the prefill's tests have it.
"""
import random

import numpy as np
import pytest
import torch

import window_oracle
import workload as kvc
from mi50_vllm_lab_amd import pth_dec

pytestmark = pytest.mark.gpu


def run(case, bt, window, sinks, nsplit=None, exact=False):
    d = case.to("cuda")
    out = torch.full((case.num_tokens, case.num_q_heads, 256), 7.0, dtype=torch.float16, device="cuda")
    pth_dec.forward_window(d.q, d.cache.key_cache, d.cache.value_cache, bt.cuda(), d.seq_lens, case.scale, d.query_start_loc, out, window,
                           sinks=sinks, nsplit=nsplit, exact=exact)
    torch.cuda.synchronize()
    return out.cpu()


def check(case, window, sinks, forms=((None, False),)):
    bt, _ = window_oracle.freed(case, window, sinks)
    ref, _, written = window_oracle.windowed(case, window, sinks, True, bt)
    for nsplit, exact in forms:
        out = run(case, bt, window, sinks, nsplit, exact)
        assert bool((out[~written] == 7.0).all())
        _, _, worst, mean = kvc.fp16_output_errors(out.double().numpy()[written], ref[written])
        assert worst <= 0 and mean <= 2e-4, (nsplit, exact, worst, mean)


BOTH = ((1, False), (3, False), (1, True), (7, True))


@pytest.mark.parametrize("ctx,new,window,sinks,bs,layout,hq,hkv", [
    (1000, 64, 100, 4, 16, "HND", 24, 4),
    (1000, 43, 100, 33, 16, "NHD", 24, 4),       # one row more than a workgroup's
    (0, 300, 100, 4, 16, "HND", 24, 4),          # a fresh prompt
    (0, 1, 1, 0, 16, "HND", 24, 4),
    (0, 33, 1, 1, 16, "HND", 6, 6),              # each row sees itself and the first key
    (500, 100, 460, 37, 16, "HND", 24, 4),       # the window leaves the sinks inside the chunk
    (500, 100, 520, 70, 16, "HND", 12, 2),
    (500, 100, 4000, 16, 16, "HND", 24, 4),      # rows that see everything
    (500, 200, 64, 900, 16, "HND", 24, 4),       # more sinks than keys
    (100, 90, 30, 0, 16, "HND", 5, 1),           # no sinks; five heads
    (300, 70, 50, 40, 8, "HND", 7, 1),           # pages inside a 16-key block
    (300, 70, 50, 40, 1, "NHD", 24, 4),
    (900, 60, 200, 50, 24, "HND", 12, 2),
    (3000, 150, 700, 37, 1584, "NHD", 12, 2),
    (2500, 130, 2048, 4, 32, "HND", 24, 4),
    (200, 20, 90, 5, 16, "HND", 200, 1),         # few tokens to a workgroup
    (200, 9, 90, 5, 16, "HND", 256, 1),
    (99000, 8, 98500, 40, 16, "HND", 6, 1),      # more 16-key blocks than the LDS table holds, unsplit
    (150000, 5, 300, 20, 24, "NHD", 6, 1),       # more pages than it holds
])
def test_one_sequence(ctx, new, window, sinks, bs, layout, hq, hkv):
    case = kvc.make_case([ctx], [new], num_q_heads=hq, num_kv_heads=hkv, block_size=bs, layout=layout, seed=ctx + window + sinks)
    check(case, window, sinks, BOTH)


@pytest.mark.parametrize("seed", range(20))
def test_random_batches(seed):
    rng = random.Random(seed)
    hq, hkv = rng.choice([(24, 4), (12, 2), (6, 6), (5, 1), (16, 1)])
    n = rng.choice([1, 2, 5, 9, 70])
    most = 400 if n < 9 else 60
    qlens = [rng.choice([0, 1, rng.randint(1, most)]) for _ in range(n)]
    qlens[-1] = rng.randint(1, most)
    ctxs = [rng.choice([0, 1, rng.randint(0, 100), rng.randint(0, 2500 if n < 9 else 500)]) for _ in range(n)]
    case = kvc.make_case(ctxs, qlens, num_q_heads=hq, num_kv_heads=hkv, block_size=rng.choice([1, 8, 16, 16, 32, 48, 1584]),
                         layout=rng.choice(["HND", "NHD"]), seed=seed, q_noncontig=rng.random() < 0.3)
    check(case, rng.choice([1, 7, 100, 700, 2048]), rng.choice([0, 1, 4, 16, 37, 128, 1000]),
          ((None, False), (rng.choice([2, 5, 16, 64]), rng.random() < 0.5)))


def test_outlier_sinks_with_hi_and_lo_weights():
    case = kvc.make_case([1500, 300], [70, 50], seed=5)
    for b in range(2):
        kvc.write_tokens(case.cache, case.block_table[b], torch.arange(4), *kvc.quantize_per_token_head(torch.randn(4, 4, 256)),
                         *kvc.quantize_per_token_head(60 * torch.randn(4, 4, 256)))
    check(case, 512, 4, ((1, True), (4, True)))


@pytest.mark.parametrize("exact", [False, True])
def test_long_chunk_against_float64_of_some_rows(exact):
    """3,000 fresh tokens on top of 500 over a window of 1,500: wide workgroups (the shorter calls here run narrow ones), several
    rounds of them, interior tiles without masks."""
    window, sinks, ctx, new = 1500, 37, 500, 3000
    case = kvc.make_case([ctx], [new], seed=9)
    bt, _ = window_oracle.freed(case, window, sinks)
    out = run(case, bt, window, sinks, exact=exact).double().numpy()
    key = torch.arange(ctx + new)
    c = case.cache
    k, v = (x[bt[0].long()[key // 16], key % 16, :, :256].double() * s[bt[0].long()[key // 16], key % 16].double()[..., None]
            for x, s in ((c.key_cache, c.k_scale), (c.value_cache, c.v_scale)))
    for i in (0, 1, 41, 42, 43, 700, 1036, 1037, 1499, 2222, 2998, 2999):
        p = ctx + i
        see = (key <= p) & ((p - key < window) | (key < sinks))
        for h in range(24):
            x = torch.mv(k[see, h // 6], case.q[i, h].double()) * case.scale
            ref = torch.softmax(x, 0) @ v[see, h // 6]
            assert kvc.fp16_output_errors(out[i, h], ref.numpy())[2] <= 0, (i, h)


@pytest.mark.parametrize("lens,bs,layout,nsplit,exact", [
    ([2100, 700], 16, "HND", 1, False), ([1500, 900, 5, 800], 16, "NHD", 2, False), ([2500], 24, "HND", 1, True), ([2900], 1, "NHD", 2, True)])
def test_wide_workgroups(lens, bs, layout, nsplit, exact):
    """More rows than narrow workgroups take in a round, over a short window: every row against float64."""
    case = kvc.make_case([300, 0, 70, 41][:len(lens)], lens, block_size=bs, layout=layout, seed=bs + len(lens))
    check(case, 150, 21, ((nsplit, exact),))


def test_a_window_of_everything_is_the_prefill():
    case = kvc.make_case([700, 90], [130, 64], seed=2)
    d = case.to("cuda")
    outs = [torch.zeros((194, 24, 256), dtype=torch.float16, device="cuda") for _ in range(2)]
    assert pth_dec.forward_rows(d.q, d.cache.key_cache, d.cache.value_cache, d.block_table, d.seq_lens, d.scale, [0, 130, 194], outs[0], 830)
    pth_dec.forward_window(d.q, d.cache.key_cache, d.cache.value_cache, d.block_table, d.seq_lens, d.scale, d.query_start_loc, outs[1], 5000)
    # both within 2e-3 of float64 before their rounding
    assert float((outs[0].float() - outs[1].float()).abs().max()) <= 4e-3 + 2.0 ** -10


def test_single_tokens_are_the_decode():
    case = kvc.make_case([700, 90, 3000], [1, 4, 2], seed=3)
    check(case, 256, 20, BOTH)
    d = case.to("cuda")
    bufs = kvc.partial_buffers(7, 24, 4, "cuda")
    outs = [torch.zeros((7, 24, 256), dtype=torch.float16, device="cuda") for _ in range(2)]
    pth_dec.decode(d.q, d.cache.key_cache, d.cache.value_cache, d.cache.k_scale, d.cache.v_scale, d.block_table, d.seq_lens,
                   d.query_start_loc, outs[0], d.scale, *bufs, 3, 4, 4, window=256, sinks=20)
    pth_dec.forward_window(d.q, d.cache.key_cache, d.cache.value_cache, d.block_table, d.seq_lens, d.scale, d.query_start_loc, outs[1],
                           256, sinks=20)
    assert float((outs[0].float() - outs[1].float()).abs().max()) <= 4e-3 + 2.0 ** -10


@pytest.mark.parametrize("nsplit", [1, 4])
def test_rows_without_a_sequence_or_keys(nsplit):
    """Rows before, between and behind the sequences stay; rows before their sequence's first key become 0."""
    case = kvc.make_case([100, 40], [30, 50], seed=4)
    d = case.to("cuda")
    q = torch.randn((120, 24, 256), device="cuda").half()
    out = torch.full((120, 24, 256), 7.0, dtype=torch.float16, device="cuda")
    qsl = torch.tensor([5, 25, 25, 60, 90], dtype=torch.int32, device="cuda")   # 20, 0, 35 and 30 rows
    lens = torch.tensor([120, 50, 0, 10], dtype=torch.int32, device="cuda")     # the third has no keys, the last fewer than rows
    bt = torch.stack([d.block_table[i] for i in (0, 0, 1, 1)])
    pth_dec.forward_window(q, d.cache.key_cache, d.cache.value_cache, bt, lens, d.scale, qsl, out, 16, sinks=3, nsplit=nsplit)
    torch.cuda.synchronize()
    for a, b in ((0, 5), (25, 60), (90, 120)):
        assert bool((out[a:b] == 7.0).all())
    assert bool((out[60:80] == 0).all())  # positions -20 .. -1
    assert bool((out[5:25] != 7.0).any(-1).all()) and bool(out[80:90].isfinite().all())
    case2 = kvc.DecodeCase(torch.cat([q[5:25], q[80:90]]).cpu(), case.cache, torch.stack([case.block_table[0], case.block_table[1]]),
                           torch.tensor([120, 10], dtype=torch.int32), torch.tensor([0, 20, 30], dtype=torch.int32), [100, 0], [20, 10], 24,
                           case.scale)
    ref, _, _ = window_oracle.windowed(case2, 16, 3)
    got = torch.cat([out[5:25], out[80:90]]).double().cpu().numpy()
    assert kvc.fp16_output_errors(got, ref)[2] <= 0


def test_offsets_beyond_the_rows_are_left_out():
    """A last offset past the rows of q: the rows that there are."""
    case = kvc.make_case([100], [30], seed=6)
    d = case.to("cuda")
    outs = []
    for last in (30, 500):
        out = torch.zeros((30, 24, 256), dtype=torch.float16, device="cuda")
        pth_dec.forward_window(d.q, d.cache.key_cache, d.cache.value_cache, d.block_table, d.seq_lens, d.scale,
                               torch.tensor([0, last], dtype=torch.int32, device="cuda"), out, 64, sinks=2)
        outs.append(out)
    assert torch.equal(*outs)


@pytest.mark.parametrize("window", [1 << 30, (1 << 31) - 1])
def test_the_largest_windows(window):
    """Rows before their sequence's first key beside a window that no position less it fits 32 bits."""
    case = kvc.make_case([0, 50], [40, 30], seed=12)
    d = case.to("cuda")
    lens = torch.tensor([10, 80], dtype=torch.int32)
    for sinks in (0, 7, (1 << 31) - 1):
        out = torch.full((70, 24, 256), 7.0, dtype=torch.float16, device="cuda")
        pth_dec.forward_window(d.q, d.cache.key_cache, d.cache.value_cache, d.block_table, lens.cuda(), d.scale, d.query_start_loc, out, window,
                               sinks=sinks)
        assert bool((out[:30] == 0).all())
        tail = kvc.DecodeCase(case.q[30:], case.cache, case.block_table, lens, torch.tensor([0, 10, 40], dtype=torch.int32), [0, 50], [10, 30],
                              24, case.scale)
        ref, _, _ = window_oracle.windowed(tail, -1, 0)
        assert kvc.fp16_output_errors(out[30:].double().cpu().numpy(), ref)[2] <= 0


def test_no_tokens_and_views_with_gaps():
    case = kvc.make_case([200], [50], seed=8)
    d = case.to("cuda")
    empty = d.q[:0]
    pth_dec.forward_window(empty, d.cache.key_cache, d.cache.value_cache, d.block_table, d.seq_lens, d.scale, d.query_start_loc,
                           torch.empty_like(empty), 64)
    q = torch.randn((50, 30, 264), device="cuda").half()
    q[:, 3:27, :256] = d.q
    out = torch.full((50, 26, 260), 7.0, dtype=torch.float16, device="cuda")
    pth_dec.forward_window(q[:, 3:27, :256], d.cache.key_cache, d.cache.value_cache, d.block_table, d.seq_lens, d.scale, d.query_start_loc,
                           out[:, 1:25, :256], 64, sinks=5)
    ref, _, _ = window_oracle.windowed(case, 64, 5)
    assert kvc.fp16_output_errors(out[:, 1:25, :256].double().cpu().numpy(), ref)[2] <= 0
    assert bool((out[:, 0] == 7).all()) and bool((out[:, 25] == 7).all()) and bool((out[..., 256:] == 7).all())


@pytest.mark.parametrize("nsplit", [None, 3])
def test_streams_and_a_captured_graph(nsplit):
    cases = [kvc.make_case([900 + 100 * i, 37, 0], [100, 20, 44], seed=i) for i in range(2)]
    window, sinks = 300, 20
    devs = [c.to("cuda") for c in cases]
    outs = [torch.zeros((164, 24, 256), dtype=torch.float16, device="cuda") for _ in cases]

    def call(i):
        d = devs[i]
        pth_dec.forward_window(d.q, d.cache.key_cache, d.cache.value_cache, d.block_table, d.seq_lens, d.scale, d.query_start_loc, outs[i],
                               window, sinks=sinks, nsplit=nsplit)

    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                call(i)
    torch.cuda.synchronize()
    for c, o in zip(cases, outs):
        assert kvc.fp16_output_errors(o.double().cpu().numpy(), window_oracle.windowed(c, window, sinks)[0])[2] <= 0
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(0)
    # other batches of as many rows and sequences: the offsets and lengths are read on the device
    for qsl, lens in (([0, 100, 120, 164], [1000, 57, 44]), ([0, 10, 50, 164], [200, 50, 10]), ([0, 0, 164, 164], [5, 57, 0]),
                      ([0, 100, 120, 164], [1000, 57, 44])):
        devs[0].query_start_loc.copy_(torch.tensor(qsl, dtype=torch.int32))
        devs[0].seq_lens.copy_(torch.tensor(lens, dtype=torch.int32))
        outs[0].fill_(7)
        graph.replay()
        torch.cuda.synchronize()
        got = outs[0].clone()
        outs[0].fill_(7)
        call(0)
        torch.cuda.synchronize()
        assert torch.equal(got, outs[0])
    assert kvc.fp16_output_errors(outs[0].double().cpu().numpy(), window_oracle.windowed(cases[0], window, sinks)[0])[2] <= 0


def test_small_workspace_and_bad_splits_are_refused():
    case = kvc.make_case([100], [30], seed=6)
    d = case.to("cuda")
    out = torch.zeros((30, 24, 256), dtype=torch.float16, device="cuda")
    for nsplit in (-1, 65):
        with pytest.raises(RuntimeError, match="nsplit"):
            pth_dec.forward_window(d.q, d.cache.key_cache, d.cache.value_cache, d.block_table, d.seq_lens, d.scale, d.query_start_loc, out, 64,
                                   nsplit=nsplit)
