"""evict against a plain selection on the CPU, exactly: the kept keys (ties to the lowest), their weights, lengths and rows, with
weights that tie, are zero, negative, infinite or NaN, sequences below, at and above the budget and empty ones, keep and recent at
their ends, long rows, block sizes 1, 16 and 1,584, both layouts, strided weights; nothing else in the cache changes; streams and a
captured graph.
"""
import math

import pytest
import torch

import workload as kvc
from mi50_vllm_lab_amd import pth_dec

pytestmark = pytest.mark.gpu


def order(x):
    return math.inf if math.isnan(x) else x


def chosen(w, n, keep, recent):
    """Keys of one sequence and kv head that stay (w: list of weights). NaN is the largest, as +inf but above it."""
    if n <= keep:
        return list(range(n))
    old = n - recent
    by = sorted(range(old), key=lambda t: (not math.isnan(w[t]), -order(w[t]) if not math.isnan(w[t]) else 0.0, t))
    return sorted(by[:keep - recent] + list(range(old, n)))


def batch(lens, hkv, bs, keep, layout, seed):
    g = torch.Generator().manual_seed(seed)
    per = [-(-n // bs) for n in lens]
    fresh = -(-keep // bs)
    blocks = sum(per) + fresh * len(lens) + 2
    c = kvc.allocate_cache(blocks, bs, hkv, layout)
    c.kv.copy_(torch.randint(-128, 128, c.kv.shape, dtype=torch.int8, generator=g))
    perm = torch.randperm(blocks, generator=g).to(torch.int32)
    bt = torch.full((len(lens), max(per + [1])), 0, dtype=torch.int32)
    at = 0
    for b, n in enumerate(per):
        bt[b, :n] = perm[at:at + n]
        at += n
    nbt = perm[at:at + fresh * len(lens)].view(len(lens), fresh)
    return c, bt, nbt


def run(c, bt, nbt, lens, w, keep, recent, cols=None, num=None):
    n, hkv = len(lens), c.num_kv_heads
    d = kvc.clone_cache(c, "cuda")
    lens_d = torch.tensor(lens, dtype=torch.int32, device="cuda")
    new_lens = torch.full((n,), 99, dtype=torch.int32, device="cuda")
    new_w = torch.full((n, hkv, cols or keep), 99.0, device="cuda")
    kept = torch.full((n, hkv, keep), 99, dtype=torch.int32, device="cuda")
    pth_dec.evict(w.cuda() if not w.is_cuda else w, d.key_cache, d.value_cache, d.k_scale, d.v_scale, bt.cuda(), lens_d, nbt.cuda(),
                  new_lens, new_w, kept, n if num is None else num, keep, recent)
    torch.cuda.synchronize()
    return d, new_lens.cpu(), new_w.cpu(), kept.cpu()


def check(c, bt, nbt, lens, w, keep, recent, got, limit=None):
    d, new_lens, new_w, kept = got
    bs, want = c.block_size, kvc.clone_cache(c)
    for b, length in enumerate(lens):
        n = max(0, min(length, w.shape[2] if limit is None else limit))
        m = min(n, keep)
        assert int(new_lens[b]) == m
        for h in range(c.num_kv_heads):
            mine = w[b, h, :n].tolist()
            stay = chosen(mine, n, keep, recent)
            assert kept[b, h].tolist() == stay + [-1] * (keep - m), (b, h)
            x = w[b, h, stay] if m else w[b, h, :0]
            assert torch.equal(new_w[b, h, :m].view(torch.int32), x.contiguous().view(torch.int32))
            assert not bool(new_w[b, h, m:].any())
            t, j = torch.tensor(stay, dtype=torch.long), torch.arange(m)
            want.kv[nbt[b].long()[j // bs], h, j % bs] = c.kv[bt[b].long()[t // bs], h, t % bs]
    assert torch.equal(d.kv.cpu(), want.kv)     # the rows, and nothing else


def weights(n, hkv, cols, kind, seed):
    g = torch.Generator().manual_seed(seed)
    w = torch.randn((n, hkv, cols), generator=g)
    if kind == "sums":
        w = (2 * w).exp()
        w[torch.rand(w.shape, generator=g) < 0.3] = 0.0
    elif kind == "ties":
        w = torch.randint(0, 4, w.shape, generator=g).float() - 1.0
        w[torch.rand(w.shape, generator=g) < 0.2] = -0.0
    elif kind == "same":
        w = torch.full_like(w, 0.25)
    elif kind == "odd":
        r = torch.rand(w.shape, generator=g)
        w[r < 0.05], w[(r > 0.1) & (r < 0.15)], w[(r > 0.2) & (r < 0.25)] = math.nan, math.inf, -math.inf
        w[(r > 0.3) & (r < 0.35)] = 1e-42
        w[(r > 0.4) & (r < 0.45)] = -math.nan
    return w


@pytest.mark.parametrize("kind", ["sums", "ties", "same", "odd", "normal"])
@pytest.mark.parametrize("lens,hkv,bs,keep,recent,layout", [
    ([100, 40, 41, 39, 0, 1], 2, 16, 40, 8, "HND"),
    ([3000, 1025, 1024, 1], 4, 16, 1000, 100, "NHD"),
    ([70, 33], 3, 1, 1, 0, "HND"),                      # one key stays, by its weight
    ([70, 33], 1, 1584, 1, 1, "HND"),                   # one key stays, the last
    ([513, 700], 2, 48, 64, 64, "NHD"),                 # only recent keys
    ([513, 700], 2, 48, 64, 0, "HND"),                  # no recent keys
    ([900, 901], 2, 16, 900, 7, "HND"),                 # one key too many
    ([17001], 1, 1584, 5000, 300, "HND"),
])
def test_against_a_plain_selection(lens, hkv, bs, keep, recent, layout, kind):
    c, bt, nbt = batch(lens, hkv, bs, keep, layout, seed=sum(lens))
    w = weights(len(lens), hkv, max(lens) + 3, kind, seed=keep)
    check(c, bt, nbt, lens, w, keep, recent, run(c, bt, nbt, lens, w, keep, recent, cols=keep + 5))


def test_long_rows():
    lens = [130001]
    c, bt, nbt = batch(lens, 2, 16, 3001, "HND", seed=2)
    w = weights(1, 2, 130001, "sums", seed=3)
    check(c, bt, nbt, lens, w, 3001, 64, run(c, bt, nbt, lens, w, 3001, 64))


def test_lengths_past_the_weights_or_the_table_are_cut():
    c, bt, nbt = batch([200, 90], 2, 16, 50, "HND", seed=6)
    w = weights(2, 2, 130, "sums", seed=7)
    check(c, bt, nbt, [200, 90], w, 50, 5, run(c, bt, nbt, [200, 90], w, 50, 5), limit=130)
    w = weights(2, 2, 400, "sums", seed=8)
    limit = bt.shape[1] * 16
    check(c, bt, nbt, [300, 90], w, 50, 5, run(c, bt, nbt, [300, 90], w, 50, 5), limit=limit)
    check(c, bt, nbt, [-3, 90], w, 50, 5, run(c, bt, nbt, [-3, 90], w, 50, 5), limit=limit)


def test_strided_weights_and_rows_behind_the_batch():
    lens = [300, 120]
    c, bt, nbt = batch(lens, 4, 16, 64, "HND", seed=9)
    w = weights(2, 4, 310, "sums", seed=9)
    big = torch.full((2, 9, 340), 1e9, device="cuda")
    view = big[:, 1::2, 7:317]
    view.copy_(w)
    check(c, bt, nbt, lens, w, 64, 10, run(c, bt, nbt, lens, view, 64, 10))
    d, new_lens, new_w, kept = run(c, bt, nbt, lens, w, 64, 10, num=1)
    assert int(new_lens[1]) == 99 and bool((new_w[1] == 99).all()) and bool((kept[1] == 99).all())
    assert torch.equal(d.kv[nbt[1].long().cuda()].cpu(), c.kv[nbt[1].long()])


def test_shared_blocks_stay():
    # two sequences on the same first blocks: each is cut by its own weights, the blocks stay for others
    c, bt, nbt = batch([160, 160], 2, 16, 48, "HND", seed=10)
    bt[1, :6] = bt[0, :6]
    w = weights(2, 2, 160, "sums", seed=10)
    check(c, bt, nbt, [160, 160], w, 48, 4, run(c, bt, nbt, [160, 160], w, 48, 4))


def test_streams_and_graph():
    lens = [500, 200, 1200]  # (the tables hold blocks for these; the replays take fewer keys of the second)
    c, bt, nbt = batch(lens, 4, 16, 100, "HND", seed=11)
    d = kvc.clone_cache(c, "cuda")
    w = weights(3, 4, 1200, "sums", seed=11).cuda()
    lens_d = torch.tensor(lens, dtype=torch.int32, device="cuda")
    new_lens, new_w = torch.zeros_like(lens_d), torch.zeros((3, 4, 100), device="cuda")
    kept = torch.zeros((3, 4, 100), dtype=torch.int32, device="cuda")
    a = (w, d.key_cache, d.value_cache, d.k_scale, d.v_scale, bt.cuda(), lens_d, nbt.cuda(), new_lens, new_w, kept, 3, 100, 10)

    def outputs():
        torch.cuda.synchronize()
        got = [x.clone() for x in (new_lens, new_w, kept, d.kv)]
        for x in (new_lens, new_w, kept):
            x.zero_()
        d.kv.copy_(c.kv)
        torch.cuda.synchronize()
        return got

    pth_dec.evict(*a)
    want = outputs()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        pth_dec.evict(*a)
    assert all(torch.equal(x, y) for x, y in zip(outputs(), want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        pth_dec.evict(*a)
    for step in range(3):
        w.copy_(weights(3, 4, 1200, "ties" if step == 1 else "sums", seed=20 + step))
        lens_d[1] = 80 + 60 * step
        graph.replay()
        got = outputs()
        pth_dec.evict(*a)
        assert all(torch.equal(x, y) for x, y in zip(got, outputs())), step
