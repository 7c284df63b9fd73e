"""Keys whose scales are not finite (a token whose values overflowed), against float64: rows that do not see such a key, because it comes
after them or has left their window, are what they are without it, also where other rows of the same key tile see it; rows that do are
not finite, whichever split it lies in. decode with sinks (split, unsplit, dealt) and forward_window (narrow and wide workgroups,
split and not, both numerics, 16-key row blocks or not).
"""
import pytest
import torch

import window_oracle
import workload as kvc
from mi50_vllm_lab_amd import pth_dec

pytestmark = pytest.mark.gpu


def poison(case, keys, what):
    """what: the scale, "k" or "v", and its value. keys: a key of each sequence."""
    scale = case.cache.k_scale if what[0] == "k" else case.cache.v_scale
    for b, k in enumerate(keys):
        scale[int(case.block_table[b, k // case.cache.block_size]), k % case.cache.block_size] = what[1]


def sees(case, keys, window, sinks, causal=True):
    """[T]: rows that see their sequence's key."""
    rows = []
    for seq, ql, k in zip(case.seqs, case.qlens, keys):
        for p in range(seq - ql, seq):
            rows.append((k <= p or not causal) and (p - k < window or k < sinks))
    return torch.tensor(rows)


def check(out, ref, bad):
    out = out.double().cpu()
    assert 0 < int(bad.sum()) < bad.numel()
    good = (~bad).numpy()
    assert bool(torch.isfinite(out[~bad]).all())
    assert kvc.fp16_output_errors(out.numpy()[good], ref[good])[2] <= 0
    assert not bool(torch.isfinite(out[bad]).any())


VALUES = [("v", float("nan")), ("v", float("inf")), ("k", float("nan"))]


@pytest.mark.parametrize("what", VALUES)
@pytest.mark.parametrize("place", ["last", "first"])
@pytest.mark.parametrize("n,nsplit,bs,g", [(3, 1, 16, 6), (3, 4, 16, 6), (3, 3, 8, 6), (11, 8, 16, 6), (2, 2, 16, 12)])
def test_decode(n, nsplit, bs, g, place, what):
    window, sinks = 64, 5
    print(f"decode: {n} sequences, {nsplit} splits, blocks of {bs}, {g} rows, {place} key, {what}", flush=True)
    case = kvc.make_case([200 + 37 * i for i in range(n)], [4] * n, num_q_heads=4 * g, num_kv_heads=4, block_size=bs, seed=n + nsplit)
    ref, _, _ = window_oracle.windowed(case, window, sinks)
    # the last token, which the earlier rows do not see, or what only the first row still sees
    keys = [s - 1 if place == "last" else s - 4 - window + 1 for s in case.seqs]
    poison(case, keys, what)
    d = case.to("cuda")
    out = torch.full((4 * n, 4 * g, 256), 7.0, dtype=torch.float16, device="cuda")
    pth_dec.decode(d.q, d.cache.key_cache, d.cache.value_cache, d.cache.k_scale, d.cache.v_scale, d.block_table, d.seq_lens,
                   d.query_start_loc, out, d.scale, *kvc.partial_buffers(4 * n, 4 * g, 16, "cuda"), n, 4, nsplit, window=window, sinks=sinks)
    torch.cuda.synchronize()
    check(out, ref, sees(case, keys, window, sinks))


@pytest.mark.parametrize("what", VALUES)
@pytest.mark.parametrize("exact", [False, True])
@pytest.mark.parametrize("ctx,new,key,nsplit,bs", [
    (300, 200, 350, 1, 16),     # of the chunk: rows before it, and rows that it has left
    (300, 200, 250, 1, 16),     # behind the chunk
    (300, 200, 350, 3, 16),
    (300, 200, 359, 2, 24),
    (300, 200, 350, 1, 8),
    (100, 2100, 1500, 1, 16),   # wide workgroups
    (100, 2100, 1500, 2, 16),
])
def test_forward_window(ctx, new, key, nsplit, bs, exact, what):
    window, sinks = 100, 5
    print(f"forward_window: {new} tokens behind {ctx}, key {key}, {nsplit} splits, blocks of {bs}, exact {exact}, {what}", flush=True)
    case = kvc.make_case([ctx], [new], block_size=bs, seed=new)
    ref, _, _ = window_oracle.windowed(case, window, sinks)
    poison(case, [key], what)
    d = case.to("cuda")
    out = torch.full((new, 24, 256), 7.0, dtype=torch.float16, device="cuda")
    pth_dec.forward_window(d.q, d.cache.key_cache, d.cache.value_cache, d.block_table, d.seq_lens, d.scale, d.query_start_loc, out, window,
                           sinks=sinks, nsplit=nsplit, exact=exact)
    torch.cuda.synchronize()
    check(out, ref, sees(case, [key], window, sinks))


@pytest.mark.parametrize("what", VALUES)
@pytest.mark.parametrize("nsplit", [1, 2, 8])
def test_a_key_alone_in_its_split(nsplit, what):
    """The last key of 225, a tile of its own: the merge does not take its rows' part for one that saw no key."""
    print(f"alone: {nsplit} splits, {what}", flush=True)
    case = kvc.make_case([224, 96], [1, 1], seed=nsplit)
    ref, _, _ = window_oracle.windowed(case, 4000, 4)
    poison(case, [224], what)                             # the other sequence has none
    bad = torch.tensor([True, False])
    d = case.to("cuda")
    for exact in (None, False, True):
        out = torch.full((2, 24, 256), 7.0, dtype=torch.float16, device="cuda")
        args = (d.block_table, d.seq_lens)
        if exact is None:
            pth_dec.decode(d.q, d.cache.key_cache, d.cache.value_cache, d.cache.k_scale, d.cache.v_scale, *args, d.query_start_loc, out, d.scale,
                           *kvc.partial_buffers(2, 24, 16, "cuda"), 2, 1, nsplit, window=4000, sinks=4)
        else:
            pth_dec.forward_window(d.q, d.cache.key_cache, d.cache.value_cache, *args, d.scale, d.query_start_loc, out, 4000, sinks=4,
                                   nsplit=nsplit, exact=exact)
        torch.cuda.synchronize()
        check(out, ref, bad)
