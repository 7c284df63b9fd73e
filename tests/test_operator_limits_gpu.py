"""The operators around a decode step at sizes beyond what one launch numbers, and on inputs at the edges of their contracts, on
the GPU.
"""
import pytest
import torch

import workload as kvc
from mi50_vllm_lab_amd import pth_dec, rotary

pytestmark = pytest.mark.gpu


def test_rotary_write_of_more_tokens_than_one_launch_takes():
    # 8.1 million tokens of 16 kv heads and one query head are 17.2 million workgroups; a launch has fewer than 2^24
    T, hq, hkv, rd = 8_100_001, 1, 16, 64
    g = torch.Generator(device="cuda").manual_seed(1)
    table = rotary.rotary_table(rd, 600, device="cuda")
    one = torch.randn((1, hq + 2 * hkv, 256), device="cuda", generator=g).half()
    x = one.expand(T, -1, -1)
    pos = torch.arange(T, device="cuda") % 600
    slots = torch.full((T,), -1, device="cuda")
    at = torch.tensor([0, 1, 4_000_000, 7_895_158, 7_895_159, 7_895_160, 7_895_161, T - 2, T - 1], device="cuda")
    slots[at] = torch.arange(len(at), device="cuda") * 3
    caches = [kvc.allocate_cache(2, 16, hkv, "HND", "cuda") for _ in range(2)]
    out = torch.empty((T, hq, 256), dtype=torch.float16, device="cuda")
    c = caches[0]
    pth_dec.rotary_cache_write(x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:], pos, table, c.key_cache, c.value_cache, c.k_scale,
                               c.v_scale, slots, query_out=out)
    # the 600 positions, in one launch
    small = torch.empty((600, hq, 256), dtype=torch.float16, device="cuda")
    c, n = caches[1], torch.full((600,), -1, device="cuda")
    y = one.expand(600, -1, -1)
    pth_dec.rotary_cache_write(y[:, :hq], y[:, hq:hq + hkv], y[:, hq + hkv:], pos[:600].clone(), table, c.key_cache, c.value_cache,
                               c.k_scale, c.v_scale, n, query_out=small)
    for t in range(0, T, 600_000):
        part = out[t:t + 600_000]
        assert torch.equal(part, small[pos[t:t + 600_000]]), t
    z = one.expand(len(at), -1, -1)
    pth_dec.rotary_cache_write(z[:, :hq], z[:, hq:hq + hkv], z[:, hq + hkv:], pos[at], table, c.key_cache, c.value_cache, c.k_scale,
                               c.v_scale, slots[at], query_out=torch.empty((len(at), hq, 256), dtype=torch.float16, device="cuda"))
    assert torch.equal(caches[0].kv, caches[1].kv)


def test_evict_with_the_largest_budget():
    # a short sequence; behind it 2^28 places to clear, a workgroup per 32 of them
    keep, bs, n = 1 << 28, 1584, 100
    c = kvc.allocate_cache(3, bs, 1, "HND", "cuda")
    c.kv.random_(-128, 128, generator=torch.Generator(device="cuda").manual_seed(2))
    before = c.kv.clone()
    old, new = torch.tensor([[0]], dtype=torch.int32, device="cuda"), torch.full((1, -(-keep // bs)), 2, dtype=torch.int32, device="cuda")
    lens, new_lens = torch.tensor([n], dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    w = torch.rand((1, 1, 200), device="cuda")
    new_w, kept = torch.full((1, 1, keep), 9.0, device="cuda"), torch.full((1, 1, keep), 9, dtype=torch.int32, device="cuda")
    pth_dec.evict(w, c.key_cache, c.value_cache, c.k_scale, c.v_scale, old, lens, new, new_lens, new_w, kept, 1, keep, 5)
    torch.cuda.synchronize()
    assert new_lens.tolist() == [n] and kept[0, 0, :n].tolist() == list(range(n)) and torch.equal(new_w[0, 0, :n], w[0, 0, :n])
    assert int(kept[0, 0, n:].max()) == -1 and int(kept[0, 0, n:].min()) == -1 and not bool(new_w[0, 0, n:].any())
    assert torch.equal(c.kv[2, 0, :n], before[0, 0, :n]) and torch.equal(c.kv[:2], before[:2]) and torch.equal(c.kv[2, 0, n:], before[2, 0, n:])


def test_key_weights_of_rows_without_a_sum_where_scores_are_not_finite():
    # e^(score - lse) of a row with lse -inf is no weight, whatever its scores are: with infinite or NaN key scales too
    case = kvc.make_case([50, 20], [2, 1], num_q_heads=12, num_kv_heads=2, block_size=16, seed=8)
    d = case.to("cuda")
    page = case.block_table[0].long()
    d.cache.k_scale[int(page[0]), 3] = float("inf")
    d.cache.k_scale[int(page[1]), 2] = float("nan")
    d.cache.k_scale[int(page[2]), 5] = float("-inf")
    lse = torch.zeros((3, 12), device="cuda")
    lse[:2] = float("-inf")
    w = torch.rand((2, 2, 60), device="cuda")
    before = w.clone()
    pth_dec.key_weights(d.q, d.cache.key_cache, d.cache.value_cache, d.cache.k_scale, d.cache.v_scale, d.block_table, d.seq_lens,
                        d.query_start_loc, lse, w, d.scale, 2, 2)
    assert torch.equal(w[0], before[0])
    assert bool(torch.isfinite(w[1]).all()) and bool((w[1, :, :21] > before[1, :, :21]).all())


def test_outputs_beside_the_inputs_in_one_buffer():
    T, hq, hkv = 37, 24, 4
    g = torch.Generator().manual_seed(3)
    buf = torch.randn((T, 2 * hq + 2 * hkv, 256), generator=g).cuda().bfloat16()
    before = buf.clone()
    pos, table = torch.arange(T, device="cuda"), rotary.rotary_table(128, 64, device="cuda")
    caches = [kvc.allocate_cache(4, 16, hkv, "HND", "cuda") for _ in range(2)]
    want = torch.empty((T, hq, 256), dtype=torch.bfloat16, device="cuda")
    for x, c, out in ((before, caches[0], want), (buf, caches[1], buf[:, hq:2 * hq])):
        pth_dec.rotary_cache_write(x[:, :hq], x[:, 2 * hq:2 * hq + hkv], x[:, 2 * hq + hkv:], pos, table, c.key_cache, c.value_cache,
                                   c.k_scale, c.v_scale, pos, query_out=out)
    assert torch.equal(buf[:, hq:2 * hq], want) and torch.equal(buf[:, :hq], before[:, :hq])
    assert torch.equal(buf[:, 2 * hq:], before[:, 2 * hq:]) and torch.equal(caches[0].kv, caches[1].kv)
    # sums and kept sums as columns of one tensor
    c = kvc.allocate_cache(40, 16, 2, "HND", "cuda")
    lens = torch.tensor([200, 90], dtype=torch.int32, device="cuda")
    bt = torch.arange(26, dtype=torch.int32, device="cuda").view(2, 13)
    nbt = torch.arange(26, 34, dtype=torch.int32, device="cuda").view(2, 4)
    sums = torch.rand((2, 2, 264), generator=g).cuda()
    outs = []
    for w, nw in ((sums[..., :200].clone(), torch.empty((2, 2, 64), device="cuda")), (sums[..., :200], sums[..., 200:])):
        nl, kept = torch.zeros_like(lens), torch.zeros((2, 2, 64), dtype=torch.int32, device="cuda")
        pth_dec.evict(w, c.key_cache, c.value_cache, c.k_scale, c.v_scale, bt, lens, nbt, nl, nw, kept, 2, 64, 8)
        outs.append((nl, nw.clone(), kept))
    assert all(torch.equal(x, y) for x, y in zip(*outs))
