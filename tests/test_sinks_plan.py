"""The tiles of a windowed sequence with sinks (Seen in pd_decode.hip) restated on the CPU: for every small length, window and number of
sinks, each seen key lies in exactly one tile of the launch, every tile holds a seen key, and what is read in place of an unseen
key (a page given back) is a seen key of the same tile, also by 16-key blocks. And what the entry refuses.
"""
import ctypes

import pytest
import torch

import workload as kvc
from mi50_vllm_lab_amd import pth_dec

TILE = 32


class Seen:
    def __init__(self, window, sinks, q_len, seq_len):
        self.lo, self.hi = max(0, seq_len - q_len - window + 1), seq_len
        self.sinks = min(sinks, self.hi)
        self.head = -(-self.sinks // TILE)
        self.gap = max(0, self.lo // TILE - self.head)

    def tiles(self):
        return (self.hi - 1) // TILE + 1 - self.gap

    def base(self, tile):
        return (tile if tile < self.head else tile + self.gap) * TILE

    def near(self, kb, k):
        if k < self.sinks:
            return k
        return min(max(k, self.lo), self.hi - 1) if self.lo < kb + TILE else self.sinks - 1

    def has(self, k):
        return (k >= self.lo or k < self.sinks) and 0 <= k < self.hi


@pytest.mark.parametrize("q_len", [1, 3, 8])
@pytest.mark.parametrize("sinks", [1, 4, 16, 31, 32, 33, 64, 70, 500])
def test_tiles_cover_what_is_seen(q_len, sinks):
    for seq_len in list(range(max(1, q_len), 140)) + [200, 255, 256, 257, 300]:
        for window in (1, 2, 15, 16, 17, 31, 32, 33, 64, 100, 400):
            s = Seen(window, sinks, q_len, seq_len)
            bases = [s.base(t) for t in range(s.tiles())]
            assert len(set(bases)) == len(bases) and all(b < seq_len for b in bases)
            covered = {k for b in bases for k in range(b, b + TILE)}
            assert all(k in covered for k in range(seq_len) if s.has(k))
            for b in bases + [s.base(s.tiles() + i) for i in range(3)]:  # (tiles past the last are addressed, not computed)
                real = b in bases
                for k in range(b, b + TILE):
                    n = s.near(b, k)
                    assert s.has(n) and (n == k if s.has(k) else True)
                    assert not real or b <= n < b + TILE
                for u in (0, 1):  # the first key of a 16-key block, rounded down to it: a block with a seen key
                    n = s.near(b, b + 16 * u) & ~15
                    assert any(s.has(k) for k in range(n, n + 16))
                    assert not real or n == b + 16 * u or not any(s.has(k) for k in range(b + 16 * u, b + 16 * u + 16))


def test_refusals():
    lib = pth_dec.load_library()
    case = kvc.make_case([37, 5], [3, 1], num_q_heads=12, num_kv_heads=2, block_size=16, seed=3)
    c = case.cache
    po, pm, pl = kvc.partial_buffers(4, 12, 8, "cpu")
    good = dict(q=case.q, kc=c.key_cache, vc=c.value_cache, ks=c.k_scale, vs=c.v_scale, bt=case.block_table, lens=case.seq_lens,
                qsl=case.query_start_loc, out=torch.zeros((4, 12, 256), dtype=torch.float16))
    parts = dict(po=po, pm=pm, pl=pl, lse=torch.zeros((4, 12)))
    numbers = dict(num_seqs=2, qmax=3, nsplit=4, window=16, sinks=4, causal=1)
    cases = [({n: None}, "null tensor descriptor") for n in list(good) + ["po", "pm", "pl"]] + [
        (dict(sinks=-1), "sinks must be"), (dict(sinks=1 << 31), "sinks must be"), (dict(window=1 << 31), "window must fit"),
        (dict(qmax=9), "[1, 48]"), (dict(nsplit=9), "nsplit must be"), (dict(lse=torch.zeros((3, 12))), "lse must be"),
        (dict(q=case.q.float()), "q must be fp16"), (dict(vc=c.key_cache), "KV cache views"),
    ]
    err = ctypes.create_string_buffer(256)

    def call(a):
        d = {n: None if a[n] is None else ctypes.byref(pth_dec.describe(a[n])) for n in list(good) + list(parts)}
        return lib.pth_dec_decode_sinks(*[d[n] for n in good], 0.1, *[d[n] for n in parts], *[a[n] for n in numbers], None, err, len(err))

    for change, msg in cases:
        assert call({**good, **parts, **numbers, **change}) == 1 and msg in err.value.decode(), (change, err.value)
    none = {**good, **parts, **numbers, "q": case.q[:0], "out": good["out"][:0], "lse": None}
    assert call(none) == 0
    with pytest.raises(RuntimeError):
        pth_dec.decode(case.q, c.key_cache, c.value_cache, c.k_scale, c.v_scale, case.block_table, case.seq_lens,
                       case.query_start_loc, good["out"], 0.1, po, pm, pl, 2, 3, 4, window=16, sinks=4)
