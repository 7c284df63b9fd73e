"""Which decode batches with a common prefix the shim sends to decode_shared, on the CPU: within what that takes, and where it was
measured faster than decode.
"""
import pytest
import torch

import workload as kvc
from mi50_vllm_lab_amd import pth_dec, vllm_shim as shim
from test_vllm_shim_prefix import run


class Meta:
    def __init__(self, n):
        self.common_prefix_len = n


def test_more_key_tiles_than_decode_shared_numbers_stay_with_decode():
    # tables of 2^18 blocks of 64 keys for 4,096 sequences and 4 kv heads: 2^32 key tiles
    assert shim.shared_prefix(Meta(8192), -1, 4, 4096, 64, 1 << 18, 64) == 0
    assert shim.shared_prefix(Meta(8192), -1, 4, 200, 64, 1 << 12, 64) == 8192
    assert shim.shared_prefix(Meta(8192), -1, 4, 40, 16, 1 << 31, 64) == 0


@pytest.mark.parametrize("num_seqs,hkv,bs,blocks", [(2, 2, 16, b) for b in (1 << 28, (1 << 29) - 8, 1 << 29, 1 << 30)] + [(500, 2, 16, 1 << 20), (500, 2, 16, 1 << 21),
                                                                                                                (500, 2, 16, (1 << 21) + (1 << 18))])
def test_the_limit_is_the_entry_s(num_seqs, hkv, bs, blocks):
    import ctypes
    c = kvc.make_case([37, 5], [3, 1], num_q_heads=12, num_kv_heads=hkv, block_size=bs, seed=3)
    d = [pth_dec.describe(x) for x in (c.q[:0], c.cache.key_cache, c.cache.value_cache, c.cache.k_scale, c.cache.v_scale, c.block_table,
                                       c.seq_lens, c.query_start_loc, torch.zeros((0, 12, 256), dtype=torch.float16))]
    d[5].sizes[0], d[5].sizes[1], d[6].sizes[0], d[7].sizes[0] = num_seqs, blocks, num_seqs, num_seqs + 1   # described, never read
    tail = [pth_dec.describe(x) for x in kvc.partial_buffers(4, 12, 4, "cpu")]
    rc = pth_dec.load_library().pth_dec_decode_shared(*map(ctypes.byref, d), ctypes.c_double(0.1), *map(ctypes.byref, tail), None, num_seqs, 3,
                                                      0, None, None, 0)
    assert rc in (0, 1) and (rc == 0) == shim.shared_tables_fit(num_seqs, hkv, blocks, bs)


# batches measured on an MI355X (sequences, query tokens each, shared keys, q and kv heads)
FASTER_SHARED = [(16, 1, 8192, 24, 4), (32, 1, 4096, 24, 4), (64, 1, 2048, 24, 4), (128, 1, 2048, 24, 4), (8, 1, 16384, 24, 4), (32, 2, 8192, 24, 4),
                 (32, 4, 8192, 24, 4), (64, 1, 4096, 12, 2), (512, 1, 1024, 24, 4)]
FASTER_DECODE = [(64, 4, 1024, 24, 4), (64, 4, 2048, 24, 4), (8, 2, 32768, 12, 2), (8, 4, 16384, 24, 4), (4, 1, 32768, 24, 4), (4, 2, 32768, 24, 4),
                 (16, 1, 2048, 24, 4), (64, 2, 1024, 24, 4)]


@pytest.mark.parametrize("seqs,ql,prefix,hq,hkv", FASTER_SHARED + FASTER_DECODE)
def test_the_faster_operator_takes_the_batch(seqs, ql, prefix, hq, hkv):
    got = shim.shared_prefix(Meta(prefix), -1, hkv, seqs, 16, 4096, 64, seqs * ql, hq)
    assert got == (prefix if (seqs, ql, prefix, hq, hkv) in FASTER_SHARED else 0)


def test_the_route_counts_the_batch_s_rows(monkeypatch):
    # 268 MB are spared either way; four tokens per sequence cost more than that gains
    assert run(monkeypatch, 2048, seqs=64)[0] == "shared" and run(monkeypatch, 2048, seqs=64, qlen=4)[0] == "decode"
