"""The operators of a bounded conversation on pages more than 2^35 bytes into a cache (offsets beyond 32 bits in bytes, and in the
8-byte units of the prefill's LDS table): a small batch's pages moved to the far end of a 35 GB cache."""
import pytest
import torch

import window_oracle
import workload as kvc
from mi50_vllm_lab_amd import pth_dec, rotary

pytestmark = pytest.mark.gpu


def test_far_pages():
    case = kvc.make_case([700, 90], [40, 3], seed=1)
    pages = 1_050_000
    kv = torch.empty((pages, 4, 16, 520), dtype=torch.int8, device="cuda")
    c = kvc.cache_views(kv, "HND")
    assert (pages - 100) * kv.stride(0) > 1 << 35
    n = case.cache.num_blocks
    first = pages - n
    kv[first:] = case.cache.kv.cuda()
    d = case.to("cuda")
    bt = d.block_table + first
    window, sinks = 200, 9
    ref, _, _ = window_oracle.windowed(case, window, sinks)
    out = torch.zeros((43, 24, 256), dtype=torch.float16, device="cuda")
    for nsplit in (1, 3):
        out.zero_()
        pth_dec.forward_window(d.q, c.key_cache, c.value_cache, bt, d.seq_lens, case.scale, d.query_start_loc, out, window, sinks=sinks,
                               nsplit=nsplit)
        assert kvc.fp16_output_errors(out.double().cpu().numpy(), ref)[2] <= 0
    tail = kvc.make_case([700, 90], [4, 3], seed=1)
    kv[first:first + tail.cache.num_blocks] = tail.cache.kv.cuda()
    t = tail.to("cuda")
    ref, _, _ = window_oracle.windowed(tail, window, sinks)
    out = torch.zeros((7, 24, 256), dtype=torch.float16, device="cuda")
    pth_dec.decode(t.q, c.key_cache, c.value_cache, c.k_scale, c.v_scale, t.block_table + first, t.seq_lens, t.query_start_loc, out, case.scale,
                   *kvc.partial_buffers(7, 24, 8, "cuda"), 2, 4, 8, window=window, sinks=sinks)
    assert kvc.fp16_output_errors(out.double().cpu().numpy(), ref)[2] <= 0
    # rows written to the last page, as to the first of a small cache
    x = torch.randn((16, 32, 256), device="cuda").half()
    w = torch.rand(256, device="cuda").half()
    table = rotary.rotary_table(64, 16, 1e4).cuda()
    pos = torch.arange(16, device="cuda")
    small = kvc.allocate_cache(1, 16, 4, "HND", "cuda")
    for cache, page in ((small, 0), (c, pages - 1)):
        pth_dec.norm_rotary_cache_write(x[:, :24], x[:, 24:28], x[:, 28:], w, w, pos, table, cache.key_cache, cache.value_cache, cache.k_scale,
                                        cache.v_scale, pos + 16 * page, query_out=torch.empty_like(x[:, :24]))
    assert torch.equal(kv[-1], small.kv[0])
    # a part-filled page forked, pages packed from the far end to the front and counted
    refs = torch.zeros(pages, dtype=torch.int32, device="cuda")
    refs[:pages - 5] = 1
    refs[pages - 1] = 1
    refs[3] = 0
    rows = torch.tensor([[pages - 1, -1]], dtype=torch.int32, device="cuda")
    lens, parents = torch.tensor([9], dtype=torch.int32, device="cuda"), torch.tensor([0, 0], dtype=torch.int32, device="cuda")
    new = torch.empty_like(refs), torch.empty((2, 2), dtype=torch.int32, device="cuda"), torch.empty(2, dtype=torch.int32, device="cuda")
    needed = torch.empty(1, dtype=torch.int32, device="cuda")
    pth_dec.fork_pages([c], refs, rows, lens, parents, *new, needed, grow=20)
    assert new[1].tolist() == [[pages - 1, 3], [pages - 5, pages - 4]] and int(needed) == 3
    assert torch.equal(kv[pages - 5, :, :9], kv[pages - 1, :, :9])
    places, used = torch.empty_like(refs), torch.empty(1, dtype=torch.int32, device="cuda")
    packed = torch.empty_like(refs), torch.empty_like(rows)
    pth_dec.compact_pages([c], refs, rows, *packed, places, used)
    assert int(used) == pages - 5 and packed[1].tolist() == [[3, -1]] and torch.equal(kv[3], small.kv[0])
