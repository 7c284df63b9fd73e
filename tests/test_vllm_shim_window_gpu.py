"""The shim's windowed layers on the GPU: a mixed batch (decoded rows, then chunks) with sinks through route(), against float64."""
import pytest
import torch

import window_oracle
import workload as kvc
from mi50_vllm_lab_amd import vllm_shim as shim

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("qlens,sinks", [([2, 1, 100, 64], 4), ([70], 0), ([1, 2, 1], 37)])
def test_route(qlens, sinks):
    shim.reset_loaders()
    ctxs = [900, 40, 3000, 10][:len(qlens)]
    case = kvc.make_case(ctxs, qlens, seed=sum(qlens))
    d = case.to("cuda")
    a = shim.Gfx950Int8Attention(num_heads=24, num_kv_heads=4, head_size=256, scale=case.scale, kv_quant_int8_per_token_head=True,
                                 is_rocm=True, is_decoder=True, sliding_window=(255, -1), sink_tokens=sinks)
    po, pm, pl = kvc.partial_buffers(case.num_tokens, 24, 64, "cuda")
    meta = shim.AttnMeta(query_start_loc=d.query_start_loc, query_start_loc_cpu=case.query_start_loc, seq_lens=d.seq_lens,
                         block_table=d.block_table, max_seq_len=max(case.seqs), softmax_segm_output=po, softmax_segm_max=pm,
                         softmax_segm_expsum=pl, seq_lens_cpu=case.seq_lens)
    out = torch.zeros((case.num_tokens, 24, 256), dtype=torch.float16, device="cuda")
    c = d.cache
    assert a.route(d.q, c.key_cache, c.value_cache, c.k_scale, c.v_scale, meta, out, max(qlens), case.num_tokens,
                   lambda *x: pytest.fail("left to the caller"))
    ref, _, _ = window_oracle.windowed(case, 256, sinks)
    assert kvc.fp16_output_errors(out.double().cpu().numpy(), ref)[2] <= 0
