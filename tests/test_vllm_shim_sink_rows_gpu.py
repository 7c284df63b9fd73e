"""The shim's layers with sink_tokens on the GPU: turns of every length, fp16 and bf16 rows, with decode's buffers and without, in the
window form (W - 1, 0), against float64."""
import pytest
import torch

import window_oracle
import workload as kvc
from mi50_vllm_lab_amd import vllm_shim as shim

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("qlens,buffers", [([1, 2, 1], True), ([1, 2, 1], False), ([10], True), ([1, 5, 1], True), ([2, 10, 100], True),
                                           ([100, 1], True), ([3, 100], True), ([3, 100], False)])
def test_route(qlens, buffers, dtype):
    shim.reset_loaders()
    sinks = 37
    case = kvc.make_case([900, 40, 3000][:len(qlens)], qlens, seed=sum(qlens))
    case.q = case.q.to(dtype).half()  # (the values that both types hold)
    d = case.to("cuda")
    a = shim.Gfx950Int8Attention(num_heads=24, num_kv_heads=4, head_size=256, scale=case.scale, kv_quant_int8_per_token_head=True,
                                 is_rocm=True, is_decoder=True, sliding_window=(255, 0), sink_tokens=sinks)
    po, pm, pl = kvc.partial_buffers(case.num_tokens, 24, 64, "cuda") if buffers else (None, None, None)
    meta = shim.AttnMeta(query_start_loc=d.query_start_loc, query_start_loc_cpu=case.query_start_loc, seq_lens=d.seq_lens,
                         block_table=d.block_table, max_seq_len=max(case.seqs), softmax_segm_output=po, softmax_segm_max=pm,
                         softmax_segm_expsum=pl, seq_lens_cpu=case.seq_lens)
    out = torch.full((case.num_tokens + 3, 24, 256), 7.0, dtype=dtype, device="cuda")
    q = torch.cat([d.q.to(dtype), torch.zeros((3, 24, 256), dtype=dtype, device="cuda")])
    c = d.cache
    assert a.route(q, c.key_cache, c.value_cache, c.k_scale, c.v_scale, meta, out, max(qlens), case.num_tokens,
                   lambda *x: pytest.fail("left to the caller"))
    torch.cuda.synchronize()
    assert bool((out[case.num_tokens:] == 7.0).all())
    got = out[:case.num_tokens].double().cpu().numpy()
    ref, _, _ = window_oracle.windowed(case, 256, sinks)
    if dtype == torch.float16:
        assert kvc.fp16_output_errors(got, ref)[2] <= 0
    else:
        # 2e-3 before the rounding to fp16, that rounding, and half a step of bf16: 2^-11 and 2^-8 relative to the value and its error
        bound = 2e-3 + (2.0 ** -11 + 2.0 ** -8) * (abs(ref) + 3e-3)
        assert bool((abs(got - ref) <= bound).all()), float((abs(got - ref) - bound).max())
