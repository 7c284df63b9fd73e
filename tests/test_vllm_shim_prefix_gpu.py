"""A decode batch with a common prefix through the shim on the GPU: the rows are decode_shared's, and agree with decode's."""
import pytest
import torch

import workload as kvc
from mi50_vllm_lab_amd import vllm_shim as shim

pytestmark = pytest.mark.gpu


def test_common_prefix_through_the_shim(monkeypatch):
    shim.reset_loaders()
    prefix, n = 4096, 20                                                     # 19 x 4,096 x 4 x 520 bytes: above the threshold
    assert shim.shared_prefix(shim.AttnMeta(None, None, None, None, common_prefix_len=prefix), -1, 4, n, 16, 512, 64) == prefix
    c = kvc.make_case([prefix + 3 * b for b in range(n)], [1] * n, num_q_heads=24, num_kv_heads=4, block_size=16, seed=9)
    c.block_table[1:, :prefix // 16] = c.block_table[0, :prefix // 16]
    d = c.to("cuda")
    impl = shim.Gfx950Int8Attention(num_heads=24, num_kv_heads=4, head_size=256, scale=c.scale, kv_quant_int8_per_token_head=True,
                                    is_rocm=True, is_decoder=True)
    seen, real = [], impl.pth_dec.decode_shared
    monkeypatch.setattr(impl.pth_dec, "decode_shared", lambda *a: (seen.append(a[-1]), real(*a)))

    def run(common):
        po, pm, pl = kvc.partial_buffers(n, 24, 64, "cuda")
        meta = shim.AttnMeta(query_start_loc=d.query_start_loc, query_start_loc_cpu=c.query_start_loc.tolist(), seq_lens=d.seq_lens,
                             block_table=d.block_table, max_seq_len=max(c.seqs), softmax_segm_output=po, softmax_segm_max=pm,
                             softmax_segm_expsum=pl, seq_lens_cpu=c.seq_lens.tolist(), common_prefix_len=common)
        out = torch.full((n, 24, 256), float("nan"), dtype=torch.float16, device="cuda")
        assert impl.route(d.q, d.cache.key_cache, d.cache.value_cache, d.cache.k_scale, d.cache.v_scale, meta, out, 1, n,
                          lambda *a: pytest.fail("fell back"))
        torch.cuda.synchronize()
        return out.double()

    a, b = run(prefix), run(0)
    assert seen == [prefix]
    # each is the exact value rounded to fp16, give or take sums of 4,100 fp32 products and P' to 22 bits (hi + lo):
    # 2^-12 of the largest value covers both, and an fp16 step between them the rest
    assert ((a - b).abs() <= 2.0 ** -10 * b.abs() + 2.0 ** -12 * b.abs().max()).all(), float((a - b).abs().max())
