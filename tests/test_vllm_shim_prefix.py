"""The shim's routing of decode batches with a common prefix, on the CPU with stand-in operators."""
import pytest
import torch

from mi50_vllm_lab_amd import vllm_shim as shim


class Ops:
    def __init__(self):
        self.calls = []

    def supported_layout(self, *a):
        return True

    def decode(self, q, kc, vc, ks, vs, bt, sl, qsl, out, scale, po, pm, pl, num_seqs, qmax, nsplit, window=-1, causal=True):
        self.calls.append(("decode", num_seqs, window))

    def decode_shared(self, q, kc, vc, ks, vs, bt, sl, qsl, out, scale, po, pm, pl, num_seqs, qmax, prefix):
        self.calls.append(("shared", num_seqs, qmax, prefix, q.shape[0]))


def run(monkeypatch, prefix, seqs=40, nseg=64, blocks=600, qlen=1, capturing=False, **kw):
    ops = Ops()
    monkeypatch.setattr(shim, "load_pth_dec", lambda: ops)
    monkeypatch.setattr(shim, "load_pth_fa", lambda: None)
    monkeypatch.setattr(shim, "_capturing", lambda d: capturing)
    a = shim.Gfx950Int8Attention(num_heads=24, num_kv_heads=4, head_size=256, scale=0.0625, kv_quant_int8_per_token_head=True,
                                 is_rocm=True, is_decoder=True, **kw)
    T, qsl = seqs * qlen, list(range(0, seqs * qlen + 1, qlen))
    part = torch.empty((1, 1, 1)).expand(T, 24, nseg)
    m = shim.AttnMeta(query_start_loc=torch.tensor(qsl, dtype=torch.int32), query_start_loc_cpu=qsl,
                      seq_lens=torch.full((seqs,), 9000, dtype=torch.int32), block_table=torch.zeros((seqs, blocks), dtype=torch.int32),
                      max_seq_len=9000, softmax_segm_output=part, softmax_segm_max=part, softmax_segm_expsum=part,
                      common_prefix_len=prefix)
    q = torch.zeros((T, 24, 256))
    kc = torch.zeros((1, 16, 4, 260), dtype=torch.int8)
    assert a.route(q, kc, kc, None, None, m, torch.zeros_like(q), qlen, T, lambda *x: None)
    return ops.calls[-1]


def test_a_long_common_prefix_is_read_once(monkeypatch):
    assert run(monkeypatch, 8192) == ("shared", 40, 1, 8192, 40)
    assert run(monkeypatch, 8192, qlen=4) == ("shared", 40, 4, 8192, 160)
    assert run(monkeypatch, 20000) == ("shared", 40, 1, 9600, 40)            # no further than the block table reaches


def test_the_bytes_spared_decide(monkeypatch):
    least = -(-shim.PTH_SHARED_MIN_BYTES // (39 * 4 * 520))
    assert run(monkeypatch, least)[0] == "shared" and run(monkeypatch, least - 1)[0] == "decode"
    assert run(monkeypatch, 9000, seqs=1)[0] == "decode" and run(monkeypatch, 0)[0] == "decode"


@pytest.mark.parametrize("kw", [dict(sliding_window=(2047, -1)), dict(nseg=3), dict(capturing=True)])
def test_what_keeps_the_decode(monkeypatch, kw):
    assert run(monkeypatch, 8192, **kw)[0] == "decode"


def test_metadata_without_the_field(monkeypatch):
    class Meta:
        pass
    assert shim.shared_prefix(Meta(), -1, 4, 40, 16, 600, 64) == 0
