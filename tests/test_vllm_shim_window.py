"""The shim's routing of windowed layers without a GPU: their prefill goes to forward_window, rows before it to decode or to the
caller, the sinks go to both operators, and what the operator does not take stays with the caller.
"""
import pytest
import torch

from mi50_vllm_lab_amd import vllm_shim as shim


class Ops:
    def __init__(self):
        self.calls = []
        self.layout = True

    def supported_layout(self, *views):
        return self.layout

    def decode(self, q, kc, vc, ks, vs, bt, sl, qsl, out, scale, po, pm, pl, num_seqs, qmax, nsplit, window=-1, causal=True, **kw):
        self.calls.append(("decode", q.shape[0], num_seqs, window, kw))

    def forward_window(self, q, kc, vc, bt, sl, scale, qsl, out, window, sinks=0, exact=False):
        self.calls.append(("window", q.shape[0], bt.shape[0], sl.tolist(), qsl.tolist(), window, sinks, exact))


@pytest.fixture
def ops(monkeypatch):
    o = Ops()
    monkeypatch.setattr(shim, "load_pth_dec", lambda: o)
    monkeypatch.setattr(shim, "load_pth_fa", lambda: o)
    return o


def impl(**kw):
    a = dict(num_heads=24, num_kv_heads=4, head_size=256, scale=1 / 16, kv_quant_int8_per_token_head=True, is_rocm=True,
             is_decoder=True, sliding_window=(1023, -1))
    a.update(kw)
    return shim.Gfx950Int8Attention(**a)


def batch(qlens, lens, dtype=torch.float16):
    qsl = torch.tensor([0] + list(torch.tensor(qlens).cumsum(0)), dtype=torch.int32)
    T = int(qsl[-1])
    m = shim.AttnMeta(query_start_loc=qsl, query_start_loc_cpu=qsl, seq_lens=torch.tensor(lens, dtype=torch.int32),
                      block_table=torch.zeros((len(lens), 300), dtype=torch.int32), max_seq_len=max(lens),
                      softmax_segm_output=torch.empty((8, 24, 16, 256)), softmax_segm_max=torch.empty((8, 24, 16)),
                      softmax_segm_expsum=torch.empty((8, 24, 16)), seq_lens_cpu=torch.tensor(lens, dtype=torch.int32))
    return torch.zeros((T, 24, 256), dtype=dtype), torch.zeros((T, 24, 256), dtype=dtype), m


def route(a, q, out, m, qlens, fallback=None):
    kc = torch.zeros((4, 16, 4, 260), dtype=torch.int8)
    return a.route(q, kc, kc, None, None, m, out, max(qlens), q.shape[0], fallback or (lambda *x: pytest.fail("fallback")))


def test_prefill_of_a_windowed_layer(ops):
    a = impl(sink_tokens=4)
    assert a.pth_fa is None and a.pth_fa_window is ops and a.window == 1024
    q, out, m = batch([2, 1, 100, 64], [500, 20, 9000, 64])
    assert route(a, q, out, m, [100])
    assert ops.calls == [("decode", 3, 2, 1024, {"sinks": 4}), ("window", 167, 2, [9000, 64], [3, 103, 167], 1024, 4, False)]


def test_decode_of_a_windowed_layer_without_sinks_is_as_before(ops):
    q, out, m = batch([2, 1], [500, 20])
    assert route(impl(), q, out, m, [2])
    assert ops.calls == [("decode", 3, 2, 1024, {})]


def test_sink_tokens_without_a_window_mean_nothing(ops):
    a = impl(sliding_window=(-1, -1), sink_tokens=9)
    assert a.sink_tokens == 0 and a.pth_fa_window is None and a.pth_fa is ops


def test_a_right_bound_of_none_is_causal(ops):
    """vLLM gives a windowed decoder layer (W - 1, 0): its prefill is taken, its decode, as before, is not."""
    a = impl(sliding_window=(1023, 0))
    assert a.pth_fa_window is ops and a.pth_dec is None
    rows = []
    q, out, m = batch([2, 100], [500, 9000])
    assert route(a, q, out, m, [100], lambda *x: rows.append(x))
    assert rows == [(0, 2, 0, 1, 2)] and ops.calls == [("window", 102, 1, [9000], [2, 102], 1024, 0, False)]
    assert impl(sliding_window=(1023, 5)).pth_fa_window is None


@pytest.mark.parametrize("spoil", ["dtype", "layout", "stride", "group", "operator"])
def test_what_stays_with_the_caller(ops, monkeypatch, spoil):
    if spoil == "layout":
        ops.layout = False
    if spoil == "operator":  # a library without it
        monkeypatch.setattr(shim, "load_pth_fa", lambda: object())
    a = impl(num_heads=1028) if spoil == "group" else impl()
    q, out, m = batch([100], [9000], torch.bfloat16 if spoil == "dtype" else torch.float16)
    if spoil == "stride":
        q = torch.zeros((100, 24, 260), dtype=torch.float16)[..., :256]
    assert not route(a, q, out, m, [100]) and not ops.calls


def test_captured_calls_do_not_look_at_the_lengths(ops):
    q, out, m = batch([100], [9000])
    m.seq_lens_cpu = None
    m.max_seq_len = 0
    assert route(impl(), q, out, m, [100]) and ops.calls[0][0] == "window"
