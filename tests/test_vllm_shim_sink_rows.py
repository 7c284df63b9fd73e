"""The shim's layers with sink_tokens, without a GPU: no row of theirs goes to the caller, whose own path knows nothing of the sinks,
whatever the window's form, the turns' lengths, the rows' type and strides and the buffers at hand; and what no operator takes raises.
"""
import pytest
import torch

from mi50_vllm_lab_amd import vllm_shim as shim


class Ops:
    def __init__(self):
        self.calls, self.layout = [], True

    def supported_layout(self, *views):
        return self.layout

    def decode(self, q, kc, vc, ks, vs, bt, sl, qsl, out, scale, po, pm, pl, num_seqs, qmax, nsplit, window=-1, causal=True, sinks=0):
        assert q.dtype == out.dtype == torch.float16
        out.fill_(2.0)
        self.calls.append(("decode", qsl.tolist(), window, sinks))

    def forward_window(self, q, kc, vc, bt, sl, scale, qsl, out, window, sinks=0):
        assert q.dtype == out.dtype == torch.float16 and q.stride(0) % 8 == 0 and q.stride(2) == out.stride(2) == 1
        assert bt.shape[0] == sl.shape[0] == qsl.shape[0] - 1
        for i in range(sl.shape[0]):
            if int(sl[i]) > 0:
                out[int(qsl[i]):int(qsl[i + 1])] = q[int(qsl[i]):int(qsl[i + 1])] + 1.0
        self.calls.append(("window", qsl.tolist(), window, sinks))


@pytest.fixture
def ops(monkeypatch):
    o = Ops()
    monkeypatch.setattr(shim, "load_pth_dec", lambda: o)
    monkeypatch.setattr(shim, "load_pth_fa", lambda: o)
    return o


def impl(**kw):
    a = dict(num_heads=24, num_kv_heads=4, head_size=256, scale=1 / 16, kv_quant_int8_per_token_head=True, is_rocm=True,
             is_decoder=True, sliding_window=(1023, 0), sink_tokens=4)
    a.update(kw)
    return shim.Gfx950Int8Attention(**a)


def route(a, qlens, lens=None, dtype=torch.float16, segments=True, strided=False, spare=0, **kw):
    lens = lens or [500 + n for n in qlens]
    qsl = torch.tensor([0] + list(torch.tensor(qlens).cumsum(0)), dtype=torch.int32)
    T = int(qsl[-1]) + spare
    part = (lambda *s: torch.empty(s)) if segments else (lambda *s: None)
    m = shim.AttnMeta(query_start_loc=qsl, query_start_loc_cpu=qsl, seq_lens=torch.tensor(lens, dtype=torch.int32),
                      block_table=torch.zeros((len(lens), 300), dtype=torch.int32), max_seq_len=max(lens),
                      softmax_segm_output=part(8, 24, 16, 256), softmax_segm_max=part(8, 24, 16),
                      softmax_segm_expsum=part(8, 24, 16), seq_lens_cpu=torch.tensor(lens, dtype=torch.int32))
    for k, v in kw.items():
        setattr(m, k, v)
    q = torch.ones((T, 24, 260 if strided else 256), dtype=dtype)[..., :256]
    out = torch.full((T, 24, 256), 7.0, dtype=dtype)
    kc = torch.zeros((4, 16, 4, 260), dtype=torch.int8)
    done = a.route(q, kc, kc, None, None, m, out, max(qlens), T, lambda *x: pytest.fail("rows left to the caller"))
    return done, out


@pytest.mark.parametrize("bounds", [(1023, 0), (1023, -1)])
@pytest.mark.parametrize("qlens,calls", [
    ([1], [("decode", [0, 1])]),
    ([1, 4, 2], [("decode", [0, 1, 5, 7])]),
    ([1, 100], [("decode", [0, 1]), ("window", [1, 101])]),
    ([2, 1, 100, 64], [("decode", [0, 2, 3]), ("window", [3, 103, 167])]),
    ([10], [("window", [0, 10])]),                       # more than decode takes, fewer than a prefill's
    ([1, 5, 1], [("window", [0, 1, 6, 7])]),
    ([10, 100], [("window", [0, 10, 110])]),
    ([100, 1], [("window", [0, 100, 101])]),             # the long turns are no suffix
    ([64, 63], [("window", [0, 64, 127])]),
])
def test_every_row_goes_to_an_operator_with_the_sinks(ops, bounds, qlens, calls):
    done, out = route(impl(sliding_window=bounds), qlens)
    assert done and ops.calls == [(name, starts, 1024, 4) for name, starts in calls]
    assert bool((out == 2.0).all()) or "window" in dict(calls)


@pytest.mark.parametrize("qlens", [[1], [1, 3], [1, 100], [10]])
@pytest.mark.parametrize("why", ["bf16", "fp32", "strided", "segments", "few segments", "decode off", "group"])
def test_what_decode_does_not_take(ops, monkeypatch, qlens, why):
    if why == "decode off":
        monkeypatch.setattr(shim, "load_pth_dec", lambda: None)
    a = impl(num_kv_heads=1) if why == "group" else impl()  # 24 x 4 rows per kv head
    done, out = route(a, qlens, dtype={"bf16": torch.bfloat16, "fp32": torch.float32}.get(why, torch.float16), segments=why != "segments",
                      strided=why == "strided", **({"softmax_segm_output": torch.empty((0, 24, 16, 256))} if why == "few segments" else {}))
    starts = [0] + list(torch.tensor(qlens).cumsum(0).tolist())
    assert done and ops.calls == [("window", starts, 1024, 4)] and bool((out == 2.0).all())


def test_rows_of_no_sequence_stay_as_they_were(ops):
    """also where the rows go through copies."""
    for dtype in (torch.float16, torch.bfloat16):
        done, out = route(impl(), [10, 3, 5], lens=[40, 0, 9], dtype=dtype, spare=2)
        assert done and bool((out[:10] == 2.0).all()) and bool((out[10:13] == 7.0).all())
        assert bool((out[13:18] == 2.0).all()) and bool((out[18:] == 7.0).all())


@pytest.mark.parametrize("change", [dict(causal=False), dict(mm_prefix_range_tensor=torch.zeros(1)), dict(rswa_prefix_lens=torch.zeros(1))])
def test_batches_that_no_operator_takes_raise(ops, change):
    with pytest.raises(RuntimeError, match="sink_tokens"):
        route(impl(), [1], **change)
    assert not ops.calls


def test_an_unknown_cache_layout_raises(ops):
    ops.layout = False
    for qlens in ([1], [100], [1, 100]):
        with pytest.raises(RuntimeError, match="sink_tokens"):
            route(impl(), qlens)
    assert not ops.calls


@pytest.mark.parametrize("change", [dict(head_size=128), dict(is_decoder=False), dict(logits_soft_cap=30.0), dict(sinks=torch.zeros(24)),
                                    dict(sliding_window=(1023, 5)), dict(num_heads=1028), dict(on_gfx950=False)])
def test_layers_that_no_operator_takes_raise(ops, change):
    with pytest.raises(RuntimeError, match="sink_tokens"):
        impl(**change)
    impl(**{**change, "sink_tokens": 0})
    impl(**{**change, "sliding_window": (-1, -1)})  # (without a window every key is seen anyway)


def test_the_prefill_operator_has_to_be_there(ops, monkeypatch):
    monkeypatch.setattr(shim, "load_pth_fa", lambda: None)
    with pytest.raises(RuntimeError, match="sink_tokens"):
        impl()
    impl(sink_tokens=0)
