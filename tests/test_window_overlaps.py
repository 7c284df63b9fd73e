"""forward_window refuses an `out` or a workspace over what the call reads, or over each other, without a GPU; tensors that share a buffer
and no byte are taken."""
import ctypes

import pytest
import torch

import workload as kvc
from mi50_vllm_lab_amd import pth_dec

T, HQ = 4, 12
WS = T * HQ * 2 * 258


@pytest.fixture(scope="module")
def lib():
    return pth_dec.load_library()


def call(lib, **kw):
    case = kvc.make_case([37, 5], [3, 1], num_q_heads=HQ, num_kv_heads=2, block_size=16, seed=3)
    c = case.cache
    a = dict(q=case.q, kc=c.key_cache, vc=c.value_cache, bt=case.block_table, lens=case.seq_lens, qsl=case.query_start_loc,
             out=torch.zeros((T, HQ, 256), dtype=torch.float16), ws=torch.zeros(WS), nsplit=2)
    for k, v in kw.items():
        a[k] = v(a) if callable(v) else v
    d = {n: ctypes.byref(pth_dec.describe(a[n])) for n in a if n != "nsplit"}
    err = ctypes.create_string_buffer(256)
    rc = lib.pth_fa_forward_window(*[d[n] for n in ("q", "kc", "vc", "bt", "lens")], 0.1, d["qsl"], d["out"], d["ws"], 2, 16, 4, a["nsplit"], 0,
                                   None, err, len(err))
    return rc, err.value.decode()


def over(t, shape, dtype, shift=0):
    """A tensor of that shape over the bytes of t (from byte `shift` on)."""
    flat = torch.as_strided(t, (t.untyped_storage().nbytes() // t.element_size(),), (1,), 0).view(torch.uint8)
    n = torch.Size(shape).numel() * torch.empty((), dtype=dtype).element_size()
    return flat[shift:shift + n].view(dtype).view(shape)


def roomy(t):
    """t at the start of a buffer that a whole `out` fits in."""
    n = t.numel()
    return torch.cat([t.reshape(-1), torch.zeros(T * HQ * 512 // t.element_size(), dtype=t.dtype)])[:n].view(t.shape)


OUT = ((T, HQ, 256), torch.float16)
big = torch.zeros((2 * T * HQ + 20, 256), dtype=torch.float16)


@pytest.mark.parametrize("change", [
    dict(out=lambda a: a["q"]),
    dict(q=big[:T * HQ].view(T, HQ, 256), out=big[7:T * HQ + 7].view(T, HQ, 256)),
    dict(q=big[:72].view(T, 18, 256)[:, :HQ], out=big[:72].view(T, 18, 256)[:, 6:]),             # heads 6 to 11 are in both
    dict(out=lambda a: over(a["kc"], *OUT)),
    dict(bt=lambda a: roomy(a["bt"]), out=lambda a: over(a["bt"], *OUT)),
    dict(lens=lambda a: roomy(a["lens"]), out=lambda a: over(a["lens"], *OUT)),
    dict(qsl=lambda a: roomy(a["qsl"]), out=lambda a: over(a["qsl"], *OUT, shift=8)),
    dict(ws=torch.zeros(WS + T * HQ * 128), out=lambda a: over(a["ws"], *OUT, shift=4 * WS - 16)),
    dict(ws=torch.zeros(WS + T * HQ * 128), q=lambda a: over(a["ws"], *OUT, shift=4 * WS - 16)),
    dict(ws=lambda a: over(a["kc"], (WS,), torch.float32, 48)),
], ids=lambda c: "+".join(c))
def test_overlaps_are_refused(lib, change):
    rc, text = call(lib, **change)
    assert rc == 1 and "must not overlap each other or what the call reads" in text, (rc, text)


@pytest.mark.parametrize("change", [
    dict(q=big[:2 * T * HQ].view(T, 2 * HQ, 256)[:, :HQ], out=big[:2 * T * HQ].view(T, 2 * HQ, 256)[:, HQ:]),   # heads of one buffer
    dict(q=big[:T * HQ].view(T, HQ, 256), out=big[T * HQ:2 * T * HQ].view(T, HQ, 256)),
    dict(ws=torch.zeros(WS + T * HQ * 128), out=lambda a: over(a["ws"], *OUT, shift=4 * WS)),
    dict(ws=lambda a: over(a["kc"], (WS,), torch.float32, 48), nsplit=1),                                       # not looked at
])
def test_neighbours_are_not(lib, change):
    rc, text = call(lib, **change)
    assert rc != 1, text  # (2: there is no GPU to launch on)


@pytest.mark.gpu
def test_heads_of_one_buffer():
    import window_oracle

    case = kvc.make_case([200], [50], seed=8)
    d = case.to("cuda")
    x = torch.full((50, 48, 256), 7.0, dtype=torch.float16, device="cuda")
    x[:, :24] = d.q
    with pytest.raises(RuntimeError, match="must not overlap"):
        pth_dec.forward_window(x[:, :24], d.cache.key_cache, d.cache.value_cache, d.block_table, d.seq_lens, d.scale, d.query_start_loc,
                               x[:, 23:47], 64, sinks=5)
    pth_dec.forward_window(x[:, :24], d.cache.key_cache, d.cache.value_cache, d.block_table, d.seq_lens, d.scale, d.query_start_loc, x[:, 24:],
                           64, sinks=5)
    ref, _, _ = window_oracle.windowed(case, 64, 5)
    assert kvc.fp16_output_errors(x[:, 24:].double().cpu().numpy(), ref)[2] <= 0


def test_more_tokens_than_a_merge_launch_numbers(lib):
    """Described, never read: 2^24 workgroups of four tokens are one too many, and only splits are merged."""
    case = kvc.make_case([37], [3], num_q_heads=1, num_kv_heads=1, block_size=16, seed=3)
    rows = lambda n: case.q[:1].expand(n, 1, 256)  # noqa: E731

    def why(n, nsplit):
        c = case.cache
        err = ctypes.create_string_buffer(256)
        d = [ctypes.byref(pth_dec.describe(t)) for t in (rows(n), c.key_cache, c.value_cache, case.block_table, case.seq_lens,
                                                        case.query_start_loc, rows(n), torch.zeros(8))]
        assert lib.pth_fa_forward_window(*d[:5], 0.1, *d[5:], 1, 16, 4, nsplit, 0, None, err, len(err)) == 1
        return err.value.decode()

    assert "2^24 workgroups" in why(2 ** 26 - 3, 2) and "2^24 workgroups" in why(2 ** 26, 64)
    assert "out rows must not overlap" in why(2 ** 26 - 4, 2) and "out rows must not overlap" in why(2 ** 26, 1)
