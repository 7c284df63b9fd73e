"""The operators around the attention (rotary cache write, running key weights, eviction, decode with the rows' logarithms)
without a GPU: what their entries refuse and with which message, empty calls, the Python face on host tensors, and
the rotary tables against their formulas.
"""
import ctypes
import math

import numpy as np
import pytest
import torch

import workload as kvc
from mi50_vllm_lab_amd import pth_dec, rotary


@pytest.fixture(scope="module")
def lib():
    return pth_dec.load_library()


def make(**kw):
    a = dict(num_q_heads=12, num_kv_heads=2, block_size=16, seed=3)
    a.update(kw)
    return kvc.make_case([37, 5], [3, 1], **a)


def call(fn, tensors, *scalars):
    """rc and message of an entry that takes its tensors first (None: a null descriptor)."""
    descs = [None if t is None else ctypes.byref(pth_dec.describe(t)) for t in tensors]
    err = ctypes.create_string_buffer(256)
    rc = fn(*descs, *scalars, None, err, len(err))
    return rc, err.value.decode()


def refusals(fn, names, good, scalars, cases):
    for change, msg in cases:
        t = {**good, **{k: v for k, v in change.items() if k in good}}
        s = {**scalars, **{k: v for k, v in change.items() if k in scalars}}
        assert set(change) <= set(good) | set(scalars)
        rc, text = call(fn, [t[n] for n in names], *s.values())
        assert rc == 1 and msg in text, (list(change), rc, text)


def test_rotary_write_refusals(lib):
    c = make().cache
    x = torch.zeros((3, 16, 256), dtype=torch.float16)
    names = ("query", "query_out", "key", "value", "positions", "cos_sin", "kc", "vc", "ks", "vs", "slots")
    good = dict(query=x[:, :12], query_out=x[:, :12], key=x[:, 12:14], value=x[:, 14:], positions=torch.zeros(3, dtype=torch.int64),
                cos_sin=torch.zeros((9, 64)), kc=c.key_cache, vc=c.value_cache, ks=c.k_scale, vs=c.v_scale,
                slots=torch.zeros(3, dtype=torch.int64))
    one = torch.zeros((1, 1, 256), dtype=torch.float16)
    cases = [({n: None}, "null tensor descriptor") for n in names] + [
        (dict(kc=c.value_cache), "KV cache views"),
        (dict(query=x[:, :12].int()), "fp16, bf16 or fp32"),
        (dict(key=x[:, 12:14].float()), "fp16, bf16 or fp32"),
        (dict(value=x[:, 14:].bfloat16()), "fp16, bf16 or fp32"),
        (dict(query=x), "query_out must be [T, Hq, 256]"),
        (dict(query=x[0]), "query must be [T, Hq, 256]"),
        (dict(query=x.view(3, 8, 512)[..., ::2]), "query must be [T, Hq, 256]"),
        (dict(query=x[:, :0], query_out=x[:, :0]), "query must be [T, Hq, 256]"),
        (dict(key=x[:, 11:14]), "[T, Hkv, 256]"),
        (dict(value=x[:2, 14:]), "[T, Hkv, 256]"),
        (dict(query_out=x[:, :12].float()), "query's dtype or fp16"),
        (dict(query_out=x[:2, :12]), "query's dtype or fp16"),
        (dict(query_out=x.view(3, 8, 512)[:, :, :256]), "query's dtype or fp16"),
        (dict(query_out=x.as_strided((3, 12, 256), (16 * 256, 256 + 4, 1))), "itself or not overlap"),
        (dict(query=x[:1, :12].expand(3, 12, 256), query_out=x[:1, :12].expand(3, 12, 256)), "rows must not overlap"),
        (dict(query_out=x[:, :1].expand(3, 12, 256)), "rows must not overlap"),
        (dict(query_out=x.as_strided((3, 12, 256), (256, 256, 1))), "rows must not overlap"),
        (dict(query_out=x.as_strided((3, 12, 256), (11 * 256 + 4, 256, 1))), "rows must not overlap"),
        (dict(query_out=x.as_strided((3, 12, 256), (256, 3 * 256 - 4, 1))), "rows must not overlap"),
        (dict(positions=torch.zeros(3, dtype=torch.int32)), "positions must be"),
        (dict(positions=torch.zeros(2, dtype=torch.int64)), "positions must be"),
        (dict(positions=torch.zeros(6, dtype=torch.int64)[::2]), "positions must be"),
        (dict(slots=torch.zeros(3, dtype=torch.int32)), "slot_mapping must be"),
        (dict(slots=torch.zeros(2, dtype=torch.int64)), "slot_mapping must be"),
        (dict(cos_sin=torch.zeros((9, 64)).double()), "cos_sin must be"),
        (dict(cos_sin=torch.zeros((9, 60))), "cos_sin must be"),
        (dict(cos_sin=torch.zeros((9, 264))), "cos_sin must be"),
        (dict(cos_sin=torch.zeros((9, 0))), "cos_sin must be"),
        (dict(cos_sin=torch.zeros((9, 128))[:, ::2]), "cos_sin must be"),
        (dict(cos_sin=torch.zeros(9 * 64 + 1)[1:].view(9, 64)), "cos_sin must be"),
        (dict(cos_sin=torch.zeros((9, 66))[:, :64]), "cos_sin must be"),
        (dict(query=x.view(-1)[1:1 + 2 * 16 * 256].view(2, 16, 256)[:, :12], query_out=x[:2, :12], key=x[:2, 12:14], value=x[:2, 14:]), "aligned to 4"),
        (dict(query=one.expand(1 << 27 | 1, 12, 256), query_out=one.expand(1 << 27 | 1, 12, 256),
              key=one.expand(1 << 27 | 1, 2, 256), value=one.expand(1 << 27 | 1, 2, 256)), "at most 2^30"),
    ]
    refusals(lib.pth_cache_write_rotary, names, good, dict(interleaved=0), cases)
    none = {k: v[:0] if k in ("query", "query_out", "key", "value", "positions", "slots") else v for k, v in good.items()}
    assert call(lib.pth_cache_write_rotary, [none[n] for n in names], 0) == (0, "")


def test_bf16_query_out_of_another_type_is_refused(lib):
    c = make().cache
    x = torch.zeros((3, 16, 256), dtype=torch.float16)
    t = [x[:, :12], x[:, :12].bfloat16(), x[:, 12:14], x[:, 14:], torch.zeros(3, dtype=torch.int64), torch.zeros((9, 64)),
         c.key_cache, c.value_cache, c.k_scale, c.v_scale, torch.zeros(3, dtype=torch.int64)]
    rc, text = call(lib.pth_cache_write_rotary, t, 0)
    assert rc == 1 and "query's dtype or fp16" in text


def test_key_weights_refusals(lib):
    case = make()
    c, big = case.cache, 1 << 31
    names = ("q", "kc", "vc", "ks", "vs", "bt", "lens", "qsl", "lse", "weights")
    good = dict(q=case.q, kc=c.key_cache, vc=c.value_cache, ks=c.k_scale, vs=c.v_scale, bt=case.block_table, lens=case.seq_lens,
                qsl=case.query_start_loc, lse=torch.zeros((4, 12)), weights=torch.zeros((2, 2, 50)))
    cases = [({n: None}, "null tensor descriptor") for n in names] + [
        (dict(q=case.q.float()), "q must be fp16"),
        (dict(q=case.q[..., :128]), "q must be fp16"),
        (dict(q=case.q.transpose(0, 1)), "q must be fp16"),
        (dict(vc=c.key_cache), "KV cache views"),
        (dict(q=case.q[:, :11]), "multiple of heads_kv"),
        (dict(qmax=0), "[1, 48]"),
        (dict(qmax=9), "[1, 48]"),
        (dict(qmax=big), "[1, 48]"),
        (dict(num_seqs=0), "row for each"),
        (dict(num_seqs=3), "row for each"),
        (dict(bt=case.block_table.long()), "row for each"),
        (dict(bt=case.block_table.t()), "row for each"),
        (dict(lens=case.seq_lens.long()), "row for each"),
        (dict(qsl=case.query_start_loc[:2]), "row for each"),
        (dict(lens=torch.zeros((4,), dtype=torch.int32)[::2]), "row for each"),
        (dict(lse=torch.zeros((3, 12))), "lse must be"),
        (dict(lse=torch.zeros((4, 12)).half()), "lse must be"),
        (dict(lse=torch.zeros((12, 4)).t()), "lse must be"),
        (dict(weights=torch.zeros((2, 3, 50))), "weights must be"),
        (dict(weights=torch.zeros((1, 2, 50))), "weights must be"),
        (dict(weights=torch.zeros((2, 2, 50)).double()), "weights must be"),
        (dict(weights=torch.zeros((2, 2, 100))[..., ::2]), "weights must be"),
        (dict(weights=torch.zeros((1, 2, 50)).expand(2, 2, 50)), "its rows apart"),
        (dict(weights=torch.zeros((2, 1, 50)).expand(2, 2, 50)), "its rows apart"),
        (dict(weights=torch.zeros(200).as_strided((2, 2, 50), (99, 50, 1))), "its rows apart"),
    ]
    scalars = dict(scale=ctypes.c_double(0.1), num_seqs=2, qmax=3)
    refusals(lib.pth_cache_key_weights, names, good, scalars, cases)
    for empty in (dict(q=case.q[:0], lse=torch.zeros((0, 12))), dict(weights=torch.zeros((2, 2, 0))),
                  dict(weights=torch.zeros((1, 1, 0)).expand(2, 2, 0))):
        t = {**good, **empty}
        assert call(lib.pth_cache_key_weights, [t[n] for n in names], *scalars.values()) == (0, "")


def test_evict_refusals(lib):
    case = make()
    c = case.cache
    names = ("weights", "kc", "vc", "ks", "vs", "bt", "lens", "nbt", "nlens", "nweights", "kept")
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    good = dict(weights=torch.zeros((2, 2, 50)), kc=c.key_cache, vc=c.value_cache, ks=c.k_scale, vs=c.v_scale, bt=case.block_table,
                lens=case.seq_lens, nbt=i32(2, 2), nlens=i32(2), nweights=torch.zeros((2, 2, 20)), kept=i32(2, 2, 20))
    cases = [({n: None}, "null tensor descriptor") for n in names] + [
        (dict(ks=c.v_scale), "KV cache views"),
        (dict(keep=0), "keep must be"),
        (dict(recent=-1), "keep must be"),
        (dict(recent=21), "keep must be"),
        (dict(keep=1 << 31), "keep must be"),
        (dict(num_seqs=0), "row for each"),
        (dict(num_seqs=3), "row for each"),
        (dict(nbt=i32(1, 2)), "row for each"),
        (dict(nbt=i32(2, 2).long()), "row for each"),
        (dict(nlens=i32(1)), "row for each"),
        (dict(lens=case.seq_lens.float()), "row for each"),
        (dict(nbt=i32(2, 1)), "must hold keep keys"),
        (dict(weights=torch.zeros((2, 3, 50))), "weights and new_weights"),
        (dict(weights=torch.zeros((2, 2, 100))[..., ::2]), "weights and new_weights"),
        (dict(nweights=torch.zeros((2, 2, 19))), "weights and new_weights"),
        (dict(nweights=torch.zeros((2, 2, 20)).half()), "weights and new_weights"),
        (dict(nweights=torch.zeros((1, 2, 20)).expand(2, 2, 20)), "its rows apart"),
        (dict(nweights=torch.zeros((2, 1, 20)).expand(2, 2, 20)), "its rows apart"),
        (dict(kept=i32(2, 2, 21)), "kept must be"),
        (dict(kept=i32(2, 2, 20).long()), "kept must be"),
        (dict(kept=i32(2, 2, 40)[..., ::2]), "kept must be"),
        (dict(nweights=good["weights"]), "must not be the old ones"),
        (dict(nlens=good["lens"]), "must not be the old ones"),
        (dict(nbt=good["bt"]), "must not be the old ones"),
    ]
    refusals(lib.pth_cache_evict, names, good, dict(num_seqs=2, keep=20, recent=4), cases)


def test_decode_lse_refusals(lib):
    case = make()
    c = case.cache
    po, pm, pl = kvc.partial_buffers(4, 12, 4, "cpu")
    front = [case.q, c.key_cache, c.value_cache, c.k_scale, c.v_scale, case.block_table, case.seq_lens, case.query_start_loc,
             torch.zeros((4, 12, 256), dtype=torch.float16)]

    def run(lse, q=case.q):
        tail = [po, pm, pl, lse]
        d = lambda ts: [None if t is None else ctypes.byref(pth_dec.describe(t)) for t in ts]  # noqa: E731
        err = ctypes.create_string_buffer(256)
        rc = lib.pth_dec_decode_lse(*d([q] + front[1:]), ctypes.c_double(0.1), *d(tail), 2, 3, 4, -1, 1, None, err, len(err))
        return rc, err.value.decode()

    for lse, msg in ((None, "null tensor descriptor"), (torch.zeros((3, 12)), "lse must be"), (torch.zeros((4, 11)), "lse must be"),
                     (torch.zeros((4, 12)).half(), "lse must be"), (torch.zeros((12, 4)).t(), "lse must be"), (torch.zeros(48), "lse must be")):
        rc, text = run(lse)
        assert rc == 1 and msg in text, (rc, text)
    rc, text = run(torch.zeros((4, 12)), q=case.q.float())
    assert rc == 1 and "q must be fp16" in text


def test_decode_shared_refusals(lib):
    case = make()
    c = case.cache
    table = case.block_table.shape[1] * 16
    front = [case.q, c.key_cache, c.value_cache, c.k_scale, c.v_scale, case.block_table, case.seq_lens, case.query_start_loc,
             torch.zeros((4, 12, 256), dtype=torch.float16)]

    def run(prefix=32, nseg=4, qmax=3, num_seqs=2, lse=None, at=None, t=None):
        ts = list(front)
        if at is not None:
            ts[at] = t
        d = lambda xs: [None if x is None else ctypes.byref(pth_dec.describe(x)) for x in xs]  # noqa: E731
        err = ctypes.create_string_buffer(256)
        rc = lib.pth_dec_decode_shared(*d(ts), ctypes.c_double(0.1), *d([*kvc.partial_buffers(4, 12, nseg, "cpu"), lse]), num_seqs, qmax,
                                       prefix, None, err, len(err))
        return rc, err.value.decode()

    one = torch.zeros((1, 1, 256), dtype=torch.float16)
    for kw, msg in (
        (dict(prefix=-1), "prefix_len must be"), (dict(prefix=table + 1), "prefix_len must be"), (dict(prefix=1 << 31), "prefix_len must be"),
        (dict(nseg=3), "at least 4 segments"), (dict(qmax=9), "[1, 48]"), (dict(qmax=0), "[1, 48]"), (dict(num_seqs=3), "too small"),
        (dict(num_seqs=0), "too small"), (dict(lse=torch.zeros((4, 11))), "lse must be"),
        (dict(at=0, t=None), "null tensor descriptor"), (dict(at=0, t=case.q.float()), "q must be fp16"),
        (dict(at=2, t=c.key_cache), "KV cache views"), (dict(at=5, t=case.block_table.long()), "must be int32"),
        (dict(at=8, t=one.expand(4, 12, 256).transpose(0, 1)), "out must be"),
    ):
        rc, text = run(**kw)
        assert rc == 1 and msg in text, (list(kw), rc, text)
    # a table wide enough for more key tiles than 32 bits number (described, never read)
    wide = pth_dec.describe(case.block_table)
    wide.sizes[1] = 1 << 30
    err = ctypes.create_string_buffer(256)
    descs = [pth_dec.describe(x) for x in front]
    descs[5] = wide
    assert lib.pth_dec_decode_shared(*[ctypes.byref(x) for x in descs], ctypes.c_double(0.1),
                                     *[ctypes.byref(pth_dec.describe(x)) for x in kvc.partial_buffers(4, 12, 4, "cpu")], None, 2, 3, 32, None,
                                     err, len(err)) == 1 and b"at most 2^25" in err.value
    assert lib.pth_dec_decode_shared(*[ctypes.byref(pth_dec.describe(x[:0] if i in (0, 8) else x)) for i, x in enumerate(front)],
                                     ctypes.c_double(0.1), *[ctypes.byref(pth_dec.describe(x)) for x in kvc.partial_buffers(4, 12, 4, "cpu")],
                                     None, 2, 3, 32, None, None, 0) == 0


def test_python_face_refuses_host_tensors():
    case = make()
    c = case.cache
    views = (c.key_cache, c.value_cache, c.k_scale, c.v_scale)
    x = torch.zeros((3, 16, 256), dtype=torch.float16)
    n64 = torch.zeros(3, dtype=torch.int64)
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    with pytest.raises(RuntimeError, match="one GPU"):
        pth_dec.rotary_cache_write(x[:, :12], x[:, 12:14], x[:, 14:], n64, torch.zeros((9, 64)), *views, n64)
    with pytest.raises(RuntimeError, match="one GPU"):
        pth_dec.decode_shared(case.q, *views, case.block_table, case.seq_lens, case.query_start_loc, torch.empty_like(case.q), 0.1,
                              *kvc.partial_buffers(4, 12, 4, "cpu"), 2, 3, 16)
    with pytest.raises(RuntimeError, match="one GPU"):
        pth_dec.key_weights(case.q, *views, case.block_table, case.seq_lens, case.query_start_loc, torch.zeros((4, 12)),
                            torch.zeros((2, 2, 50)), 0.1, 2, 3)
    with pytest.raises(RuntimeError, match="one GPU"):
        pth_dec.evict(torch.zeros((2, 2, 50)), *views, case.block_table, case.seq_lens, i32(2, 2), i32(2), torch.zeros((2, 2, 20)),
                      i32(2, 2, 20), 2, 20, 4)


# ---- rotary tables ----

def test_rotary_table_is_the_rounded_cosine_and_sine():
    t = rotary.rotary_table(64, 70001, base=1e6)
    assert t.shape == (70001, 64) and t.dtype == torch.float32
    for p in (0, 1, 65535, 65536, 70000):
        angle = p * np.power(1e6, -np.arange(0, 64, 2, dtype=np.float64) / 64)
        # the angle carries 2^-52 relative, the cosine as much absolutely; then one rounding to fp32
        want = np.concatenate([np.cos(angle), np.sin(angle)])
        assert np.abs(t[p].double().numpy() - want).max() <= 2.0 ** -24 * 0.5 + 70000 * 2.0 ** -51


def test_rotary_scalings():
    dim, base = 128, 10000.0
    plain, one = rotary.rotary_frequencies(dim, base)
    assert one == 1.0 and plain[0] == 1.0
    lin, _ = rotary.rotary_frequencies(dim, base, {"type": "linear", "factor": 4})
    assert torch.equal(lin, plain / 4)
    ntk, _ = rotary.rotary_frequencies(dim, base, {"type": "ntk", "factor": 8})
    assert ntk[0] == 1.0 and abs(float(ntk[-1] * 8 / plain[-1]) - 1) < 1e-12 and bool((ntk <= plain).all())
    s = {"type": "yarn", "factor": 16, "original_max_position": 4096}
    yarn, mult = rotary.rotary_frequencies(dim, base, s)
    turns = 4096 * plain / (2 * math.pi)
    kept, slow = turns > 40, turns < 0.8
    assert bool(kept.any()) and bool(slow.any())
    assert torch.equal(yarn[kept], plain[kept])
    assert torch.allclose(yarn[slow], plain[slow] / 16, rtol=1e-12)
    between = ~kept & ~slow
    assert bool((yarn[between] <= plain[between]).all()) and bool((yarn[between] >= plain[between] / 16).all())
    assert abs(mult - (0.1 * math.log(16) + 1)) < 1e-12
    assert rotary.rotary_frequencies(dim, base, {**s, "attention_factor": 1.5})[1] == 1.5
    table = rotary.rotary_table(dim, 3, base, s)
    assert torch.allclose(table[0], torch.cat([torch.full((64,), mult), torch.zeros(64)]))


def test_rotary_tables_refuse():
    for bad in (dict(rotary_dim=0), dict(rotary_dim=7), dict(rotary_dim=64, scaling={"type": "other", "factor": 2}),
                dict(rotary_dim=64, scaling={"type": "linear", "factor": 0.5})):
        with pytest.raises(ValueError):
            rotary.rotary_frequencies(**bad)
    with pytest.raises(ValueError):
        rotary.rotary_table(64, -1)
    assert rotary.rotary_table(64, 0).shape == (0, 64)
