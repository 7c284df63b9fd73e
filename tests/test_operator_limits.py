"""Calls at the edges of what the operators around a decode step take, without a GPU: empty batches with views of other strides or
types, and sizes at which a 32-bit index or the number of workgroups of a launch would not do (described, never read).
"""
import ctypes

import pytest
import torch

import workload as kvc
from mi50_vllm_lab_amd import pth_dec


@pytest.fixture(scope="module")
def lib():
    return pth_dec.load_library()


def case():
    return kvc.make_case([37, 5], [3, 1], num_q_heads=12, num_kv_heads=2, block_size=16, seed=3)


def call(fn, descs, *scalars):
    err = ctypes.create_string_buffer(256)
    rc = fn(*[ctypes.byref(d) for d in descs], *scalars, None, err, len(err))
    return rc, err.value.decode()


def describe(*ts):
    return [pth_dec.describe(t) for t in ts]


def views(c):
    return c.key_cache, c.value_cache, c.k_scale, c.v_scale


# ---- no tokens ----

@pytest.mark.parametrize("dtype,out", [
    ("fp16", lambda hq: torch.empty((0, hq, 256), dtype=torch.float16)),
    ("fp32", lambda hq: torch.empty((0, hq, 256), dtype=torch.float16)),
    ("bf16", lambda hq: torch.empty((0, hq + 1, 256), dtype=torch.bfloat16)[:, 1:]),
    ("fp32", lambda hq: torch.empty((0, hq, 512))[..., :256]),
])
def test_rotary_write_of_no_tokens_into_another_tensor(lib, dtype, out):
    c = case().cache
    x = torch.empty((0, 16, 256), dtype={"fp16": torch.float16, "fp32": torch.float32, "bf16": torch.bfloat16}[dtype])
    n = torch.zeros(0, dtype=torch.int64)
    # (the data of all empty tensors is the null pointer: that does not make query_out the query)
    assert call(lib.pth_cache_write_rotary, describe(x[:, :12], out(12), x[:, 12:14], x[:, 14:], n, torch.zeros((9, 64)), *views(c), n),
                0) == (0, "")


# ---- sizes that 32-bit steps or a launch would not do ----

def weights_args(change):
    c = case()
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    d = dict(zip(("q", "kc", "vc", "ks", "vs", "bt", "lens", "qsl", "lse", "weights"), describe(
        c.q, *views(c.cache), c.block_table, c.seq_lens, c.query_start_loc, torch.zeros((4, 12)), torch.zeros((2, 2, 50)))))
    e = dict(zip(("weights", "kc", "vc", "ks", "vs", "bt", "lens", "nbt", "nlens", "nweights", "kept"), describe(
        torch.zeros((2, 2, 50)), *views(c.cache), c.block_table, c.seq_lens, i32(2, 2), i32(2), torch.zeros((2, 2, 20)), i32(2, 2, 20))))
    for t in (d, e):
        for name, (dim, size) in change.items():
            if name in t:
                rows = 1
                t[name].sizes[dim] = size
                for i in (2, 1, 0) if t[name].ndim == 3 else (1, 0):
                    t[name].strides[i], rows = rows, rows * t[name].sizes[i]
    return d, e


@pytest.mark.parametrize("keys", [(1 << 28) + 1, (1 << 31) - 1])
def test_rows_of_more_keys_than_2_to_the_28(lib, keys):
    d, e = weights_args({"weights": (2, keys)})
    rc, text = call(lib.pth_cache_key_weights, d.values(), ctypes.c_double(0.1), 2, 3)
    assert rc == 1 and "at most 2^28 keys" in text
    rc, text = call(lib.pth_cache_evict, e.values(), 2, 20, 4)
    assert rc == 1 and "at most 2^28 keys" in text
    rc, text = call(lib.pth_cache_evict, weights_args({"nweights": (2, keys)})[1].values(), 2, 20, 4)
    assert rc == 1 and "at most 2^28 keys" in text
    e = weights_args({"nweights": (2, keys), "kept": (2, keys), "nbt": (1, keys)})[1]
    rc, text = call(lib.pth_cache_evict, e.values(), 2, keys, 4)
    assert rc == 1 and "keep must be in [1, 2^28]" in text


# ---- outputs that overlap what the call reads ----

def test_rotary_query_out_over_parts_of_the_inputs(lib):
    c, T = case().cache, 3
    x = torch.zeros((T, 40, 256), dtype=torch.float16)
    flat = torch.zeros(T * 40 * 256 * 2, dtype=torch.float16)
    n, table = torch.zeros(T, dtype=torch.int64), torch.zeros((9, 64))

    def run(q, out, k=x[:, 36:38], v=x[:, 38:]):
        return call(lib.pth_cache_write_rotary, describe(q, out, k, v, n, table, *views(c), n), 0)

    q = x[:, :12]
    for out, msg in (
        (x[:, 1:13], "itself or not overlap"), (x[:, 11:23], "itself or not overlap"),
        (x.view(-1)[4:4 + 2 * 40 * 256 + 12 * 256].as_strided((T, 12, 256), (40 * 256, 256, 1)), "itself or not overlap"),
        (x.as_strided((T, 12, 256), (13 * 256, 256, 1), 13 * 256), "itself or not overlap"),
        (x[:, 25:37], "key or value"), (x[:, 28:40], "key or value"), (x[:, 27:39], "key or value"),
    ):
        rc, text = run(q, out)
        assert rc == 1 and msg in text, (rc, text)
    rc, text = run(q, q, k=x[:, 10:12])
    assert rc == 1 and "key or value" in text                       # in place over the key
    f32 = flat.view(torch.float32)[:T * 40 * 256].view(T, 40, 256)
    rc, text = run(f32[:, :12], flat.view(T, 80, 256)[:, 23:35], f32[:, 36:38], f32[:, 38:])
    assert rc == 1 and "itself or not overlap" in text              # its bytes, though of another type
    # apart: other heads of a buffer, halves of wider rows, another run of tokens, behind the fp32 heads, one token of other strides
    wide = torch.zeros((T, 12, 512), dtype=torch.float16)
    more = torch.zeros((2 * T, 40, 256), dtype=torch.float16)
    for q, out, kv in ((q, x[:, 12:24], x), (x[:, 12:24], x[:, :12], x), (q, q, x), (wide[..., :256], wide[..., 256:], x), (more[:T, :12], more[T:, :12], more[:T]),
                       (f32[:, :12], flat.view(T, 80, 256)[:, 24:36], f32)):
        rc, text = run(q, out, kv[:, 36:38], kv[:, 38:])
        assert rc != 1, text


def test_evict_outputs_over_other_tensors(lib):
    c = case()
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    names = ("weights", "kc", "vc", "ks", "vs", "bt", "lens", "nbt", "nlens", "nweights", "kept")
    good = dict(zip(names, (torch.zeros((2, 2, 50)), *views(c.cache), c.block_table, c.seq_lens, i32(2, 2), i32(2), torch.zeros((2, 2, 20)),
                            i32(2, 2, 20))))
    both, ints = torch.zeros((2, 2, 80)), i32(200)
    run = lambda **kw: call(lib.pth_cache_evict, describe(*[{**good, **kw}[n] for n in names]), 2, 20, 4)  # noqa: E731
    kept = both.view(-1)[:80].view(torch.int32).view(2, 2, 20)
    for kw, msg in (
        (dict(weights=both[..., :50], nweights=both[..., 49:69]), "those that it reads"),
        (dict(weights=both[..., 30:], nweights=both[..., 11:31]), "those that it reads"),
        (dict(weights=both[..., :50], kept=kept), "those that it reads"),
        (dict(nweights=both[..., 60:], kept=both.view(-1)[60:140].view(torch.int32).view(2, 2, 20)), "eviction writes must not overlap"),
        (dict(lens=ints[:2], nlens=ints[1:3]), "those that it reads"),
        (dict(nlens=ints[3:5], kept=ints[4:84].view(2, 2, 20)), "eviction writes must not overlap"),
        (dict(nbt=ints[:4].view(2, 2), nlens=ints[3:5]), "those that it reads"),
        (dict(nbt=ints[80:84].view(2, 2), kept=ints[4:84].view(2, 2, 20)), "those that it reads"),
    ):
        rc, text = run(**kw)
        assert rc == 1 and msg in text, (list(kw), rc, text)
    for kw in ({}, dict(weights=both[..., :50], nweights=both[..., 50:70]), dict(weights=both[..., 30:], nweights=both[..., 10:30]),
               dict(weights=both[:, :, :50], nweights=both[:, :, 55:]), dict(lens=ints[:2], nlens=ints[2:4], kept=ints[4:84].view(2, 2, 20),
                                                                            nbt=ints[84:88].view(2, 2))):
        rc, text = run(**kw)
        assert rc != 1, (list(kw), text)
