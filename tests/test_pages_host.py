"""norm_rotary_cache_write, fork_pages and compact_pages without a GPU: what their entries refuse and with which message, empty calls,
workspace sizes, the Python face on host tensors, and the lists that the GPU tests compare with on states worked out by hand.
"""
import ctypes

import pytest
import torch

import page_oracle
import workload as kvc
from mi50_vllm_lab_amd import pth_dec


@pytest.fixture(scope="module")
def lib():
    return pth_dec.load_library()


def ref(t):
    return None if t is None else ctypes.byref(t if isinstance(t, pth_dec.PdTensor) else pth_dec.describe(t))


def i32(*s):
    return torch.zeros(s, dtype=torch.int32)


def many(caches):
    return (pth_dec.PdTensor * max(1, len(caches)))(*[pth_dec.describe(c) for c in caches])


def call_fork(lib, **change):
    kv = kvc.allocate_cache(40, 16, 2).kv
    a = dict(caches=[kv, kv.clone()], refs=i32(40), table=i32(3, 7), lens=i32(3), parents=i32(5), new_refs=i32(40), new_table=i32(5, 7),
             new_lens=i32(5), needed=i32(1), ws=i32(lib.pth_cache_pages_workspace(40, 3, 5)), grow=1, window=-1, sinks=0, layers=None)
    assert set(change) <= set(a)
    a.update({k: v(a) if callable(v) else v for k, v in change.items()})
    err = ctypes.create_string_buffer(256)
    caches = None if a["caches"] is None else many(a["caches"])
    layers = a["layers"] if a["layers"] is not None else len(a["caches"] or [])
    rc = lib.pth_cache_fork_pages(caches, layers, *[ref(a[k]) for k in ("refs", "table", "lens", "parents", "new_refs", "new_table",
                                                                          "new_lens", "needed", "ws")], a["grow"], a["window"],
                                  a["sinks"], None, err, len(err))
    return rc, err.value.decode()


def call_compact(lib, **change):
    kv = kvc.allocate_cache(40, 16, 2).kv
    a = dict(caches=[kv], refs=i32(40), table=i32(3, 7), new_refs=i32(40), new_table=i32(3, 7), places=i32(40), used=i32(1),
             ws=i32(lib.pth_cache_pages_workspace(40, 0, 0)), layers=None)
    assert set(change) <= set(a)
    a.update({k: v(a) if callable(v) else v for k, v in change.items()})
    err = ctypes.create_string_buffer(256)
    caches = None if a["caches"] is None else many(a["caches"])
    layers = a["layers"] if a["layers"] is not None else len(a["caches"] or [])
    rc = lib.pth_cache_compact_pages(caches, layers, *[ref(a[k]) for k in ("refs", "table", "new_refs", "new_table", "places", "used",
                                                                             "ws")], None, err, len(err))
    return rc, err.value.decode()


def strided(sizes, strides, dtype=pth_dec.PD_DTYPE_INT8, data=4096):
    """A view that is described, never read."""
    d = pth_dec.PdTensor()
    d.data, d.dtype, d.ndim = data, dtype, len(sizes)
    for i, (n, s) in enumerate(zip(sizes, strides)):
        d.sizes[i], d.strides[i] = n, s
    return d


BAD_CACHES = [
    (dict(caches=None), "null tensor descriptor"),
    (dict(caches=[]), "1 to 128 caches"),
    (dict(layers=129), "1 to 128 caches"),
    (dict(caches=lambda a: [a["caches"][0].view(torch.uint8)]), "caches must be int8"),
    (dict(caches=lambda a: [a["caches"][0][..., :260]]), "caches must be int8"),
    (dict(caches=lambda a: [a["caches"][0][0]]), "caches must be int8"),
    (dict(caches=lambda a: [a["caches"][0].view(-1)[4:4 + 39 * 2 * 16 * 520].view(39, 2, 16, 520)]), "caches must be int8"),
    (dict(caches=lambda a: [a["caches"][0], kvc.allocate_cache(41, 16, 2).kv]), "same sizes and strides"),
    (dict(caches=lambda a: [a["caches"][0], kvc.allocate_cache(40, 16, 2, "NHD").kv]), "same sizes and strides"),
    (dict(caches=lambda a: [a["caches"][0][:1].expand(40, 2, 16, 520)]), "rows must not overlap"),
    (dict(caches=lambda a: [a["caches"][0].as_strided((40, 2, 16, 520), (16640, 512, 1040, 1))]), "rows must not overlap"),
    (dict(caches=lambda a: [a["caches"][0].as_strided((30, 2, 16, 520), (16640 - 520, 8320, 520, 1))]), "rows must not overlap"),
]


def test_fork_refusals(lib):
    cases = BAD_CACHES + [({n: None}, "null tensor descriptor") for n in ("refs", "table", "lens", "new_refs", "new_table", "new_lens",
                                                                         "needed", "ws")] + [
        (dict(refs=i32(39)), "an entry for each page"),
        (dict(refs=i32(41)), "an entry for each page"),
        (dict(new_refs=i32(40).long()), "an entry for each page"),
        (dict(new_refs=i32(80)[::2]), "an entry for each page"),
        (dict(table=i32(3, 7).long()), "block tables must be"),
        (dict(table=i32(7, 3).t()), "block tables must be"),
        (dict(table=i32(3, 8)), "same columns"),
        (dict(table=i32(8193, 7), lens=i32(8193)), "at most 8192 rows"),
        (dict(new_table=i32(8193, 7)), "at most 8192 rows"),
        (dict(lens=i32(2)), "an entry for each row"),
        (dict(lens=i32(3).long()), "an entry for each row"),
        (dict(new_lens=i32(4)), "an entry for each row"),
        (dict(parents=i32(4)), "an entry for each new row"),
        (dict(parents=i32(5).long()), "an entry for each new row"),
        (dict(parents=None), "an entry for each new row"),
        (dict(needed=i32(0)), "needed must be"),
        (dict(grow=-1), "at least 0"),
        (dict(sinks=-1), "at least 0"),
        (dict(grow=1 << 31), "fit in 32 bits"),
        (dict(window=1 << 31), "fit in 32 bits"),
        (dict(new_table=i32(1, 7).expand(5, 7)), "rows must not overlap"),
        (dict(new_table=i32(40).as_strided((5, 7), (6, 1))), "rows must not overlap"),
        (dict(new_table=lambda a: a["table"][:3], new_lens=i32(3), parents=i32(3)), "must not overlap the old ones"),
        (dict(new_lens=lambda a: a["parents"]), "must not overlap"),
        (dict(new_refs=lambda a: a["refs"][:40], needed=lambda a: a["refs"][3:4]), "must not overlap"),
        (dict(needed=lambda a: a["new_lens"][1:2]), "must not overlap"),
        (dict(ws=lambda a: a["ws"][:-1]), "workspace must be"),
        (dict(ws=lambda a: torch.zeros(a["ws"].numel() + 1, dtype=torch.int32)[1:]), "workspace must be"),
        (dict(ws=lambda a: a["ws"].float()), "workspace must be"),
    ]
    for change, msg in cases:
        rc, text = call_fork(lib, **change)
        assert rc == 1 and msg in text, (list(change), rc, text)


def test_old_tensors_as_the_new_ones_need_rows_that_keep_their_places(lib):
    one = i32(100)
    rc, text = call_fork(lib, parents=None, new_table=lambda a: one[7:28].view(3, 7), table=one[:21].view(3, 7), new_lens=i32(3))
    assert rc == 1 and "the old ones or not overlap" in text
    rc, text = call_fork(lib, parents=None, new_table=i32(3, 7), new_lens=lambda a: one[1:4], lens=one[:3])
    assert rc == 1 and "the old ones or not overlap" in text


def test_compact_refusals(lib):
    cases = BAD_CACHES + [({n: None}, "null tensor descriptor") for n in ("refs", "table", "new_refs", "new_table", "places", "used",
                                                                         "ws")] + [
        (dict(refs=i32(39)), "an entry for each page"),
        (dict(places=i32(39)), "an entry for each page"),
        (dict(places=i32(40).long()), "an entry for each page"),
        (dict(new_table=i32(4, 7)), "same rows and columns"),
        (dict(new_table=i32(3, 8)), "same rows and columns"),
        (dict(used=i32(0)), "used must be"),
        (dict(new_table=i32(1, 7).expand(3, 7)), "rows must not overlap"),
        (dict(new_refs=lambda a: a["refs"], places=lambda a: a["refs"]), "must not overlap"),
        (dict(table=lambda a: a["new_table"].view(7, 3).as_strided((3, 7), (5, 1))), "the old ones or not overlap"),
        (dict(ws=lambda a: a["ws"][:-1]), "workspace must be"),
    ]
    for change, msg in cases:
        rc, text = call_compact(lib, **change)
        assert rc == 1 and msg in text, (list(change), rc, text)


def test_pools_and_rows_beyond_the_limits(lib):
    """Described, never read."""
    err = ctypes.create_string_buffer(256)
    for sizes, strides in (([(1 << 22) + 1, 1, 1, 520], [520, 520, 520, 1]), ([2, 1 << 11, 1 << 10, 520], [520 << 21, 520, 520 << 11, 1]),
                           ([0, 1, 1, 520], [520, 520, 520, 1])):
        c = (pth_dec.PdTensor * 1)(strided(sizes, strides))
        rc = lib.pth_cache_compact_pages(c, 1, *[ref(i32(1)) for _ in range(7)], None, err, len(err))
        assert rc == 1 and b"2^22 pages" in err.value
    w = lib.pth_cache_pages_workspace
    assert w(0, 1, 1) == 0 and w((1 << 22) + 1, 1, 1) == 0 and w(1, -1, 1) == 0
    assert w(1, 0, 0) == 66 and w(1025, 3, 5) == 2 * 65 + 3 + 20 + 1


def test_more_entries_than_32_bits_count(lib):
    cols = 2 ** 30 - 1
    table = lambda rows: strided((rows, cols), (cols, 1), pth_dec.PD_DTYPE_INT32)  # noqa: E731
    assert call_fork(lib, table=table(3), new_table=table(5)) == (1, "at most 2^31 - 1 entries in the new block table")


def test_norm_rotary_refusals(lib):
    c = kvc.make_case([37, 5], [3, 1], num_q_heads=12, num_kv_heads=2, block_size=16, seed=3).cache
    x = torch.zeros((3, 17, 256), dtype=torch.float16)
    names = ("query", "query_out", "key", "value", "qw", "kw", "positions", "cos_sin", "kc", "vc", "ks", "vs", "slots")
    good = dict(query=x[:, :12], query_out=x[:, :12], key=x[:, 12:14], value=x[:, 14:16], qw=x[0, 16], kw=x[1, 16],
                positions=torch.zeros(3, dtype=torch.int64), cos_sin=torch.zeros((9, 64)), kc=c.key_cache, vc=c.value_cache,
                ks=c.k_scale, vs=c.v_scale, slots=torch.zeros(3, dtype=torch.int64))
    inf = float("inf")
    cases = [({n: None}, "null tensor descriptor") for n in names] + [
        (dict(qw=torch.zeros(256).double()), "query_weight and key_weight"),
        (dict(qw=torch.zeros(256)), "query_weight and key_weight"),          # one dtype for both
        (dict(qw=torch.zeros(256).bfloat16(), kw=torch.zeros(256).bfloat16()), "query_weight and key_weight"),
        (dict(kw=torch.zeros(255).half()), "query_weight and key_weight"),
        (dict(kw=torch.zeros((1, 256)).half()), "query_weight and key_weight"),
        (dict(kw=torch.zeros(512).half()[::2]), "query_weight and key_weight"),
        (dict(kw=torch.zeros(257).half()[1:]), "query_weight and key_weight"),
        (dict(qw=x[1, 3]), "query_out must not overlap the weights"),
        (dict(query_out=x[:, 1:13]), "itself or not overlap"),
        (dict(value=x[:, 14:16].float()), "fp16, bf16 or fp32"),
        (dict(eps=-1e-6), "eps must be"), (dict(eps=inf), "eps must be"), (dict(eps=float("nan")), "eps must be"),
        (dict(offset=inf), "eps must be"), (dict(offset=float("nan")), "eps must be"),
        (dict(cos_sin=torch.zeros((9, 60))), "cos_sin must be"),
    ]
    err = ctypes.create_string_buffer(256)
    for change, msg in cases:
        t = {**good, "eps": 1e-6, "offset": 0.0, **change}
        d = [ref(t[n]) for n in names]
        rc = lib.pth_cache_write_norm_rotary(*d[:6], t["eps"], t["offset"], *d[6:], 0, None, err, len(err))
        assert rc == 1 and msg in err.value.decode(), (list(change), rc, err.value)
    none = {k: v[:0] if k in ("query", "query_out", "key", "value", "positions", "slots") else v for k, v in good.items()}
    d = [ref(none[n]) for n in names]
    assert lib.pth_cache_write_norm_rotary(*d[:6], 1e-6, 0.0, *d[6:], 0, None, err, len(err)) == 0


def test_host_tensors_are_refused():
    kv, t = kvc.allocate_cache(4, 16, 2).kv, i32(3, 7)
    with pytest.raises(RuntimeError, match="on one GPU"):
        pth_dec.fork_pages([kv], i32(4), t, i32(3), None, i32(4), t, i32(3), i32(1))
    with pytest.raises(RuntimeError, match="on one GPU"):
        pth_dec.compact_pages([kv], i32(4), t, i32(4), t, i32(4), i32(1))
    with pytest.raises(TypeError):
        pth_dec.compact_pages([3], i32(4), t, i32(4), t, i32(4), 7)
    x = torch.zeros((3, 8, 256), dtype=torch.float16)
    c = kvc.allocate_cache(4, 16, 2)
    with pytest.raises(RuntimeError, match="on one GPU"):
        pth_dec.norm_rotary_cache_write(x, x[:, :2], x[:, 2:4], x[0, 0], x[0, 1], i32(3).long(), torch.zeros((9, 64)), c.key_cache,
                                        c.value_cache, c.k_scale, c.v_scale, i32(3).long())


def test_lists_by_hand():
    f = page_oracle.fork
    # one row of 5 keys in pages of 4, room for 4 more: page 7 goes on, one page is taken
    assert f([0, 0, 1, 0, 0, 0, 0, 1], [[2, 7, -1, -1]], [5], None, 4, 4, grow=4) == (
        [[2, 7, 0, -1]], [5], [1, 0, 1, 0, 0, 0, 0, 1], 1, [])
    # both children share page 2; the second copies page 7's one key
    assert f([0, 0, 1, 0, 0, 0, 0, 1], [[2, 7, -1, -1]], [5], [0, 0], 4, 4) == (
        [[2, 7, -1, -1], [2, 0, -1, -1]], [5, 5], [1, 0, 2, 0, 0, 0, 0, 1], 1, [(7, 0, 1)])
    # the row ends, an empty one begins
    assert f([0, 0, 1, 0, 0, 0, 0, 1], [[2, 7, -1, -1]], [5], [-1], 4, 4, grow=3) == ([[-1] * 4], [0], [0] * 8, 0, [])
    assert page_oracle.compact([0, 1, 0, 2, 1], [[3, -1, 4], [3, 1, 2]]) == ([[0, -1, 2], [0, 1, -1]], [2, 1, 1, 0, 0], [-1, 1, -1, 0, 2], 3)
