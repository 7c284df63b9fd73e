"""fork_pages and compact_pages refuse caches that share bytes with one another or with the tables, without a GPU: which caches do is
compared with every byte of small ones. A cache that is given twice counts once. On the GPU: caches interleaved in one buffer with
their tables beside them, one of them given twice.
"""
import ctypes
import random

import pytest
import torch

import page_oracle
import workload as kvc
from mi50_vllm_lab_amd import pth_dec
from test_pages_host import call_compact, call_fork, i32, strided

ROW = 520


def geometry(rng):
    """Sizes and nested strides of a small cache, its dims in any order, with gaps here and there."""
    sizes = [rng.randint(1, 4), rng.randint(1, 3), rng.randint(1, 4)]
    strides, span = [0, 0, 0], ROW
    for d in rng.sample(range(3), 3):
        strides[d] = span + rng.choice([0, 0, 8, 520, 1040, 3000])
        span += strides[d] * (sizes[d] - 1)
    for d in range(3):
        if sizes[d] == 1:
            strides[d] = rng.choice([0, 8, 520, 80000])
    return sizes, strides


def row_starts(sizes, strides):
    return [a * strides[0] + b * strides[1] + c * strides[2] for a in range(sizes[0]) for b in range(sizes[1]) for c in range(sizes[2])]


def caches_refused(lib, sizes, strides, shifts):
    """Whether the caches alone are why a call fails (the counts' size is wrong, which is looked at after them)."""
    c = (pth_dec.PdTensor * len(shifts))(*[strided(sizes + [ROW], strides + [1], data=1 << 20) for _ in shifts])
    for x, s in zip(c, shifts):
        x.data = (1 << 20) + s
    err = ctypes.create_string_buffer(256)
    wrong = ctypes.byref(pth_dec.describe(i32(77)))
    assert lib.pth_cache_compact_pages(c, len(shifts), *[wrong] * 7, None, err, len(err)) == 1
    assert err.value in (b"the caches' rows must not overlap", b"refs, new_refs and places must be contiguous int32 with an entry for each page")
    return b"caches" in err.value


@pytest.mark.parametrize("seed", range(12))
def test_caches_that_share_bytes(seed):
    lib, rng, found = pth_dec.load_library(), random.Random(seed), [0, 0]
    for _ in range(150):
        sizes, strides = geometry(rng)
        rows = row_starts(sizes, strides)
        for _ in range(6):
            pick = lambda: rng.choice([s for s in strides if s] + [ROW]) * rng.randint(0, 3)  # noqa: E731
            shift = abs(pick() - pick()) + rng.choice([0, 0, 8, 512, 520, 528])
            if shift == 0:
                continue
            meet = any(abs(x + shift - y) < ROW for x in rows for y in rows)
            assert caches_refused(lib, sizes, strides, [0, shift]) == meet, (sizes, strides, shift)
            assert caches_refused(lib, sizes, strides, [shift, 1 << 24, 0]) == meet
            found[meet] += 1
    assert min(found) > 100


def test_layers_side_by_side_and_a_cache_given_twice():
    lib = pth_dec.load_library()
    sizes, page = [30, 2, 16], 2 * 16 * ROW
    for layers in (2, 128):
        inside = [layers * page, 16 * ROW, ROW]                       # [pages, layers, heads, keys]
        assert not caches_refused(lib, sizes, inside, [i * page for i in range(layers)])
        assert caches_refused(lib, sizes, inside, [i * page - (8 if i == layers - 1 else 0) for i in range(layers)])
    own = [page, 16 * ROW, ROW]
    assert not caches_refused(lib, sizes, own, [0, 30 * page, 0, 30 * page])
    assert caches_refused(lib, sizes, own, [0, 29 * page])


@pytest.mark.parametrize("call,names", [(call_fork, ("refs", "table", "lens", "parents", "new_refs", "new_table", "new_lens", "needed", "ws")),
                                        (call_compact, ("refs", "table", "new_refs", "new_table", "places", "used", "ws"))])
def test_tables_over_a_cache(call, names):
    lib = pth_dec.load_library()
    kv = kvc.allocate_cache(40, 16, 2).kv
    flat = kv.view(-1).view(torch.int32)
    for name in names:
        for at in (0, flat.numel() // 2 // 4 * 4, -1):
            def over(a, name=name, at=at):
                n = a[name].numel()
                return (flat[at:at + n] if at >= 0 else flat[(flat.numel() - n) // 4 * 4:][:n]).view(a[name].shape)

            for caches in ([kv], [kv, kv.clone()], [kv.clone(), kv]):
                rc, text = call(lib, **{"caches": caches, name: over})
                assert (rc, text) == (1, "the caches must not overlap the other tensors"), (name, at, rc, text)


@pytest.mark.gpu
@pytest.mark.parametrize("seed", range(6))
def test_interleaved_layers_beside_their_tables(seed):
    rng = random.Random(seed)
    bs, hkv, pages, layers, rows, cols = 8, 2, 30, 3, 4, 5
    page = hkv * bs * ROW
    pool = torch.randint(-128, 128, (pages * layers * page + 4 * 400,), dtype=torch.int8, device="cuda",
                         generator=torch.Generator(device="cuda").manual_seed(seed))
    kvs = [pool[:pages * layers * page].view(pages, layers, hkv, bs, ROW)[:, i] for i in range(layers)]
    ints = pool[pages * layers * page:].view(torch.int32)
    lens = [rng.randint(0, cols * bs - 3) for _ in range(rows)]
    free, refs, table = rng.sample(range(pages), pages), [0] * pages, [[-1] * cols for _ in range(rows)]
    for b, n in enumerate(lens):
        for c in range(-(-n // bs)):
            table[b][c] = free.pop()
            refs[table[b][c]] = 1
    parents = [rng.randrange(rows) for _ in range(5)]
    want = page_oracle.fork(refs, table, lens, parents, cols, bs, grow=1)
    old = [k.clone() for k in kvs]
    at = 0

    def take(*shape):
        nonlocal at
        n = torch.Size(shape).numel()
        at += n
        return ints[at - n:at].view(shape)

    r, t, s, p = take(pages), take(rows, cols), take(rows), take(5)
    for x, v in ((r, refs), (t, table), (s, lens), (p, parents)):
        x.copy_(torch.tensor(v, dtype=torch.int32))
    nt, ns, nr, need = take(5, cols), take(5), take(pages), take(1)
    pth_dec.fork_pages([*kvs, kvs[1]], r, t, s, p, nr, nt, ns, need, grow=1)
    torch.cuda.synchronize()
    assert (nt.tolist(), ns.tolist(), nr.tolist(), need.tolist()[0]) == tuple(want[:4])
    for k, o in zip(kvs, old):
        for src, dst, keys in want[4]:
            o[dst, :, :keys] = o[src, :, :keys]
        assert torch.equal(k, o)
    # and packed, the same cache twice
    want = page_oracle.compact(nr.tolist(), nt.tolist())
    before, places, used = [k.clone() for k in kvs], i32(pages).cuda(), i32(1).cuda()
    live = [i for i, x in enumerate(nr.tolist()) if x > 0]
    pth_dec.compact_pages([kvs[0], *kvs], nr, nt, nr, nt, places, used)
    torch.cuda.synchronize()
    assert (nt.tolist(), nr.tolist(), places.tolist(), used.tolist()[0]) == tuple(want)
    for k, o in zip(kvs, before):
        for i in live:
            assert torch.equal(k[want[2][i]], o[i])
