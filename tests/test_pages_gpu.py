"""fork_pages and compact_pages on the GPU against lists (tests/page_oracle.py), every table entry, count and cache byte: random
pools and tables with holes, entries that name no page, shared and part-filled pages; rows that fork, end, are empty or go on; room
for no, a few and thousands of keys; more pages wanted than free; block sizes 1 to 1,584, both layouts, rows with gaps, pages
whose copies are not 16-byte aligned; pools beyond one count; in place, on another stream and in a captured graph.
"""
import random

import pytest
import torch

import page_oracle
import workload as kvc
from mi50_vllm_lab_amd import pth_dec

pytestmark = pytest.mark.gpu


def i32(x, shape=None):
    t = torch.tensor(x, dtype=torch.int32)
    return (t.view(shape) if shape else t).cuda()


def raw_caches(layers, pages, hkv, bs, layout, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    make = lambda *s: torch.randint(-128, 128, s, dtype=torch.int8, device="cuda", generator=g)  # noqa: E731
    if layout == "HND":
        return [make(pages, hkv, bs, 520) for _ in range(layers)]
    if layout == "NHD":
        return [make(pages, bs, hkv, 520).transpose(1, 2) for _ in range(layers)]
    if layout == "gaps":      # rows apart, in no dense order
        return [make(pages, hkv + 1, bs, 528)[:, :hkv, :, 8:] for _ in range(layers)]
    return [make(pages, hkv, bs + 1, 520)[:, :, :bs] for _ in range(layers)]  # heads apart


def pool(rng, rows, pages, cols, bs, holes=0.2, shared=0.2, odd=0.05):
    """(counts, table, lengths) of a random state: pages that rows share, holes, entries that name no page, rows longer or shorter
    than their entries."""
    order = rng.sample(range(pages), pages)
    table = []
    for _ in range(rows):
        row = []
        for _ in range(cols):
            x = rng.random()
            if x < holes or not order:
                row.append(-1)
            elif x < holes + odd:
                row.append(rng.choice([-7, pages, pages + 3, 2 ** 31 - 1]))
            elif x < holes + odd + shared and any(e >= 0 for r in table for e in r if e < pages):
                row.append(rng.choice([e for r in table for e in r if 0 <= e < pages]))
            else:
                row.append(order.pop())
        table.append(row)
    refs = [0] * pages
    for row in table:
        for e in row:
            if 0 <= e < pages:
                refs[e] += 1
    for p in rng.sample(range(pages), pages // 10):  # named by tables that are not here
        refs[p] += 1
    lens = [rng.choice([-3, 0, 1, bs - 1, bs, rng.randint(0, cols * bs), cols * bs, cols * bs + 5]) for _ in range(rows)]
    return refs, table, lens


def run_fork(caches, refs, table, lens, parents, cols, bs, grow, window, sinks, in_place=False):
    rows = len(table) if parents is None else len(parents)
    t = [i32(refs), i32(table, (len(table), cols)), i32(lens)]
    par = None if parents is None else i32(parents)
    new = t if in_place else [torch.full_like(t[0], 99), torch.full((rows, cols), 99, dtype=torch.int32, device="cuda"),
                              torch.full((rows,), 99, dtype=torch.int32, device="cuda")]
    needed = torch.full((1,), 99, dtype=torch.int32, device="cuda")
    pth_dec.fork_pages(caches, t[0], t[1], t[2], par, new[0], new[1], new[2], needed, grow=grow, window=window, sinks=sinks)
    torch.cuda.synchronize()
    if not in_place:
        assert t[0].tolist() == list(refs) and t[1].tolist() == [list(r) for r in table] and t[2].tolist() == list(lens)
    return new[1].tolist(), new[2].tolist(), new[0].tolist(), int(needed)


def check_fork(caches, refs, table, lens, parents, cols, bs, grow=0, window=-1, sinks=0, in_place=False):
    want = page_oracle.fork(refs, table, lens, parents, cols, bs, grow, window, sinks)
    expected = [kv.clone() for kv in caches]
    for kv in expected:
        for a, b, keys in want[4]:
            kv[b, :, :keys] = kv[a, :, :keys]
    got = run_fork(caches, refs, table, lens, parents, cols, bs, grow, window, sinks, in_place)
    assert got == want[:4]
    for kv, x in zip(caches, expected):
        assert torch.equal(kv, x)
    return want


@pytest.mark.parametrize("seed", range(40))
def test_fork_of_random_pools(seed):
    rng = random.Random(seed)
    bs = rng.choice([1, 3, 16, 16, 32, 1584])
    hkv, layout = rng.choice([(4, "HND"), (2, "NHD"), (1, "HND"), (3, "gaps"), (2, "heads")])
    pages = rng.choice([1, 7, 63, 64, 65, 200, 1023, 1024, 1025, 2500]) if bs < 100 else rng.choice([3, 20])
    rows, cols = rng.choice([1, 2, 9, 40, 300]), rng.choice([1, 2, 5, 30, 260])
    if rows * cols > 4000:
        rows = max(1, 4000 // cols)
    refs, table, lens = pool(rng, rows, pages, cols, bs, shared=rng.choice([0.0, 0.3]))
    parents = None if rng.random() < 0.4 else [rng.choice([-1, -5, rows, 2 ** 31 - 1] + [rng.randrange(rows)] * 20)
                                               for _ in range(rng.choice([1, 3, rows, 2 * rows, 257]))]
    grow, sinks = rng.choice([0, 1, bs, 3 * bs + 1, cols * bs]), rng.choice([0, 1, bs, 2 * bs + 1])
    window = rng.choice([-1, 0, 1, bs, 2 * bs + 1, cols * bs // 2 + 1])
    caches = raw_caches(rng.choice([1, 3]), pages, hkv, bs, layout, seed)
    check_fork(caches, refs, table, lens, parents, cols, bs, grow, window, sinks, in_place=parents is None and rng.random() < 0.5)


@pytest.mark.parametrize("in_place", [False, True])
def test_counts_below_zero_are_free_pages(in_place):
    """A page that is taken is counted from 0, whatever said that it was free, and no second call takes it again."""
    refs, table, lens = [-3, 1, -1, 0, -2 ** 31, 1, -2], [[1, -1, -1], [5, -1, -1]], [16, 20]
    caches = raw_caches(1, 7, 2, 16, "HND", 3)
    new_table, new_lens, counts, wanted, _ = check_fork(caches, refs, table, lens, None, 3, 16, grow=1, in_place=in_place)
    assert counts == [1, 1, 1, 0, 0, 1, 0] and wanted == 2
    again = check_fork(caches, counts, new_table, [32, 32], None, 3, 16, grow=1, in_place=in_place)
    assert sorted(e for row in again[0] for e in row if e >= 0) == [0, 1, 2, 3, 4, 5]


def test_fork_takes_thousands_of_pages():
    """Rows that take more pages than a workgroup has threads, across many counts of 1,024."""
    rng = random.Random(1)
    pages, cols = 9000, 1500
    refs, table, lens = [rng.choice([0, 0, 1]) for _ in range(pages)], [[-1] * cols for _ in range(3)], [0, 0, 0]
    caches = raw_caches(1, pages, 1, 1, "HND", 0)
    want = check_fork(caches, refs, table, lens, [2, 0, 1, 2], cols, 1, grow=1400)
    assert want[3] == 4 * 1400
    refs = [1] * (pages - 700) + [0] * 700  # fewer than wanted: the last columns stay empty
    want = check_fork(caches, refs, table, lens, None, cols, 1, grow=600)
    assert want[3] == 1800 and want[0][1][99] == pages - 1 and want[0][1][100] == -1


def test_children_of_one_parent():
    """The first child goes on in the part-filled page, the others in copies; a page that another table names too is copied for all."""
    bs, cols = 16, 4
    refs = [1] * 6 + [0] * 10
    table, lens = [[3, 1, -1, -1], [2, 0, 5, -1]], [21, 35]
    caches = raw_caches(2, 16, 4, bs, "HND", 3)
    want = check_fork(caches, refs, table, lens, [1, 0, 1, 1], cols, bs, grow=1)
    assert want[0] == [[2, 0, 5, -1], [3, 1, -1, -1], [2, 0, 6, -1], [2, 0, 7, -1]]
    refs[5] = 2
    want = check_fork(caches, refs, table, lens, [1, 0, 1, 1], cols, bs, grow=1)
    assert want[0][0] == [2, 0, 6, -1] and want[2][5] == 1


def test_pages_behind_the_window_are_given_back():
    """A row of 100 keys, window 33, 5 sinks, pages of 16: its next token, at position 100, sees keys 68 .. 100, so pages 1, 2 and
    3 go; page 0 holds the sinks."""
    refs, table = [1] * 7 + [0] * 3, [[0, 1, 2, 3, 4, 5, 6, -1]]
    caches = raw_caches(1, 10, 2, 16, "NHD", 3)
    want = check_fork(caches, refs, table, [100], None, 8, 16, grow=1, window=33, sinks=5)
    assert want[0] == [[0, -1, -1, -1, 4, 5, 6, -1]] and want[2] == [1, 0, 0, 0, 1, 1, 1, 0, 0, 0]
    want = check_fork(caches, refs, table, [100], None, 8, 16, grow=1, window=37, sinks=5)   # sees 64: page 4's first key
    assert want[0] == [[0, -1, -1, -1, 4, 5, 6, -1]]
    want = check_fork(caches, refs, table, [100], None, 8, 16, grow=1, window=38, sinks=0)   # sees 63: page 3's last key
    assert want[0] == [[-1, -1, -1, 3, 4, 5, 6, -1]]


@pytest.mark.parametrize("rows,parents", [(0, None), (0, [0, 1]), (3, [])])
def test_fork_without_rows(rows, parents):
    """No old rows: new rows are empty. No new rows: every old row ends."""
    table = [[0, 2, -1], [1, -1, -1], [4, 0, 3]][:rows]
    refs = [2, 1, 1, 1, 1, 0] if rows else [1] * 6
    check_fork(raw_caches(1, 6, 1, 4, "HND", 2), refs, table, [5, 6, 7][:rows], parents, 3, 4, grow=2)


def test_steps_in_a_captured_graph():
    """A graph of one step in place, replayed: every row grows by a key a step and loses the pages that its window has left."""
    bs, cols, rows, pages, window, sinks = 4, 12, 5, 70, 9, 3
    refs, table, lens = [0] * pages, [[-1] * cols for _ in range(rows)], [0, 1, 7, 8, 20]
    caches = raw_caches(1, pages, 2, bs, "HND", 9)
    table, _, refs, _, _ = page_oracle.fork(refs, table, [0] * rows, None, cols, bs, grow=20)
    t = [i32(refs), i32(table, (rows, cols)), i32(lens)]
    needed = torch.zeros(1, dtype=torch.int32, device="cuda")
    one = torch.ones(rows, dtype=torch.int32, device="cuda")

    def step():
        pth_dec.fork_pages(caches, t[0], t[1], t[2], None, t[0], t[1], t[2], needed, grow=1, window=window, sinks=sinks)

    keep = [x.clone() for x in t]
    step()  # (loads the code before the capture)
    for x, y in zip(t, keep):
        x.copy_(y)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for _ in range(20):
        table, lens, refs, wanted, _ = page_oracle.fork(refs, table, lens, None, cols, bs, 1, window, sinks)
        graph.replay()
        torch.cuda.synchronize()
        assert (t[1].tolist(), t[2].tolist(), t[0].tolist(), int(needed)) == (table, lens, refs, wanted)
        t[2].add_(one)
        lens = [n + 1 for n in lens]


def test_the_largest_pool():
    """4,194,304 pages (of one 520-byte row): as many counts as the prefix holds."""
    pages = 1 << 22
    g = torch.Generator(device="cuda").manual_seed(0)
    kv = torch.randint(-128, 128, (pages, 1, 1, 520), dtype=torch.int8, device="cuda", generator=g)
    refs = (torch.rand(pages, device="cuda", generator=g) < 0.6).int()
    free = (refs == 0).nonzero()[:, 0]
    rows, cols = 40, 60000
    table = torch.full((rows, cols), -1, dtype=torch.int32, device="cuda")
    lens = torch.zeros(rows, dtype=torch.int32, device="cuda")
    new, needed = (torch.empty_like(refs), torch.empty_like(table), torch.empty_like(lens)), torch.zeros(1, dtype=torch.int32, device="cuda")
    pth_dec.fork_pages([kv], refs, table, lens, None, *new, needed, grow=cols)
    want = torch.full((rows * cols,), -1, dtype=torch.int32, device="cuda")
    n = min(free.numel(), rows * cols)
    want[:n] = free[:n].int()
    assert int(needed) == rows * cols and free.numel() < rows * cols  # (more than there are)
    assert torch.equal(new[1].view(-1), want)
    counts = refs.clone()
    counts[free[:n]] = 1
    assert torch.equal(new[0], counts)
    # compaction of the pool as it was, with tables that name some of its pages
    live = (refs > 0).nonzero()[:, 0]
    used, moved = live.numel(), int((live >= live.numel()).sum())
    table[:, ::3] = live[torch.randint(0, used, table[:, ::3].shape, device="cuda", generator=g)].int()
    places = torch.full((pages,), -1, dtype=torch.int32, device="cuda")
    places[live[:used - moved]] = live[:used - moved].int()
    places[live[used - moved:]] = free[:moved].int()
    rows_want = kv.clone()
    rows_want[free[:moved]] = kv[live[used - moved:]]
    got, count = torch.empty_like(places), torch.zeros(1, dtype=torch.int32, device="cuda")
    pth_dec.compact_pages([kv], refs, table, new[0], new[1], got, count)
    assert int(count) == used and torch.equal(got, places) and torch.equal(kv, rows_want)
    assert torch.equal(new[1], torch.where(table >= 0, places[table.clamp(min=0).long()], -1))
    assert torch.equal(new[0], (torch.arange(pages, device="cuda") < used).int())


def test_two_streams_at_once():
    rng = random.Random(4)
    states = [pool(rng, 40, 1500, 30, 16) for _ in range(2)]
    want = [page_oracle.fork(*s, None, 30, 16, 9, 100, 4) for s in states]
    caches = [raw_caches(2, 1500, 2, 16, "HND", i) for i in range(2)]
    ts = [[i32(s[0]), i32(s[1], (40, 30)), i32(s[2])] for s in states]
    new = [[torch.zeros_like(x) for x in t] for t in ts]
    needed = [torch.zeros(1, dtype=torch.int32, device="cuda") for _ in ts]
    streams = [torch.cuda.Stream() for _ in ts]
    torch.cuda.synchronize()
    for _ in range(20):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                pth_dec.fork_pages(caches[k], *ts[k], None, *new[k], needed[k], grow=9, window=100, sinks=4)
    torch.cuda.synchronize()
    for k in range(2):
        assert (new[k][1].tolist(), new[k][2].tolist(), new[k][0].tolist(), int(needed[k])) == want[k][:4]


def check_compact(caches, refs, table, cols, in_place=False):
    table_want, counts, places, used = page_oracle.compact(refs, table)
    expected = [kv.clone() for kv in caches]
    for p, to in enumerate(places):
        if to >= 0 and to != p:
            for kv, x in zip(expected, caches):
                kv[to] = x[p]
    r, t = i32(refs), i32(table, (len(table), cols))
    new = (r, t) if in_place else (torch.full_like(r, 99), torch.full_like(t, 99))
    got_places, got_used = torch.full_like(r, 99), torch.full((1,), 99, dtype=torch.int32, device="cuda")
    pth_dec.compact_pages(caches, r, t, *new, got_places, got_used)
    torch.cuda.synchronize()
    assert (new[1].tolist(), new[0].tolist(), got_places.tolist(), int(got_used)) == (table_want, counts, places, used)
    for kv, x in zip(caches, expected):
        assert torch.equal(kv, x)


@pytest.mark.parametrize("seed", range(30))
def test_compact_of_random_pools(seed):
    rng = random.Random(100 + seed)
    bs = rng.choice([1, 3, 16, 32, 1584])
    hkv, layout = rng.choice([(4, "HND"), (2, "NHD"), (1, "HND"), (3, "gaps"), (2, "heads")])
    pages = rng.choice([1, 7, 63, 64, 65, 200, 1023, 1024, 1025, 2500]) if bs < 100 else rng.choice([3, 20])
    rows, cols = rng.choice([0, 1, 9, 40]), rng.choice([1, 5, 30, 260])
    refs, table, _ = pool(rng, rows, pages, cols, bs)
    if seed % 7 == 0:
        refs = [0] * pages
    if seed % 7 == 1:
        refs = [max(1, r) for r in refs]
    check_compact(raw_caches(rng.choice([1, 3]), pages, hkv, bs, layout, seed), refs, table, cols, in_place=rng.random() < 0.5)


def test_compact_of_the_lower_and_the_upper_half():
    for refs in ([1] * 1500 + [0] * 1500, [0] * 1500 + [3] * 1500):
        table = [list(range(1500 * (refs[0] == 0), 1500 * (refs[0] == 0) + 1500))]
        check_compact(raw_caches(1, 3000, 1, 2, "HND", 0), refs, table, 1500)


def test_compact_in_a_captured_graph():
    rng = random.Random(8)
    states = [pool(rng, 9, 1300, 30, 4) for _ in range(3)]
    caches = raw_caches(2, 1300, 2, 4, "HND", 1)
    r, t = i32(states[0][0]), i32(states[0][1], (9, 30))
    places, used = torch.zeros_like(r), torch.zeros(1, dtype=torch.int32, device="cuda")
    out = torch.zeros_like(r), torch.zeros_like(t)
    pth_dec.compact_pages(caches, r, t, *out, places, used)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        pth_dec.compact_pages(caches, r, t, *out, places, used)
    for refs, table, _ in states:
        r.copy_(i32(refs))
        t.copy_(i32(table, (9, 30)))
        before = [kv.clone() for kv in caches]
        graph.replay()
        torch.cuda.synchronize()
        want = page_oracle.compact(refs, table)
        assert (out[1].tolist(), out[0].tolist(), places.tolist(), int(used)) == want
        for kv, x in zip(caches, before):
            for p, to in enumerate(want[2]):
                if to >= 0 and to != p:
                    x[to] = x[p]
            assert torch.equal(kv, x)


def test_paged_caches_are_taken_as_they_are():
    c = [kvc.allocate_cache(4, 16, 2, "NHD", "cuda") for _ in range(2)]
    for x in c:
        x.kv.copy_(torch.randint(-128, 128, x.kv.shape, dtype=torch.int8))
    before = [x.kv.clone() for x in c]
    r, t = i32([0, 0, 2, 1]), i32([[2, 3], [2, -1]])
    places, used = torch.zeros_like(r), torch.zeros(1, dtype=torch.int32, device="cuda")
    pth_dec.compact_pages(c, r, t, r, t, places, used)
    assert t.tolist() == [[0, 1], [0, -1]] and r.tolist() == [2, 1, 0, 0] and places.tolist() == [-1, -1, 0, 1] and int(used) == 2
    for x, b in zip(c, before):
        assert torch.equal(x.kv[:2], b[2:]) and torch.equal(x.kv[2:], b[2:])
