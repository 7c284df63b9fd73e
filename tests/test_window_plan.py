"""The windowed prefill's launch restated on the CPU (fw_count, fw_order and FwSeen in pd_prefill_wide.hip, window_splits in
pd_plan.hpp): every (query tile, kv head, split) is some workgroup's and no two workgroups share one; every key that a row of a query
tile sees is in exactly one of its tiles, what is read in place of another is a seen key of the same tile, tiles taken without a
mask hold only keys that every row sees; the planned splits; and what the entry refuses.
"""
import ctypes
import os
import random
import re

import pytest
import torch

import workload as kvc
from mi50_vllm_lab_amd import pth_dec

TILE = 32
CSRC = os.path.join(os.path.dirname(pth_dec.__file__), "csrc")


def order(lin, count):
    xcd, whole = lin % 8, count // 256 * 256
    if lin < whole:
        return lin // 256 * 256 + xcd * 32 + lin // 8 % 32
    rest = count - whole
    return whole + xcd * (rest // 8) + min(xcd, rest % 8) + (lin - whole) // 8


def job_of(at, total, each):
    sharers = 8 // each if each < 8 else 1
    most = 32 * sharers
    run = at // (most * each)
    width = min(most, total - most * run)
    job, pos = divmod(at - run * most * each, width)
    return total - 1 - most * run - (pos % 32 * sharers + pos // 32 if width == most else pos), job


@pytest.mark.parametrize("hkv,nsplit", [(1, 1), (4, 1), (2, 3), (4, 16), (3, 1), (5, 1), (2, 1)])
def test_every_workgroup_has_work_of_its_own(hkv, nsplit):
    for total in (1, 2, 7, 31, 32, 33, 64, 65, 127, 128, 129, 192, 193, 256, 257, 300):
        each = hkv * nsplit
        count, seen = total * each, set()
        for lin in range(count):
            x, job = job_of(order(lin, count), total, each)
            seen.add((x, job // nsplit, job % nsplit))
        assert len(seen) == count and all(0 <= x < total and 0 <= g < hkv for x, g, _ in seen)


@pytest.mark.parametrize("hkv", [1, 2, 4, 8])
def test_no_xcd_has_more_of_a_fresh_prompt(hkv):
    """A prompt's tiles grow with their number: in whole rounds of 256 workgroups the XCDs get the same sum but for a tile's step."""
    total = 768 // hkv
    work = [0] * 8
    for lin in range(total * hkv):
        work[lin % 8] += job_of(order(lin, total * hkv), total, hkv)[0]
    assert max(work) - min(work) <= 8 * 96


@pytest.mark.parametrize("group", [1, 6, 200])
def test_tiles_of_all_sequences_fit_the_launch(group):
    rng = random.Random(group)
    for _ in range(300):
        news = [rng.choice([0, 1, rng.randint(1, 700)]) for _ in range(rng.randint(1, 90))]
        for rows in (128, 256):
            assert sum(-(-n * group // rows) for n in news) <= sum(news) * group // rows + len(news)


class Seen:
    def __init__(self, window, sinks, pmin, pmax, seq_len):
        self.window, self.pmin, self.pmax = window, pmin, pmax
        self.hi = min(seq_len, pmax + 1)
        self.lo = max(0, pmin - window + 1)
        self.sinks = max(0, min(sinks, self.hi))
        self.head = -(-self.sinks // TILE)
        self.gap = max(0, self.lo // TILE - self.head)
        self.tiles = max(0, ((self.hi - 1) // TILE + 1 if self.hi > 0 else 0) - self.gap)
        whole = -(-max(0, pmax - window + 1) // TILE)
        self.turn = whole - self.gap if whole > 0 and (whole + 1) * TILE <= pmin + 1 and whole - self.gap >= self.head else 0

    def base(self, n):
        t = n + self.turn - (self.tiles if n + self.turn >= self.tiles else 0)
        return (t if t < self.head else t + self.gap) * TILE

    def near(self, kb, k):
        if k < self.sinks:
            return k
        return min(max(k, self.lo), self.hi - 1) if self.lo < kb + TILE else self.sinks - 1

    def masked(self, kb):
        return kb + TILE - 1 > self.pmin or (kb + TILE > self.sinks and self.pmax - kb >= self.window)


@pytest.mark.parametrize("span", [1, 2, 43])
@pytest.mark.parametrize("sinks", [0, 1, 4, 31, 32, 33, 70, 500])
def test_tiles_cover_what_is_seen(span, sinks):
    for pmin in [-5, -1] + list(range(0, 100)) + [127, 128, 160, 191, 250]:
        for window in (1, 2, 16, 31, 32, 33, 64, 100, 400):
            pmax = pmin + span - 1
            s = Seen(window, sinks, pmin, pmax, pmax + 1)
            sees = lambda p, k: 0 <= k <= p and (p - k < window or k < sinks)  # noqa: E731
            some = {k for k in range(pmax + 1) if any(sees(p, k) for p in (*range(pmin, pmax + 1),))} if span < 3 else \
                {k for k in range(pmax + 1) if k < sinks or k > pmin - window}
            bases = [s.base(n) for n in range(s.tiles)]
            assert len(set(bases)) == len(bases)
            covered = {k for b in bases for k in range(b, b + TILE)}
            assert some <= covered
            for b in bases:
                assert any(k in some for k in range(b, b + TILE))
                for k in range(b, b + TILE):
                    assert s.near(b, k) in some and b <= s.near(b, k) < b + TILE and (k not in some or s.near(b, k) == k)
                    if not s.masked(b):
                        assert sees(pmin, k) and sees(pmax, k)
                for u in (0, 16):
                    n = s.near(b, b + u) & ~15
                    assert b <= n < b + TILE and any(k in some for k in range(n, n + 16))
            if s.turn:
                assert not s.masked(bases[0])


def test_planned_splits():
    text = open(os.path.join(CSRC, "pd_plan.hpp")).read()
    times = [tuple(map(float, re.search(r"%s = \{([\d.]+), ([\d.]+), ([\d.]+)\}" % n, text).groups())) for n in ("kFwWide", "kFwNarrow")]
    merge, mb = map(float, re.search(r"kFwMergeUs = ([\d.]+), kFwPartialUsPerMb = ([\d.]+);", text).groups())
    most = int(re.search(r"kFwMaxSplits = (\d+);", text).group(1))
    lib = pth_dec.load_library()

    def want(T, seqs, hq, hkv, window, sinks, keys, exact, cus=256):
        g = hq // hkv

        def key_tiles(rows):
            span = window + -(-rows // g) + 31
            return -(-min(span, max(1, keys)) // 32) + -(-min(sinks, max(0, keys - span)) // 32)

        best = None
        for s in range(1, most + 1):
            if s > 1 and s * 4 > key_tiles(128):
                break
            for rows, t in ((256, times[0]), (128, times[1])):
                items = (-(-T * g // rows) + (seqs - 1) // 2) * hkv * s
                us = -(-items // cus) * (-(-key_tiles(rows) // s) * t[exact] + t[2])
                us += merge + mb * T * hq * s * 1032 / 1e6 if s > 1 else 0
                if best is None or us < best[0]:
                    best = (us, s)
        return best[1]

    rng = random.Random(3)
    for _ in range(300):
        hq, hkv = rng.choice([(24, 4), (12, 2), (6, 6), (16, 1)])
        a = (rng.choice([1, 16, 64, 300, 2048, 8192]), rng.choice([1, 2, 9, 70]), hq, hkv, rng.choice([1, 100, 1000, 4096]),
             rng.choice([0, 4, 500]), rng.choice([0, 100, 5000, 100000]), rng.choice([0, 1]))
        assert lib.pth_fa_window_splits(*a) == want(*a), a
    assert lib.pth_fa_window_splits(8192, 1, 24, 4, 4096, 4, 100000, 0) == 1   # three rounds of wide workgroups
    assert lib.pth_fa_window_splits(1024, 1, 24, 4, 1024, 4, 100000, 0) == 1   # 192 narrow ones
    assert lib.pth_fa_window_splits(64, 1, 24, 4, 2048, 4, 100000, 0) > 4      # 12 of them
    for bad in ((0, 1, 24, 4, 9, 0, 9, 0), (9, 0, 24, 4, 9, 0, 9, 0), (9, 1, 24, 5, 9, 0, 9, 0), (9, 1, 24, 4, 0, 0, 9, 0), (9, 1, 24, 0, 9, 0, 9, 0)):
        assert lib.pth_fa_window_splits(*bad) == 1


def test_refusals():
    lib = pth_dec.load_library()
    case = kvc.make_case([37, 5], [3, 1], num_q_heads=12, num_kv_heads=2, block_size=16, seed=3)
    c = case.cache
    big = 1 << 31
    good = dict(q=case.q, kc=c.key_cache, vc=c.value_cache, bt=case.block_table, lens=case.seq_lens, qsl=case.query_start_loc,
                out=torch.zeros((4, 12, 256), dtype=torch.float16), ws=torch.zeros(4 * 12 * 2 * 258))
    numbers = dict(num_seqs=2, window=16, sinks=4, nsplit=2, exact=0)
    err = ctypes.create_string_buffer(256)

    def call(a):
        d = {n: None if a[n] is None else ctypes.byref(pth_dec.describe(a[n])) for n in good}
        return lib.pth_fa_forward_window(*[d[n] for n in ("q", "kc", "vc", "bt", "lens")], 0.1, d["qsl"], d["out"], d["ws"],
                                         *[a[n] for n in numbers], None, err, len(err))

    cases = [({n: None}, "null tensor descriptor") for n in good if n != "ws"] + [
        (dict(q=case.q.float()), "q must be fp16"), (dict(q=case.q[0]), "q must be fp16"),
        (dict(q=case.q[..., :128]), "q must be fp16"), (dict(out=good["out"].float()), "out must be fp16"),
        (dict(out=good["out"][:3]), "out must be fp16"), (dict(out=good["out"][:, :11]), "out must be fp16"),
        (dict(q=torch.zeros(4 * 12 * 256 + 4).half()[4:].view(4, 12, 256)), "16-byte aligned"),
        (dict(out=torch.zeros(4 * 12 * 256 + 2).half()[2:].view(4, 12, 256)), "8-byte aligned"),
        (dict(out=good["out"][:1].expand(4, 12, 256)), "out rows must not overlap"),
        (dict(kc=c.key_cache[..., :256]), "4D int8 rows"), (dict(vc=c.key_cache), "260 bytes in"),
        (dict(q=case.q[:, :11], out=good["out"][:, :11]), "multiple of heads_kv"),
        (dict(num_seqs=0), "row for each"), (dict(num_seqs=3), "row for each"), (dict(bt=case.block_table.long()), "row for each"),
        (dict(lens=case.seq_lens.long()), "row for each"), (dict(qsl=case.query_start_loc[:2]), "row for each"),
        (dict(window=0), "window must be"), (dict(window=-1), "window must be"), (dict(window=big), "window must be"),
        (dict(sinks=-1), "sinks at least 0"), (dict(sinks=big), "sinks at least 0"),
        (dict(nsplit=0), "nsplit must be"), (dict(nsplit=65), "nsplit must be"),
        (dict(ws=None), "workspace must be"), (dict(ws=good["ws"][:-1]), "workspace must be"), (dict(ws=good["ws"].half()), "workspace must be"),
        (dict(ws=torch.zeros(4 * 12 * 2 * 258 + 1)[1:]), "workspace must be"),
        (dict(q=case.q[:1].expand(1 << 27, 12, 256), out=good["out"][:1].expand(1 << 27, 12, 256)), "at most 2^30"),
    ]
    for change, msg in cases:
        assert call({**good, **numbers, **change}) == 1 and msg in err.value.decode(), (list(change), err.value)
    assert call({**good, **numbers, "q": case.q[:0], "out": good["out"][:0]}) == 0
    with pytest.raises(RuntimeError, match="on one GPU"):
        pth_dec.forward_window(case.q, c.key_cache, c.value_cache, case.block_table, case.seq_lens, 0.1, case.query_start_loc,
                               good["out"], 16)
