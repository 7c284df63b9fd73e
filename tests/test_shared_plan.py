"""pd_shared_kernel's deal, restated in Python with the source's constants: whatever the batch, the pieces of the prefix cover
every (row tile, kv head) once, the own segments cover every own key tile once, and all segments lie between 0 and the note.
"""
import os
import random
import re

import pytest

from mi50_vllm_lab_amd import pth_dec

SRC = open(os.path.join(os.path.dirname(pth_dec.__file__), "csrc", "pd_shared.hip")).read()


def const(name):
    return int(re.search(r"\b%s = (\d+)[;,]" % name, SRC).group(1))


TILE, PTILE1, PTILE2, PSEG, MERGE, OWN, SNAP = (const("kSh" + n) for n in (
    "Tile", "PrefixTile1", "PrefixTile2", "PrefixSegment", "MergeRows", "OwnUnits", "Snap"))
BIG = 0x3ffffff


def plan(own, tokens, ptiles, hkv, hq, nwg, nseg, blocks):
    """(workgroups of the prefix, pieces, row tiles): own: own key tiles of each sequence (0: no work); blocks: row blocks
    of a prefix wave."""
    segs = min(nseg, 64) - 1
    total = hkv * sum(t + OWN if t else 0 for t in own)
    longest = max(own)
    nrt = -(-tokens * (hq // hkv) // (128 * blocks))
    items = nrt * hkv if ptiles else 0
    if not items:
        return 0, 0, nrt
    costs = []
    for lane in range(64):
        rounds = 1 if lane < 48 else lane - 46
        pieces = lane + 1 if rounds == 1 else 1
        w = -(-items * pieces // rounds)
        if not (w + (total > 0) <= nwg and pieces <= segs - 2 and pieces <= ptiles):
            costs.append((BIG, lane, pieces, w))
            continue
        us = rounds * (PSEG + -(-ptiles // pieces) * (PTILE1 if blocks == 1 else PTILE2)) + tokens * hq * pieces // MERGE
        share = max(-(-total // (nwg - w)), longest // (segs - pieces - 1)) if total else 0
        costs.append((min(max(us, share * TILE), BIG), lane, pieces, w))
    cost, _, pieces, w = min(costs)
    if cost == BIG:
        wp = max(1, nwg - nwg // 8) if total else nwg
        return (nwg - 1 if wp >= nwg and total else wp), 1, nrt
    return w, pieces, nrt


def own_deal(tiles, groups, nwg, cap):
    """{(sequence, group): [(segment, first, last)]} of pd_shared_kernel's own part on nwg workgroups and cap segments."""
    units = lambda t: t + OWN if t else 0  # noqa: E731
    total, longest, items = groups * sum(map(units, tiles)), max(tiles), len(tiles) * groups
    share = max(-(-total // nwg), (longest + cap - 2) // (cap - 1), 2)
    ns = min(nwg // items, cap)
    got = {}
    if ns >= 1 and -(-longest // ns) <= share:
        for w in range(items * ns):
            item, seg = divmod(w, ns)
            b, g = divmod(item, groups)
            per = -(-tiles[b] // ns)
            if tiles[b] and seg * per < tiles[b]:
                got.setdefault((b, g), []).append((seg, seg * per, min(tiles[b], (seg + 1) * per)))
        return got
    snap = min(SNAP, share // 8)
    lead = OWN + snap
    starts = [groups * sum(map(units, tiles[:b])) for b in range(len(tiles))]

    def locate(pos):
        k = sum(starts[i] + groups * units(t) <= pos for i, t in enumerate(tiles))
        return k, starts[k], tiles[k]

    def bound(x):
        raw = min(x * share, total)
        if raw in (0, total):
            return raw
        _, start, t = locate(raw)
        off = (raw - start) % units(t)
        if off <= lead:
            return raw - off
        return raw + units(t) - off if units(t) - off <= snap else raw

    for w in range(nwg):
        pos, end = bound(w), bound(w + 1)
        while pos < end:
            b, start, t = locate(pos)
            g = (pos - start) // units(t)
            item = start + g * units(t)
            first = 0 if pos - item <= lead else pos - item - OWN
            last = t if end - item >= units(t) else end - item - OWN
            got.setdefault((b, g), []).append((w - min(item + lead, item + units(t) - 1) // share, first, last))
            if last < t:
                break
            pos = item + units(t)
    return got


@pytest.mark.parametrize("seed", range(12))
def test_every_tile_once(seed):
    r = random.Random(seed)
    for _ in range(60):
        hkv, g = r.choice([1, 2, 4, 8]), r.choice([1, 4, 6, 7])
        n, qmax = r.randint(1, r.choice([3, 40, 300])), r.choice([1, 1, 2, 4])
        nseg, nwg = r.choice([4, 5, 16, 64, 128]), r.choice([2, 40, 256, 304])
        tiles = [r.choice([0, 1, r.randint(1, 20), r.randint(1, r.choice([64, 2000]))]) for _ in range(n)]
        tokens = sum(r.randint(1, qmax) for t in tiles if t)
        if not tokens:
            continue
        ptiles = r.choice([0, 1, r.randint(1, 60), r.randint(1, 4000)])
        blocks, rows = 1 + (tokens * g > 128), tokens * g
        wp, ns, nrt = plan(tiles, tokens, ptiles, hkv, hkv * g, nwg, nseg, blocks)
        share = -(-(-(-rows // nrt)) // (16 * blocks)) * 16 * blocks     # rows of a tile
        assert share <= 128 * blocks and (nrt - 1) * share < rows <= nrt * share
        segs = min(nseg, 64) - 1
        assert 0 <= wp < nwg and ns <= segs - 2 and (ns >= 1) == (wp >= 1) == (ptiles > 0)
        seen = set()
        for w in range(wp):
            for x in range(w, nrt * hkv * ns, wp):
                rt, gp = x % nrt, x // nrt
                piece, head = gp % ns, gp // ns
                first, last = piece * ptiles // ns, (piece + 1) * ptiles // ns
                assert first < last and (rt, head, piece) not in seen
                seen.add((rt, head, piece))
        assert len(seen) == nrt * hkv * ns
        cap = segs - ns
        got = own_deal(tiles, hkv, nwg - wp, cap)
        for b, t in enumerate(tiles):
            for head in range(hkv):
                pieces = sorted(got.get((b, head), []))
                if not t:
                    assert not pieces
                    continue
                assert [s for s, _, _ in pieces] == list(range(len(pieces))) and len(pieces) <= cap
                assert [f for _, f, _ in pieces] == [0] + [x for _, _, x in pieces[:-1]] and pieces[-1][2] == t
                assert all(f < x for _, f, x in pieces)


def test_more_items_than_workgroups_run_in_rounds():
    wp, ns, nrt = plan([4] * 512, 2048, 100, 4, 24, 40, 64, 2)
    assert ns == 1 and wp < 40 and nrt * 4 > 40
    wp, ns, nrt = plan([4] * 4096, 16384, 100, 4, 24, 40, 64, 2)     # more than 17 rounds
    assert ns == 1 and 1 <= wp < 40
