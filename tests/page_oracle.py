"""Page tables and counts as lists: what fork_pages and compact_pages give, entry by entry. Test support."""


def fork(refs, table, lens, parents, columns, block_size, grow=0, window=-1, sinks=0):
    """(new table, new lengths, new counts, pages wanted, copies [(from, to, keys)])."""
    pages = len(refs)
    free = [p for p in range(pages) if refs[p] <= 0]
    counts, out, sizes, copies, wanted, met = [max(0, r) for r in refs], [], [], [], 0, set()
    names = lambda e: 0 <= e < pages  # noqa: E731
    for row in table:
        for e in row:
            if names(e):
                counts[e] -= 1
    for p in (range(len(table)) if parents is None else parents):
        row, n = [-1] * columns, 0
        if 0 <= p < len(table):
            n = max(0, lens[p])
            for c in range(columns):
                e, k0 = table[p][c], c * block_size
                if k0 >= n + grow:
                    continue
                if k0 + block_size <= n:
                    behind = window > 0 and all(sinks <= k < n + 1 - window for k in (k0, k0 + block_size - 1))
                    row[c] = e if names(e) and not behind else -1
                elif names(e) and refs[e] == 1 and p not in met:
                    row[c] = e
                else:
                    row[c] = free[wanted] if wanted < len(free) else -1
                    if names(e) and k0 < n and row[c] >= 0:
                        copies.append((e, row[c], n - k0))
                    wanted += 1
            met.add(p)
        for e in row:
            if e >= 0:
                counts[e] += 1
        out.append(row)
        sizes.append(n)
    return out, sizes, counts, wanted, copies


def compact(refs, table):
    """(new table, new counts, places, used pages)."""
    live = [p for p in range(len(refs)) if refs[p] > 0]
    places, counts = [-1] * len(refs), [0] * len(refs)
    holes = [p for p in range(len(live)) if refs[p] <= 0]
    for p in live:
        places[p] = p if p < len(live) else holes.pop(0)
        counts[places[p]] = refs[p]
    return [[places[e] if 0 <= e < len(refs) else -1 for e in row] for row in table], counts, places, len(live)
