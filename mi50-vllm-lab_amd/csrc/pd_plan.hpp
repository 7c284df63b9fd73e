// The times by which the prefill's plan (pd_python.cpp, on the host before the call) and its launches (pd_prefill.hip)
// choose among the kernels, in one place so that what is planned is what runs. Plain C++.
#pragma once

#include <stdint.h>

namespace pd {

// us per 32-key tile of a workgroup, one per CU, measured on MI355X (24 q / 4 kv heads): 192 rows, 256 rows, and a unit of
// the dealt launch's line (192 rows, K and V widened exactly, the planning and the seams of the pieces in it).
struct FaTimes {
    double tile, wide_tile, deal_unit;
};
constexpr FaTimes kFaTimes = {1.62, 1.85, 1.75};
constexpr FaTimes kFaTimesExact = {1.9, 2.2, 2.08};  // P' as fp16 hi + lo
constexpr const FaTimes& fa_times(bool exact) { return exact ? kFaTimesExact : kFaTimes; }

// Whether 256-row workgroups take less time for all rounds of one workgroup per CU: they have to save a round (2,048
// tokens x 4 splits: 3 rounds of 256 against 4, 2.92 ms against 3.30; 2,048 unsplit: one round of either, 3.7
// against 3.15).
constexpr bool fa_wide_saves(int64_t wide_rounds, int64_t rounds, bool exact) {
    return (double)wide_rounds * fa_times(exact).wide_tile < (double)rounds * fa_times(exact).tile;
}

// The deal of pd_prefill_balanced_kernel.
constexpr unsigned kFaSegmentUnits = 10;  // set-up and stores of a segment, ~16 us, in key tiles
constexpr unsigned kFaMinShare = 16;      // units of a workgroup: below, pieces cost more than they save
// An item is cut evenly where that gives no workgroup more than a share and this part of one.
constexpr unsigned kFaAlignedPart = 32;
// What the plan adds to an equal share: up to 20 more units in the longest workgroup (a share's ends fall on items'
// starts, and its last segment's set-up is its own), and planning on the device and merge, us. A dealt launch has to
// be rated 5 % faster.
constexpr int64_t kFaDealSpareUnits = 20;
constexpr double kFaDealFixedUs = 20.0;
constexpr double kFaDealMargin = 0.95;

// Windowed launches (pd_window_kernel): workgroups of 256 rows, or of 128, which take 1.5 us a key tile instead of 1.85 but fewer to
// set up and store, and are twice as many, for launches that do not fill the GPU. us, one workgroup per CU at a time: a
// tile, exact numerics' tile, set-up and stores with the launch; the merge launch of splits and their partials' way to memory and back.
// Measured and rated (24 q / 4 kv heads, over 30,000 keys), wide and narrow: 2,048 tokens over 512 keys 58 (56) and 79 (82), over 4,096
// 265 (263) and 416 (417); 1,024 over 1,024 85 (85) and 65 (64); 64 over 2,048 in 10 splits 39 (42) and 31 (31); 600 over
// 4,096 in 2 153 (155) and 124 (123); 4,096 in 2 482 (482). Exact: 2,048 over 4,096 wide 330 (334), over 512 74 (68); narrow 1,024 over 1,024 74 (74),
// 64 over 2,048 in 10 33 (33), 600 over 4,096 in 2 139 (141); 4,096 in 2 wide 592 (587).
struct FwTimes {
    double tile, tile_exact, setup;
};
constexpr FwTimes kFwWide = {1.85, 2.38, 20.0}, kFwNarrow = {1.5, 1.76, 12.0};
constexpr double kFwMergeUs = 5.0, kFwPartialUsPerMb = 0.25;
constexpr int64_t kFwMaxSplits = 16;  // of the plan, with 4 tiles each at the least
struct FwCall {
    int64_t tokens, seqs, heads_q, heads_kv, window, sinks, table_keys, cus;
    bool exact;
};
// key tiles of a query tile of `rows` rows
inline int64_t fw_key_tiles(const FwCall& c, int64_t rows) {
    const int64_t G = c.heads_q / c.heads_kv, span = c.window + (rows + G - 1) / G + 31;
    const int64_t keys = c.table_keys > 1 ? c.table_keys : 1, far = c.table_keys > span ? c.table_keys - span : 0;
    return ((span < keys ? span : keys) + 31) / 32 + ((c.sinks < far ? c.sinks : far) + 31) / 32;
}
inline double fw_us(const FwCall& c, int64_t rows, int64_t splits, const FwTimes& t) {
    const int64_t G = c.heads_q / c.heads_kv, tiles = (fw_key_tiles(c, rows) + splits - 1) / splits;
    // (half of the sequences' last query tiles are taken to be part-filled ones of their own)
    const int64_t items = ((c.tokens * G + rows - 1) / rows + (c.seqs - 1) / 2) * c.heads_kv * splits;
    const double us = (double)((items + c.cus - 1) / c.cus) * ((double)tiles * (c.exact ? t.tile_exact : t.tile) + t.setup);
    return splits == 1 ? us : us + kFwMergeUs + kFwPartialUsPerMb * (double)(c.tokens * c.heads_q) * (double)splits * 1032 / 1e6;
}
// Whether a call with this many splits runs on narrow workgroups.
inline bool fw_narrow(const FwCall& c, int64_t splits) { return fw_us(c, 128, splits, kFwNarrow) < fw_us(c, 256, splits, kFwWide); }
// The splits that are rated fastest on either.
inline int64_t fw_splits(const FwCall& c) {
    int64_t best = 1;
    double best_us = 0;
    for (int64_t s = 1; s <= kFwMaxSplits && (s == 1 || s * 4 <= fw_key_tiles(c, 128)); ++s) {
        const double wide = fw_us(c, 256, s, kFwWide), narrow = fw_us(c, 128, s, kFwNarrow), us = narrow < wide ? narrow : wide;
        if (s == 1 || us < best_us) best = s, best_us = us;
    }
    return best;
}

}  // namespace pd
