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

// Key splits of a windowed launch (pd_window_kernel): `items` workgroups per split, each of `tiles` key tiles, one per CU at a time. A
// workgroup's set-up and stores, the merge launch, and the partials' way to memory and back, us. Measured and rated (24 q / 4 kv heads): 64
// tokens over 2,048 keys 137 unsplit, 40 at 10 splits, 39 at 16 (144, 39, 38); 600 over 4,096 261, 156 at 2, 100 at 4 (268, 157,
// 103); 1,024 260 and 164 at 2 (268, 160), 2 rounds at 3 217; 4,096 521 and 489 at 2 (537, 487).
constexpr double kFwSetupUs = 18.0, kFwMergeUs = 5.0, kFwPartialUsPerMb = 0.25;
constexpr int64_t kFwMaxSplits = 16;
inline int64_t window_splits(int64_t items, int64_t tiles, int64_t rows, int64_t cus, bool exact) {
    int64_t best = 1;
    double best_us = 0;
    for (int64_t s = 1; s <= kFwMaxSplits && (s == 1 || s * 4 <= tiles); ++s) {
        const int64_t rounds = (items * s + cus - 1) / cus;
        double us = (double)rounds * ((double)((tiles + s - 1) / s) * fa_times(exact).wide_tile + kFwSetupUs);
        if (s > 1) us += kFwMergeUs + kFwPartialUsPerMb * (double)rows * (double)s * 1032 / 1e6;
        if (s == 1 || us < best_us) best = s, best_us = us;
    }
    return best;
}

}  // namespace pd
