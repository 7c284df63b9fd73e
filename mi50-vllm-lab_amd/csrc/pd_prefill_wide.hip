// Chunked prefill with 256 query rows per workgroup, for launches of several rounds of workgroups
// (pd_prefill.hip's kernel takes 192). Same interface and partials. The (token, head of one kv head) pairs of a
// sequence are its rows, token-major; a workgroup takes kFwRows consecutive rows (4 waves of 4
// blocks of 16) and streams every visible 32-key tile once:
//   HBM -> LDS   the waves copy a step of two tiles together (9 copies each) into a 6-tile ring,
//                two steps ahead; one barrier per step publishes it and frees its predecessor;
//   int8 -> fp16 each wave widens the operands that it reads in registers, exactly (no bias), between the
//                products of the operand before (score_products, value_products);
//   MFMA         S^T = K Q^T and O^T += V^T P'^T on fp16 MFMA with fp32 accumulation; Q in 128 vector
//                registers, O in all 256 accumulation registers.
// What bounds it: a tile's 32 blocks of 4 MFMAs and 8 conversions take 2,327 cycles and its softmax 884 (measured
// alone), but under that load the card runs at 1.5-2.0 GHz instead of 2.4; the whole tile takes 1.85 us (2.35
// GHz), where 192 rows take 1.62 us in pd_prefill.hip: 13 % less per row. It pays where its larger
// workgroups do not cost a round (launch_prefill): 2,048 tokens over 61,440 keys (24 q / 4 kv heads) 3.15 ms ->
// 2.92 in 4 splits. A widening through LDS once per workgroup (3.29 ms: the LDS latency shows) and two waves of
// 32 rows per SIMD (3.66 ms: each conversion then serves half the products) were slower. The exact widening
// leaves the default numerics' error at its fp16 weights: 2.1e-4 of the result at 63,488 keys, 7.9e-3 with the
// biased one.
// kExact (pth_fa_forward_exact) carries P' as fp16 hi + lo, which doubles the P.V products; the
// default rounds P' once to fp16.
#include <type_traits>

#include "pd_tile.hpp"
#include "pth_dec.h"

namespace pd {

constexpr int kFwWaves = 4;
constexpr int kFwRB = 4;                          // 16-row blocks per wave
static_assert(kFwRows == kFwWaves * kFwRB * 16, "rows of a workgroup");
constexpr int kFwStep = 2;                        // tiles per barrier
constexpr int kFwAhead = 2;                       // steps in flight
constexpr int kFwRing = kFwStep * (kFwAhead + 1);  // tile slots
// A slot: the K and V images of pd_tile.hpp (V from byte 260 of the row, so its 16 blocks hold whole
// dim blocks), then the tile's scales: k_scale [32], v_scale [32].
constexpr int kFwImgV = kImgV;
constexpr int kFwImgS = 16 * kBlk;
constexpr int kFwSlot = kFwImgS + 256;
constexpr int kFwCopies = 4 * kFwStep + 1;        // copies of a wave per step
constexpr int kFwBt = 6144;                       // 16-key blocks (or pages) of the LDS block table

// The products of one widened operand `cur` with the four row blocks of a wave, and between them the
// widening of the next operand from its bytes (w0, w1): a 16x16x32 MFMA keeps the matrix core busy
// for 16 cycles and leaves the issue slots of about three of these conversions. The order is
// written out because the compiler gathers the conversions before the products. (The trailing
// s_nop keeps the last conversion two slots from the next block's first product, which reads it.)
#define PD_CVT(d, w, half, byte, keep) \
    "v_cvt_f16_i16_sdwa " d ", sext(" w ") dst_sel:WORD_" half " dst_unused:UNUSED_" keep " src0_sel:BYTE_" byte "\n\t"
#define PD_PRODUCTS_AND_WIDEN(C0, C1, C2, C3)                                    \
    "v_mfma_f32_16x16x32_f16 %0, %8, %9, " C0 "\n\t"                              \
    PD_CVT("%4", "%13", "0", "0", "PAD") PD_CVT("%5", "%13", "0", "2", "PAD") PD_CVT("%6", "%14", "0", "0", "PAD") \
    "v_mfma_f32_16x16x32_f16 %1, %8, %10, " C1 "\n\t"                             \
    PD_CVT("%7", "%14", "0", "2", "PAD") PD_CVT("%4", "%13", "1", "1", "PRESERVE") PD_CVT("%5", "%13", "1", "3", "PRESERVE") \
    "v_mfma_f32_16x16x32_f16 %2, %8, %11, " C2 "\n\t"                             \
    PD_CVT("%6", "%14", "1", "1", "PRESERVE") PD_CVT("%7", "%14", "1", "3", "PRESERVE")    \
    "v_mfma_f32_16x16x32_f16 %3, %8, %12, " C3 "\n\ts_nop 0"
// scores: accumulators in vector registers (the softmax reads them)
template <bool kFirst>
__device__ __forceinline__ half8_t score_products(float4_t& s0, float4_t& s1, float4_t& s2, float4_t& s3, half8_t cur,
                                                  half8_t q0, half8_t q1, half8_t q2, half8_t q3, unsigned w0,
                                                  unsigned w1) {
    uint4_t n;
    if constexpr (kFirst)
        asm volatile(PD_PRODUCTS_AND_WIDEN("0", "0", "0", "0")
                     : "=&v"(s0), "=&v"(s1), "=&v"(s2), "=&v"(s3), "=&v"(n.x), "=&v"(n.y), "=&v"(n.z), "=&v"(n.w)
                     : "v"(cur), "v"(q0), "v"(q1), "v"(q2), "v"(q3), "v"(w0), "v"(w1));
    else
        asm volatile(PD_PRODUCTS_AND_WIDEN("%0", "%1", "%2", "%3")
                     : "+v"(s0), "+v"(s1), "+v"(s2), "+v"(s3), "=&v"(n.x), "=&v"(n.y), "=&v"(n.z), "=&v"(n.w)
                     : "v"(cur), "v"(q0), "v"(q1), "v"(q2), "v"(q3), "v"(w0), "v"(w1));
    return __builtin_bit_cast(half8_t, n);
}
// values: O stays in the accumulation registers
__device__ __forceinline__ half8_t value_products(float4_t& o0, float4_t& o1, float4_t& o2, float4_t& o3, half8_t cur,
                                                  half8_t p0, half8_t p1, half8_t p2, half8_t p3, unsigned w0,
                                                  unsigned w1) {
    uint4_t n;
    asm volatile(PD_PRODUCTS_AND_WIDEN("%0", "%1", "%2", "%3")
                 : "+a"(o0), "+a"(o1), "+a"(o2), "+a"(o3), "=&v"(n.x), "=&v"(n.y), "=&v"(n.z), "=&v"(n.w)
                 : "v"(cur), "v"(p0), "v"(p1), "v"(p2), "v"(p3), "v"(w0), "v"(w1));
    return __builtin_bit_cast(half8_t, n);
}
__device__ __forceinline__ void value_products_only(float4_t& o0, float4_t& o1, float4_t& o2, float4_t& o3, half8_t cur,
                                                    half8_t p0, half8_t p1, half8_t p2, half8_t p3) {
    asm volatile("v_mfma_f32_16x16x32_f16 %0, %4, %5, %0\n\tv_mfma_f32_16x16x32_f16 %1, %4, %6, %1\n\t"
                 "v_mfma_f32_16x16x32_f16 %2, %4, %7, %2\n\tv_mfma_f32_16x16x32_f16 %3, %4, %8, %3"
                 : "+a"(o0), "+a"(o1), "+a"(o2), "+a"(o3)
                 : "v"(cur), "v"(p0), "v"(p1), "v"(p2), "v"(p3));
}
// The same for two row blocks (narrow workgroups): four conversions behind each product. A product reads an accumulator of the block
// before 11 issue slots after it was written, or as the very register it accumulates into, which needs none.
#define PD_PRODUCTS_AND_WIDEN_2(C0, C1)                                          \
    "v_mfma_f32_16x16x32_f16 %0, %6, %7, " C0 "\n\t"                              \
    PD_CVT("%2", "%9", "0", "0", "PAD") PD_CVT("%3", "%9", "0", "2", "PAD") PD_CVT("%4", "%10", "0", "0", "PAD") \
    PD_CVT("%5", "%10", "0", "2", "PAD")                                         \
    "v_mfma_f32_16x16x32_f16 %1, %6, %8, " C1 "\n\t"                              \
    PD_CVT("%2", "%9", "1", "1", "PRESERVE") PD_CVT("%3", "%9", "1", "3", "PRESERVE") \
    PD_CVT("%4", "%10", "1", "1", "PRESERVE") PD_CVT("%5", "%10", "1", "3", "PRESERVE") "s_nop 1"
template <bool kFirst>
__device__ __forceinline__ half8_t score_products(float4_t& s0, float4_t& s1, half8_t cur, half8_t q0, half8_t q1, unsigned w0,
                                                  unsigned w1) {
    uint4_t n;
    if constexpr (kFirst)
        asm volatile(PD_PRODUCTS_AND_WIDEN_2("0", "0")
                     : "=&v"(s0), "=&v"(s1), "=&v"(n.x), "=&v"(n.y), "=&v"(n.z), "=&v"(n.w)
                     : "v"(cur), "v"(q0), "v"(q1), "v"(w0), "v"(w1));
    else
        asm volatile(PD_PRODUCTS_AND_WIDEN_2("%0", "%1")
                     : "+v"(s0), "+v"(s1), "=&v"(n.x), "=&v"(n.y), "=&v"(n.z), "=&v"(n.w)
                     : "v"(cur), "v"(q0), "v"(q1), "v"(w0), "v"(w1));
    return __builtin_bit_cast(half8_t, n);
}
__device__ __forceinline__ half8_t value_products(float4_t& o0, float4_t& o1, half8_t cur, half8_t p0, half8_t p1, unsigned w0,
                                                  unsigned w1) {
    uint4_t n;
    asm volatile(PD_PRODUCTS_AND_WIDEN_2("%0", "%1")
                 : "+a"(o0), "+a"(o1), "=&v"(n.x), "=&v"(n.y), "=&v"(n.z), "=&v"(n.w)
                 : "v"(cur), "v"(p0), "v"(p1), "v"(w0), "v"(w1));
    return __builtin_bit_cast(half8_t, n);
}
__device__ __forceinline__ void value_products_only(float4_t& o0, float4_t& o1, half8_t cur, half8_t p0, half8_t p1) {
    asm volatile("v_mfma_f32_16x16x32_f16 %0, %2, %3, %0\n\tv_mfma_f32_16x16x32_f16 %1, %2, %4, %1"
                 : "+a"(o0), "+a"(o1)
                 : "v"(cur), "v"(p0), "v"(p1));
}
// Wait states between asm MFMAs and the first other instruction that touches their results (the
// operands keep the compiler from moving such an instruction before the wait).
__device__ __forceinline__ void settle_scores(float4_t (&s)[2][2]) {
    asm volatile("s_nop 15" : "+v"(s[0][0]), "+v"(s[0][1]), "+v"(s[1][0]), "+v"(s[1][1]));
}
__device__ __forceinline__ void settle_scores(float4_t (&s)[kFwRB][2]) {
    asm volatile("s_nop 15" : "+v"(s[0][0]), "+v"(s[0][1]), "+v"(s[1][0]), "+v"(s[1][1]), "+v"(s[2][0]), "+v"(s[2][1]),
                 "+v"(s[3][0]), "+v"(s[3][1]));
}
__device__ __forceinline__ void settle_values(float4_t (&o)[16]) {
    asm volatile("s_nop 15" : "+a"(o[0]), "+a"(o[1]), "+a"(o[2]), "+a"(o[3]), "+a"(o[4]), "+a"(o[5]), "+a"(o[6]), "+a"(o[7]));
    asm volatile("" : "+a"(o[8]), "+a"(o[9]), "+a"(o[10]), "+a"(o[11]), "+a"(o[12]), "+a"(o[13]), "+a"(o[14]), "+a"(o[15]));
}
// The wait before the products of P' (see settle_operand), once for all of its row blocks.
template <bool kExact>
__device__ __forceinline__ void settle_weights(half8_t (&p)[2], half8_t (&lo)[2]) {
    if constexpr (kExact)
        asm volatile("s_nop 1" : "+v"(p[0]), "+v"(p[1]), "+v"(lo[0]), "+v"(lo[1]));
    else
        asm volatile("s_nop 1" : "+v"(p[0]), "+v"(p[1]));
}
template <bool kExact>
__device__ __forceinline__ void settle_weights(half8_t (&p)[kFwRB], half8_t (&lo)[kFwRB]) {
    if constexpr (kExact)
        asm volatile("s_nop 1" : "+v"(p[0]), "+v"(p[1]), "+v"(p[2]), "+v"(p[3]), "+v"(lo[0]), "+v"(lo[1]), "+v"(lo[2]), "+v"(lo[3]));
    else
        asm volatile("s_nop 1" : "+v"(p[0]), "+v"(p[1]), "+v"(p[2]), "+v"(p[3]));
}

constexpr int kFwLdsBt = kFwRing * kFwSlot;
constexpr int kFwLdsScr = kFwLdsBt + kFwBt * 4;  // 4 KiB per wave for the rescale of O
constexpr int kFwLdsBytes = kFwLdsScr + kFwWaves * 4096;
constexpr int kFwLdsPos = kFwLdsBytes;           // windowed: the rows' positions
constexpr int kFwWindowLdsBytes = kFwLdsPos + kFwRows * 4;
static_assert(kFwWindowLdsBytes <= 160 * 1024, "gfx950 has 160 KiB of LDS per CU");

// The keys that the rows [tok0, tok_last] of a sequence see with a sliding window and sinks: [lo, hi) and the first `sinks`.
// Tiles are numbered over what is seen: [0, head) hold the sinks, from `head` on a tile lies `gap` tiles further than its number. They are
// taken from the first one on that every row sees all of, and those before it last: the rows' running maxima then start from 32
// keys each, not from the few of the sinks or of the window's ragged end, and seldom have to be raised, which rescales O.
struct FwSeen {
    int lo, hi, sinks, head, gap;
    int turn, tiles;  // tile n is the (n + turn)-th of `tiles`
    __device__ __forceinline__ int base(int n) const {
        const int tile = n + turn - (n + turn >= tiles ? tiles : 0);
        return (tile < head ? tile : tile + gap) * kTile;
    }
    // a key of the tile at kb that is seen, k itself if it is
    __device__ __forceinline__ int near(int kb, int k) const {
        if (k < sinks) return k;
        return lo < kb + kTile ? min(max(k, lo), hi - 1) : sinks - 1;
    }
    __device__ __forceinline__ bool has(int k) const { return ((k >= lo) | (k < sinks)) & (k < hi); }
};

// Query tiles of a windowed launch: each sequence's rows [query_start[i], query_start[i + 1]) in runs of kRows, sequence by sequence;
// sequences without keys have none. (A wave looks 64 sequences up at a time.)
struct FwItem {
    int b, tile, first, ntok;  // sequence, its query tile, its first row, its tokens
};
struct FwTiles {
    unsigned tiles0, incl0;    // this lane's sequence (of the first 64): its tiles, the tiles up to and with it
    int first0, end0;
    unsigned total;
};
template <int kRows>
__device__ __forceinline__ unsigned fw_tiles(const FaWindow& w, const int* seq_lens, int G, int i, int& first, int& end) {
    const int c = min(i, w.num_seqs - 1);
    first = max(0, w.query_start[c]);
    end = min(w.query_start[c + 1], w.num_tokens);
    const bool live = i < w.num_seqs && end > first && seq_lens[c] > 0;
    return live ? (unsigned)(((int64_t)(end - first) * G + kRows - 1) / kRows) : 0u;
}
template <int kRows>
__device__ __forceinline__ FwTiles fw_count(const FaWindow& w, const int* seq_lens, int G) {
    const int lane = threadIdx.x & 63;
    FwTiles t;
    t.tiles0 = fw_tiles<kRows>(w, seq_lens, G, lane, t.first0, t.end0);
    t.incl0 = wave_scan(t.tiles0);
    t.total = (unsigned)__builtin_amdgcn_readlane((int)t.incl0, 63);
    for (int c = 64; c < w.num_seqs; c += 64) {
        int first, end;
        t.total += (unsigned)__builtin_amdgcn_readlane((int)wave_scan(fw_tiles<kRows>(w, seq_lens, G, c + lane, first, end)), 63);
    }
    return t;
}
// Query tile x < total.
template <int kRows>
__device__ __forceinline__ FwItem fw_item(const FaWindow& w, const int* seq_lens, int G, const FwTiles& t, unsigned x) {
    const int lane = threadIdx.x & 63;
    unsigned before = 0;
    for (int c = 0;; c += 64) {
        int first = t.first0, end = t.end0;
        unsigned tiles = t.tiles0, incl = t.incl0;
        if (c > 0) {
            tiles = fw_tiles<kRows>(w, seq_lens, G, c + lane, first, end);
            incl = wave_scan(tiles);
        }
        const int k = __popcll(__ballot(before + incl <= x));
        if (k < 64) {
            const unsigned at = before + (unsigned)__builtin_amdgcn_readlane((int)(incl - tiles), k);
            const int q0 = __builtin_amdgcn_readlane(first, k), q1 = __builtin_amdgcn_readlane(end, k);
            return {c + k, (int)(x - at), q0, q1 - q0};
        }
        before += (unsigned)__builtin_amdgcn_readlane((int)incl, 63);
    }
}
// The place of workgroup `lin` of `count` in the order of the work: the 8 XCDs, which the hardware deals workgroups to in turn, take 32
// neighbours (one per CU) each, in turn as well, so that what runs at once on an XCD shares an L2's keys; the rest of less than 256
// goes to them in equal runs.
__device__ __forceinline__ unsigned fw_order(unsigned lin, unsigned count) {
    const unsigned xcd = lin % 8u, whole = count / 256u * 256u;
    if (lin < whole) return lin / 256u * 256u + xcd * 32u + lin / 8u % 32u;
    const unsigned rest = count - whole;
    return whole + xcd * (rest / 8u) + min(xcd, rest % 8u) + (lin - whole) / 8u;
}

// The order of the work of `total` query tiles with `each` jobs (kv heads and splits) of every one: runs of 32 query tiles, the last tiles first
// (those of a fresh prompt see the most keys), and in a run job by job. With fewer than 8 jobs a run is as many times longer as fills the 8
// XCDs, and those that share a job take its tiles by turns, so that none gets only the long or the short ones: 8,192 fresh tokens over a window
// of 4,096 take 628 us so and 683 where each takes 32 neighbours, 4,096 of them 248 and 268, 4 chunks of 2,048 257 and 282.
struct FwJob {
    unsigned tile, job;
};
__device__ __forceinline__ FwJob fw_job(unsigned at, unsigned total, unsigned each) {
    const unsigned sharers = each < 8u ? 8u / each : 1u, most = 32u * sharers;
    const unsigned run = at / (most * each), width = min(most, total - most * run);
    const unsigned in = at - run * most * each, job = in / width, pos = in - job * width;
    return {total - 1 - most * run - (width == most ? pos % 32u * sharers + pos / 32u : pos), job};
}

// A workgroup of pd_prefill_wide_kernel and, with kWindow, of pd_window_kernel.
template <bool kFast, bool kExact, bool kSplit, class T, bool kWindow, int kRB>
__device__ __forceinline__ void wide_workgroup(const FaParams& a, const FaWindow& win, unsigned char* lds) {
    constexpr int kLdsBt = kFwLdsBt, kLdsScr = kFwLdsScr, kRows = 16 * kRB * kFwWaves;
    int x, g, b, qt, split, ntok = a.Sq, first = 0;
    if constexpr (kWindow) {
        const FwTiles tiles = fw_count<kRows>(win, a.seq_lens, a.G);
        const unsigned lin = blockIdx.x + gridDim.x * blockIdx.y, each = gridDim.y * (unsigned)a.nsplit, count = tiles.total * each;
        if (lin >= count) return;
        const FwJob mine = fw_job(fw_order(lin, count), tiles.total, each);
        x = (int)mine.tile;
        g = (int)(mine.job / (unsigned)a.nsplit);
        split = (int)(mine.job - (unsigned)g * (unsigned)a.nsplit);
        const FwItem item = fw_item<kRows>(win, a.seq_lens, a.G, tiles, (unsigned)x);
        b = item.b, qt = item.tile, ntok = item.ntok, first = item.first;
    } else {
        // Workgroups are dispatched to the 8 XCDs round robin (linear id L to XCD L % 8), and each XCD
        // has its own L2. Every query tile of a (sequence, kv head) streams the same keys, so the
        // logical workgroup index (query tile fastest) is laid out XCD by XCD: XCD x takes a
        // contiguous range of it, and the query tiles sharing a kv head mostly share an L2.
        const unsigned nx = gridDim.x, ny = gridDim.y, nwg = nx * ny * gridDim.z;
        const unsigned lin = blockIdx.x + nx * (blockIdx.y + ny * blockIdx.z);
        const unsigned xcd = lin % 8u;
        const unsigned lidx = xcd * (nwg / 8u) + min(xcd, nwg % 8u) + lin / 8u;
        // x = split * (query tiles) + query tile: the query tiles of one split and kv head (which
        // stream the same keys) stay neighbours in the XCD order
        x = (int)(lidx % nx), g = (int)((lidx / nx) % ny), b = (int)(lidx / (nx * ny));
        const int nqt = kSplit ? (int)nx / a.nsplit : (int)nx;
        qt = kSplit ? x % nqt : x, split = kSplit ? x / nqt : 0;
    }
    const int tid = threadIdx.x, l = tid & 63;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int G = a.G;
    // rows of this workgroup: [row0, row0 + nrow) of the sequence's (token, head) rows
    const int64_t row0 = (int64_t)qt * kRows;
    const int nrow = (int)min((int64_t)kRows, (int64_t)ntok * G - row0);
    const int tok0 = (int)(row0 / G), tok_last = (int)((row0 + nrow - 1) / G);
    const int tok0_row = (int)(row0 - (int64_t)tok0 * G);  // rows of the first token that come before
    const int seq_len = a.seq_lens[b];
    const int qabs = !kWindow && a.q_abs ? a.q_abs[b] : seq_len - ntok;
    // keys any row can see: [0, min(seq_len, last row's position + 1))
    const int hi = min(seq_len, qabs + tok_last + 1);
    int ntiles = hi > 0 ? (hi - 1) / kTile + 1 : 0;
    const int pmin = qabs + tok0;                      // smallest row position
    FwSeen seen = {0, hi, 0, 0, 0, 0, 0};
    if constexpr (kWindow) {
        seen.lo = max(0, pmin - win.window + 1);
        seen.sinks = max(0, min(win.sinks, hi));
        seen.head = (seen.sinks + kTile - 1) / kTile;
        seen.gap = max(0, seen.lo / kTile - seen.head);
        seen.tiles = ntiles = max(0, ntiles - seen.gap);
        const int whole = (max(0, qabs + tok_last - win.window + 1) + kTile - 1) / kTile;  // the window's first tile that all rows see
        if (whole > 0 && (whole + 1) * kTile <= pmin + 1 && whole - seen.gap >= seen.head) seen.turn = whole - seen.gap;
    }
    // this workgroup's run of key tiles [t0, t1): all of them unless the keys are split
    const int per = kSplit ? (ntiles + a.nsplit - 1) / a.nsplit : ntiles;
    const int t0 = kSplit ? min(ntiles, split * per) : 0, t1 = kSplit ? min(ntiles, t0 + per) : ntiles;

    // The lane number as a value of its own: what is computed from it stays where it is used instead
    // of being kept in registers across the tile loop.
    auto lane_here = [&]() __attribute__((always_inline)) {
        int x = l;
        asm volatile("" : "+v"(x));
        return x;
    };

    // ---- rows of this wave: row r = 64 w + 16 rb + li -> (token, head). Looked up again where
    //      needed (the tile loop has no registers to keep them) ----
    struct Row {
        bool valid;
        int tok, head;
    };
    const float per_token = 1.f / (float)G;
    auto row_at = [&](int r) __attribute__((always_inline)) {
        Row x;
        x.valid = r < nrow;
        r = tok0_row + (x.valid ? r : 0);  // row of the workgroup's first token's rows
        if constexpr (kWindow)
            x.tok = (int)(((float)r + 0.5f) * per_token);  // r / G: at most 512, half a row from the next token
        else
            x.tok = r / G;
        x.head = r - x.tok * G;
        x.tok += tok0;
        return x;
    };
    auto row_of = [&](int rb) __attribute__((always_inline)) { return row_at(16 * kRB * w + 16 * rb + (lane_here() & 15)); };
    half8_t qop[kRB][8];
    auto load_q = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int rb = 0; rb < kRB; ++rb) {
            const Row r = row_of(rb);
            const T* qrow = static_cast<const T*>(a.q) + (kWindow ? (int64_t)first * a.q_st : (int64_t)b * a.q_sb) +
                            (int64_t)(g * G + r.head) * a.q_sh + (int64_t)r.tok * a.q_st;
#pragma unroll
            for (int st = 0; st < 8; ++st) {
                const half8_t v = load_q8<T>(qrow + 64 * (st >> 1) + 16 * (l >> 4) + 8 * (st & 1));
                // (windowed: a row that is not there holds the first one's values, which go nowhere)
                qop[rb][st] = kWindow || r.valid ? v : (half8_t)(_Float16)0.0f;
            }
            // one row block's loads at a time: four do not fit the registers in fp32
            if constexpr (!kWindow)
                asm volatile("" : "+v"(qop[rb][0]), "+v"(qop[rb][1]), "+v"(qop[rb][2]), "+v"(qop[rb][3]), "+v"(qop[rb][4]),
                             "+v"(qop[rb][5]), "+v"(qop[rb][6]), "+v"(qop[rb][7]));
        }
    };
    // Windowed launches have few tiles each: their first copies are under way before Q is loaded, all of it in one trip.
    if constexpr (!kWindow) load_q();
    asm volatile("" ::: "memory");  // every Q load is issued before the block table is read

    lds_u8* L = (lds_u8*)lds;
    const unsigned lds_base = (unsigned)(uintptr_t)L;
    const int8_t* gbase = a.kc + (int64_t)g * a.k_sh;
    // ---- block table of the workgroup's keys into LDS: for bs % 16 == 0 the byte offset / 8 of
    //      every 16-key block's first row, else the page numbers ----
    PageTable pt;
    pt.glob = (const_int_ptr)(uintptr_t)(a.block_table + (int64_t)b * a.bt_stride);
    pt.lds = (const lds_int*)(L + kLdsBt);
    pt.rows16 = nullptr;
    pt.pfirst = 0;
    {
        const int* bt_glob = a.block_table + (int64_t)b * a.bt_stride;
        lds_int* dst = (lds_int*)(L + kLdsBt);
        if constexpr (kFast) {
            const int nblk = 2 * (t1 - t0);  // the workgroup's tiles t0 + i / 2
            pt.in_lds = a.bt32 && nblk <= kFwBt;
            if (pt.in_lds) {
                for (int i = tid; i < nblk; i += kFwWaves * 64) {
                    const int kb = kWindow ? seen.base(t0 + (i >> 1)) : (t0 + (i >> 1)) * kTile;
                    const int klast = min(kb + kTile - 1, hi - 1);
                    const int key0 = (kWindow ? seen.near(kb, kb + 16 * (i & 1)) : min(kb + 16 * (i & 1), klast)) & ~15;
                    const int lb = a.bs_shift >= 0 ? key0 >> a.bs_shift : key0 / a.block_size;
                    const int64_t off = (int64_t)bt_glob[lb] * a.k_sb + (int64_t)(key0 - lb * a.block_size) * a.k_ss;
                    dst[i] = (int)(unsigned)((uint64_t)off >> 3);
                }
            }
        } else {
            const int npages = hi > 0 ? (hi - 1) / a.block_size + 1 : 0;
            pt.in_lds = npages <= kFwBt;
            if (pt.in_lds)
                for (int i = tid; i < npages; i += kFwWaves * 64) dst[i] = bt_glob[i];
        }
    }
    if constexpr (kWindow) {
        const Row row = row_at(tid);
        ((lds_int*)(L + kFwLdsPos))[tid] = row.valid ? qabs + row.tok : -1;
    }
    __syncthreads();  // the LDS block table is complete

    // Relative scores carry +kPLog2: p' = 2^(s - m + kPLog2) = 16 p, so P' = p' * v_scale spans the
    // same fp16 range as in the decode kernel; l accumulates p' and the final 1 / l removes it.
    constexpr float kPLog2 = 4.0f;
    float l_run[kRB];
    // per row: the score offset -m + kPLog2 (kPLog2 while the row has seen no key) and the
    // relative score above which the running max m must be raised (any finite score while fresh)
    float nm_run[kRB], thr_run[kRB];
    float4_t oacc[kRB][16];
#pragma unroll
    for (int rb = 0; rb < kRB; ++rb) {
        l_run[rb] = 0.f;
        nm_run[rb] = kPLog2;
        thr_run[rb] = kNegInf;
#pragma unroll
        for (int m = 0; m < 16; ++m) oacc[rb][m] = (float4_t)0.f;
    }

    // tiles [0, n_int) are visible to every row of the workgroup: keys below its first row's
    // position and below hi
    const int n_int = min(pmin + 1 >= 0 ? (pmin + 1) / kTile : 0, hi / kTile);

    // ---- this lane's positions in a slot ----
    // K operand (32-dim step pair c, 16-key block u): 16 source bytes of key row 16 u + li
    int kro[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) kro[c] = ((l & 15) >> 2) * kBlk + 256 * (l & 3) + 64 * (c ^ (l & 3)) + 16 * (l >> 4);
    // transposed V reads: 8 keys of one dim of block m (lanes 2 i, 2 i + 1 of a 16-lane group name tile
    // row tkey); odd row groups hold blocks 0..7 in their second half
    int vro_lo, vro_hi;
    {
        const int h = l >> 4, i = (l & 15) >> 1;
        const int tkey = i < 4 ? 4 * h + i : 12 + 4 * h + i;
        const int at = kFwImgV + ((tkey & 3) + 4 * (tkey >> 4)) * kBlk + 256 * h + 8 * (l & 1);
        vro_lo = at + ((h & 1) ? 128 : 0);
        vro_hi = at - ((h & 1) ? 128 : 0);
    }
    const int sro = kFwImgS + 16 * (l >> 4);  // scales of keys 16 u + 4 lg + j at + 64 u + 4 j

    uint4_t kr[3];       // K bytes of step i = 4 u + c: [i % 3]
    float4_t sc[4];      // k_scale of keys 4 lg .. (u = 0, 1), then v_scale
    auto kread = [&](const lds_u8* S, int i) __attribute__((always_inline)) {
        kr[i % 3] = *(const lds_uint4*)(S + kro[i & 3] + (i >> 2) * 4 * kBlk);
    };
    // the first reads of a tile: two K steps and the scales
    auto tile_start = [&](const lds_u8* S) __attribute__((always_inline)) {
        kread(S, 0);
        kread(S, 1);
#pragma unroll
        for (int j = 0; j < 4; ++j) sc[j] = *(const lds_float4*)(S + sro + 64 * j);
    };

    // ---- tile n from its slot S (its first reads are under way); mid() runs between the scores and the
    //      softmax, next() before the last products ----
    auto tile = [&](int n, const lds_u8* S, auto mid, auto next) __attribute__((always_inline)) {
        float4_t sacc[kRB][2];
        constexpr int kVAhead = kRB == 4 ? 2 : 4;  // (a narrow workgroup's products of an operand take half as long)
        int2_t vr[16];
        auto vread = [&](int m) __attribute__((always_inline)) {
            vr[m] = __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_int2*)(S + (m < 8 ? vro_lo : vro_hi) + 16 * m));
        };
        half8_t op = widen_i8x8_exact(kr[0].x, kr[0].y);
        settle_operand(op);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int u = i >> 2, c = i & 3;
            if (i < 6)
                kread(S, i + 2);
            else if (i == 6)
                vread(0);
            else {
#pragma unroll
                for (int m = 1; m < kVAhead; ++m) vread(m);
            }
            // the operand after the last is the first of V
            const unsigned w0 = i < 7 ? kr[(i + 1) % 3].x : (unsigned)vr[0].x, w1 = i < 7 ? kr[(i + 1) % 3].y : (unsigned)vr[0].y;
            if constexpr (kRB == 4) {
                if (c == 0)
                    op = score_products<true>(sacc[0][u], sacc[1][u], sacc[2][u], sacc[3][u], op, qop[0][2 * c], qop[1][2 * c],
                                              qop[2][2 * c], qop[3][2 * c], kr[i % 3].z, kr[i % 3].w);
                else
                    op = score_products<false>(sacc[0][u], sacc[1][u], sacc[2][u], sacc[3][u], op, qop[0][2 * c], qop[1][2 * c],
                                               qop[2][2 * c], qop[3][2 * c], kr[i % 3].z, kr[i % 3].w);
                op = score_products<false>(sacc[0][u], sacc[1][u], sacc[2][u], sacc[3][u], op, qop[0][2 * c + 1],
                                           qop[1][2 * c + 1], qop[2][2 * c + 1], qop[3][2 * c + 1], w0, w1);
            } else {
                if (c == 0)
                    op = score_products<true>(sacc[0][u], sacc[1][u], op, qop[0][2 * c], qop[1][2 * c], kr[i % 3].z, kr[i % 3].w);
                else
                    op = score_products<false>(sacc[0][u], sacc[1][u], op, qop[0][2 * c], qop[1][2 * c], kr[i % 3].z, kr[i % 3].w);
                op = score_products<false>(sacc[0][u], sacc[1][u], op, qop[0][2 * c + 1], qop[1][2 * c + 1], w0, w1);
            }
        }
        float ks[8], vs[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            ks[e] = sc[e >> 2][e & 3] * a.scale_log2;
            vs[e] = sc[2 + (e >> 2)][e & 3];
        }
        mid();
        settle_scores(sacc);
        float sv[kRB][8];
#pragma unroll
        for (int rb = 0; rb < kRB; ++rb)
#pragma unroll
            for (int e = 0; e < 8; ++e) sv[rb][e] = __builtin_fmaf(sacc[rb][e >> 2][e & 3], ks[e], nm_run[rb]);
        if constexpr (kWindow) {
            const int kb = seen.base(n);
            if (kb + kTile - 1 > pmin || (kb + kTile > seen.sinks && qabs + tok_last - kb >= win.window)) {
                // some row does not see all of the tile; keys that none sees may hold garbage scales: v_scale 0
                const int lane = lane_here(), key = kb + 4 * (lane >> 4);
                const lds_int* pos = (const lds_int*)(L + kFwLdsPos) + 16 * kRB * w + (lane & 15);
                const bool sinks = kb < seen.sinks;  // uniform
#pragma unroll
                for (int e = 0; e < 8; ++e) vs[e] = seen.has(key + 16 * (e >> 2) + (e & 3)) ? vs[e] : 0.f;
#pragma unroll
                for (int rb = 0; rb < kRB; ++rb) {
                    const int ahead = pos[16 * rb] - key;  // of the tile's first key of this lane; a row that is not there is at -1
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const int d = ahead - 16 * (e >> 2) - (e & 3);
                        bool sees = (unsigned)d < (unsigned)win.window;  // 0 <= d < window
                        if (sinks) sees = sees | ((d >= 0) & (key + 16 * (e >> 2) + (e & 3) < seen.sinks));
                        sv[rb][e] = sees ? sv[rb][e] : kNegInf;
                    }
                }
                // A seen key whose v_scale is not finite: 0 too, lest 0 times it reach the rows that do not see it. To those that do its
                // score says so, as +inf: NaN here and through the merge. (Rare and out of line: a select per score took 1 to 5 %.)
                float sum = vs[0] * 0.f;
#pragma unroll
                for (int e = 1; e < 8; ++e) sum = __builtin_fmaf(vs[e], 0.f, sum);
                if (__builtin_expect(__builtin_amdgcn_ballot_w64(sum != 0.f) != 0, 0)) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const bool finite = fabsf(vs[e]) < kInf;
#pragma unroll
                        for (int rb = 0; rb < kRB; ++rb) sv[rb][e] = finite || sv[rb][e] == kNegInf ? sv[rb][e] : kInf;
                        vs[e] = finite ? vs[e] : 0.f;
                    }
                }
            }
        } else if (n >= n_int) {  // the tile crosses the causal diagonal or seq_len
            const int key = n * kTile + 4 * (lane_here() >> 4);
            // keys past seq_len may hold garbage scales (even NaN): v_scale 0 makes their P' 0
#pragma unroll
            for (int e = 0; e < 8; ++e) vs[e] = key + 16 * (e >> 2) + (e & 3) < hi ? vs[e] : 0.f;
#pragma unroll
            for (int rb = 0; rb < kRB; ++rb) {
                const Row row = row_of(rb);
                const int last = row.valid ? min(hi - 1, qabs + row.tok) : -1;
#pragma unroll
                for (int e = 0; e < 8; ++e) sv[rb][e] = key + 16 * (e >> 2) + (e & 3) <= last ? sv[rb][e] : kNegInf;
            }
        }
        uint64_t need = 0;
#pragma unroll
        for (int rb = 0; rb < kRB; ++rb) {
            float mx = kNegInf;
#pragma unroll
            for (int e = 0; e < 8; ++e) mx = fmaxf(mx, sv[rb][e]);
            need |= __builtin_amdgcn_ballot_w64(mx > thr_run[rb]);
        }
        // rare: raise the running max of the rows that need it, shift their scores, rescale their
        // state (O is still zero while every row of a block is fresh: no rescale then)
        if (need != 0) {
#pragma unroll
            for (int rb = 0; rb < kRB; ++rb) {
                float mloc = kNegInf;
#pragma unroll
                for (int e = 0; e < 8; ++e) mloc = fmaxf(mloc, sv[rb][e]);
                const float mrow = xor_max(xor_max(mloc, 16), 32) - kPLog2;  // tile max relative to m
                const bool fresh = thr_run[rb] == kNegInf;
                const bool raise = fresh ? mrow > kNegInf : mrow > kLazy;
                const float shift = raise ? mrow : 0.f;
                const float alpha = fresh ? 0.f : __builtin_amdgcn_exp2f(-shift);
                nm_run[rb] -= shift;
                if (raise) thr_run[rb] = kLazy + kPLog2;
#pragma unroll
                for (int e = 0; e < 8; ++e) sv[rb][e] -= shift;
                l_run[rb] *= alpha;
                if (__builtin_amdgcn_ballot_w64(raise && !fresh) != 0) {
                    settle_values(oacc[rb]);
#pragma unroll
                    for (int m = 0; m < 16; m += 4)
                        agpr_scale4_via_lds(oacc[rb][m], oacc[rb][m + 1], oacc[rb][m + 2], oacc[rb][m + 3], alpha,
                                            lds_base + kLdsScr + 4096 * w + 16 * lane_here());
                }
            }
        }
        // p' = 2^sv, P' = p' * v_scale in fp16, O^T += V^T P'^T
        half8_t pop[kRB], plo[kRB];
#pragma unroll
        for (int rb = 0; rb < kRB; ++rb) {
            float psum = 0.f;
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
                const float p0 = __builtin_amdgcn_exp2f(sv[rb][e]);
                const float p1 = __builtin_amdgcn_exp2f(sv[rb][e + 1]);
                psum = e == 0 ? p0 : psum + p0;
                psum += p1;
                if constexpr (kExact) {
                    half2_t ph, pl;
                    split_fp16x2(p0, vs[e], p1, vs[e + 1], ph, pl);
                    pop[rb][e] = ph.x;
                    pop[rb][e + 1] = ph.y;
                    plo[rb][e] = pl.x;
                    plo[rb][e + 1] = pl.y;
                } else {
                    const half2_t ph = __builtin_convertvector((float2_t){p0 * vs[e], p1 * vs[e + 1]}, half2_t);
                    pop[rb][e] = ph.x;
                    pop[rb][e + 1] = ph.y;
                }
            }
            l_run[rb] += psum;
        }
        settle_weights<kExact>(pop, plo);
#pragma unroll
        for (int m = 0; m < 16; ++m) {
            if (m + kVAhead < 16) vread(m + kVAhead);
            if (m == (kRB == 4 ? 14 : 12)) next();
            if constexpr (kRB == 4) {
                if constexpr (kExact) value_products_only(oacc[0][m], oacc[1][m], oacc[2][m], oacc[3][m], op, plo[0], plo[1], plo[2], plo[3]);
                if (m < 15)
                    op = value_products(oacc[0][m], oacc[1][m], oacc[2][m], oacc[3][m], op, pop[0], pop[1], pop[2], pop[3],
                                        (unsigned)vr[m + 1].x, (unsigned)vr[m + 1].y);
                else
                    value_products_only(oacc[0][m], oacc[1][m], oacc[2][m], oacc[3][m], op, pop[0], pop[1], pop[2], pop[3]);
            } else {
                if constexpr (kExact) value_products_only(oacc[0][m], oacc[1][m], op, plo[0], plo[1]);
                if (m < 15)
                    op = value_products(oacc[0][m], oacc[1][m], op, pop[0], pop[1], (unsigned)vr[m + 1].x, (unsigned)vr[m + 1].y);
                else
                    value_products_only(oacc[0][m], oacc[1][m], op, pop[0], pop[1]);
            }
        }
    };

    const int nsteps = (t1 - t0 + kFwStep - 1) / kFwStep;
    const bool busy = 16 * kRB * w < nrow;  // a wave without rows only copies

    auto tile_loop = [&](auto lds_flag) __attribute__((always_inline)) {
        constexpr bool kLds = decltype(lds_flag)::value;
        // Starts of the 16-key blocks that this wave's copies of a step read: block u of the step's two tiles and
        // both blocks of tile u (for the scales); with the table in LDS its entries are read together.
        struct Blocks {
            int e[3];  // block u of tile 1 - u, then blocks 0 and 1 of tile u
        };
        const int u = w >> 1;
        auto step_tile = [&](int s, int j) __attribute__((always_inline)) { return min(t0 + kFwStep * s + j, t1 - 1); };
        auto fetch = [&](int s, Blocks& x) __attribute__((always_inline)) {
            if constexpr (kFast && kLds) {
                const int other = step_tile(s, 1 - u) - t0, own = step_tile(s, u) - t0;
                x.e[0] = pt.lds[2 * other + u];
                x.e[1] = pt.lds[2 * own];
                x.e[2] = pt.lds[2 * own + 1];
            }
        };
        auto block_base = [&](int entry, int n, int u) __attribute__((always_inline)) -> const int8_t* {
            if constexpr (kLds) {
                return gbase + ((int64_t)(unsigned)__builtin_amdgcn_readfirstlane(entry) << 3);
            } else {
                const int kb = kWindow ? seen.base(n) : n * kTile, klast = min(kb + kTile - 1, hi - 1);
                const int key0 = (kWindow ? seen.near(kb, kb + 16 * u) : min(kb + 16 * u, klast)) & ~15;
                const int lb = a.bs_shift >= 0 ? key0 >> a.bs_shift : key0 / a.block_size;
                return gbase + (int64_t)pt.glob[lb] * a.k_sb + (int64_t)(key0 - lb * a.block_size) * a.k_ss;
            }
        };
        auto row_base = [&](int n, int row) __attribute__((always_inline)) -> const int8_t* {
            const int key = kWindow ? seen.near(seen.base(n), seen.base(n) + row) : min(n * kTile + row, hi - 1);
            const int lb = a.bs_shift >= 0 ? key >> a.bs_shift : key / a.block_size;
            return gbase + pt.get<kLds>(lb) * a.k_sb + (int64_t)(key - lb * a.block_size) * a.k_ss;
        };
        // This wave's copies of step s: K and V blocks 2 w, 2 w + 1 of both tiles, and 32 scales of tile w >> 1
        // (k_scale for even w, v_scale for odd; lanes 32 (w & 1) .., the others copy nothing). The tile
        // past an odd end is the last one again, so that every step is kFwCopies copies.
        auto issue = [&](int s, int slot0, const Blocks& x) __attribute__((always_inline)) {
            const int k4 = 2 * (w & 1);
            // this lane's source bytes of a K and of a V copy (4 rows x 256 bytes each) and of a scale
            const int lh = lane_here(), qq = lh >> 4, c16 = lh & 15;
            const unsigned kvo = (unsigned)(kFast ? qq * a.k_ss : 0) + 16u * (unsigned)(c16 ^ (4 * qq));
            const unsigned vvo = (unsigned)(kFast ? 4 * qq * a.k_ss : 0) + 260u + 16u * (unsigned)(c16 ^ (8 * (qq & 1)));
            const unsigned first = lds_base + (unsigned)slot0;
            const int8_t *src, *b0, *b1;
            if constexpr (kFast) {
                b0 = block_base(x.e[1], step_tile(s, u), 0);
                b1 = block_base(x.e[2], step_tile(s, u), 1);
            }
#pragma unroll
            for (int j = 0; j < kFwStep; ++j) {
                const unsigned slot = first + (unsigned)(j * kFwSlot);
                if constexpr (kFast) {
                    const int8_t* base = j == u ? (u ? b1 : b0) : block_base(x.e[0], step_tile(s, 1 - u), u);
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        dma16_s(base + (int64_t)(4 * (k4 + h)) * a.k_ss, kvo, slot + kImgK + (2 * w + h) * kBlk);
                        dma16_s(base + (int64_t)(k4 + h) * a.k_ss, vvo, slot + kFwImgV + (2 * w + h) * kBlk);
                    }
                } else {
                    const int n = step_tile(s, j);
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        dma16_v<0>(row_base(n, 16 * u + 4 * (k4 + h) + qq) + kvo, slot + kImgK + (2 * w + h) * kBlk);
                        dma16_v<0>(row_base(n, 16 * u + (k4 + h) + 4 * qq) + vvo, slot + kFwImgV + (2 * w + h) * kBlk);
                    }
                }
            }
            if constexpr (kFast)
                src = ((lh >> 4) & 1 ? b1 : b0) + (unsigned)(c16 * a.k_ss);
            else
                src = row_base(step_tile(s, u), lh & 31);
            if ((lh >> 5) == (w & 1))
                dma4_v(reinterpret_cast<const int*>(src + (lh < 32 ? 256 : 516)), first + (unsigned)(u * kFwSlot + kFwImgS));
        };
        constexpr int kStepBytes = kFwStep * kFwSlot, kRingBytes = kFwRing * kFwSlot;
        Blocks blk;
        int slot_in = 0, slot_out = 0;  // ring positions (bytes) of the next step to copy and to compute
        auto issue_next = [&](int s) __attribute__((always_inline)) {
            fetch(s, blk);
            issue(s, slot_in, blk);
            slot_in = slot_in + kStepBytes == kRingBytes ? 0 : slot_in + kStepBytes;
        };
        for (int s = 0; s < min(nsteps, kFwAhead); ++s) issue_next(s);
        if constexpr (kWindow) load_q();
        const int ntl = t1 - t0;
        // Where the loop lies matters, because one wave per SIMD hides no instruction fetch, of 32 bytes each: the same loop at eight
        // places, 4 bytes apart, takes 3.65 to 3.75 ms for 2,560 tokens over 61,440 keys with
        // fp16 rows (4.68 to 4.79 exact), 2,048 exact and split 3.66 to 3.69 with fp32 rows and 3.58 to 3.65 with fp16 ones; over a window of 4,096
        // behind 30,000 keys 994 to 1,011 us for 8,192 tokens (exact), 120 to 123 for 512 split in two.
        // So it is placed, at what was best for each form; the alignment keeps it there whatever comes before. The padding runs once.
        constexpr int kPlace = kWindow ? (kSplit ? 5 : 1) : kExact ? (kSplit ? 0 : 3) : kSplit ? 1 : 4;
        asm volatile(".p2align 5\n\t.rept %0\n\ts_nop 0\n\t.endr" ::"n"(kPlace));
#pragma unroll 1
        for (int i = 0; i < ntl; ++i) {
            const int s = i / kFwStep;
            const bool first = i % kFwStep == 0;
            const lds_u8* S = L + slot_out;
            slot_out = slot_out + kFwSlot == kRingBytes ? 0 : slot_out + kFwSlot;
            if (first) {
                // this wave's copies of step s have landed; then every wave's, and step s - 1 is done
                if (s + 1 < nsteps)
                    wait_vm<kFwCopies>();
                else
                    wait_vm<0>();
                __syncthreads();
                tile_start(S);
            }
            const bool more = first && s + kFwAhead < nsteps;
            if (busy)
                tile(t0 + i, S, [&]() __attribute__((always_inline)) { if (more) issue_next(s + kFwAhead); },
                     // (after the last tile of a step these reads are thrown away)
                     [&]() __attribute__((always_inline)) { tile_start(L + slot_out); });
            else if (more)
                issue_next(s + kFwAhead);
        }
    };
    if (pt.in_lds)
        tile_loop(std::true_type{});
    else
        tile_loop(std::false_type{});

    // ---- normalise and store: out[b, tok, g G + hh, :]; with the keys split, the unnormalised
    //      partial O, the running max m and the sum l of the row instead ----
    if constexpr (kWindow && !kSplit) {
        // Through LDS (the ring is free once every wave is done): a lane has 4 dims of 16 rows' worth in each accumulator, and its stores
        // of 8 bytes take 7.4 us of a workgroup, whole rows side by side 4.0. Each thread works out one row's place.
        constexpr int kRow = 2 * kDim + 16;  // bytes of a row in LDS, its neighbours on other banks
        constexpr int kPart = kFwRing * kFwSlot / kFwWaves / 16 * 16;
        static_assert(16 * kRow <= kPart && kRows * 8 <= kFwWaves * 4096, "a row block's rows fit a wave's part of the ring, places the scratch");
        typedef _Float16 half4_t __attribute__((ext_vector_type(4)));
        typedef __attribute__((address_space(3))) half4_t lds_half4;
        lds_u64* place = (lds_u64*)(L + kLdsScr);
        __syncthreads();
        {
            const Row row = row_at(tid);
            place[tid] = (uint64_t)(((int64_t)first + row.tok) * a.o_st + (int64_t)(g * G + row.head) * a.o_sh);
        }
        __syncthreads();
        if (!busy) return;
        lds_u8* mine = L + w * kPart;
#pragma unroll
        for (int rb = 0; rb < kRB; ++rb) {
            const int lane = lane_here(), lg = lane >> 4, li = lane & 15;
            settle_values(oacc[rb]);
            const float l_row = xor_sum(xor_sum(l_run[rb], 16), 32);
            const float inv = l_row > 0.f ? 1.f / l_row : 0.f;
#pragma unroll
            for (int m = 0; m < 16; ++m) {
                const float4_t v = oacc[rb][m] * inv;
                *(lds_half4*)(mine + li * kRow + 32 * m + 8 * lg) = half4_t{(_Float16)v.x, (_Float16)v.y, (_Float16)v.z, (_Float16)v.w};
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) {  // two rows at a time
                const int at = 2 * j + (lane >> 5), r = 16 * kRB * w + 16 * rb + at;
                const uint4_t v = *(const lds_uint4*)(mine + at * kRow + 16 * (lane & 31));
                T* to = static_cast<T*>(a.out) + (int64_t)place[r] + 8 * (lane & 31);
                if (r < nrow) __builtin_memcpy(__builtin_assume_aligned(to, 8), &v, 16);
            }
        }
        return;
    }
#pragma unroll
    for (int rb = 0; rb < kRB; ++rb) {
        const int lg = l >> 4;
        settle_values(oacc[rb]);
        const float l_row = xor_sum(xor_sum(l_run[rb], 16), 32);
        const Row row = row_of(rb);
        if (!row.valid) continue;
        const int tok = row.tok, head = g * G + row.head;
        if constexpr (kSplit) {
            const int64_t pr = (((kWindow ? (int64_t)first : (int64_t)b * a.Sq) + tok) * a.Hq + head) * a.nsplit + split;
            float* prow = a.part_o + pr * kDim + 4 * lg;
#pragma unroll
            for (int m = 0; m < 16; ++m) *reinterpret_cast<float4_t*>(prow + 16 * m) = oacc[rb][m];
            if (lg == 0) {
                // (a row whose only scores here are NaN is not one that saw no key: +inf, lest the merge leave its sum out)
                a.part_m[pr] = kWindow && l_row != l_row ? kInf : thr_run[rb] == kNegInf ? kNegInf : kPLog2 - nm_run[rb];
                a.part_l[pr] = l_row;
            }
        } else {
            const float inv = l_row > 0.f ? 1.f / l_row : 0.f;
            T* orow = static_cast<T*>(a.out) + (int64_t)b * a.o_sb + (int64_t)tok * a.o_st + (int64_t)head * a.o_sh + 4 * lg;
#pragma unroll
            for (int m = 0; m < 16; ++m) store_out4<T>(orow + 16 * m, oacc[rb][m] * inv);
        }
    }
}

template <bool kFast, bool kExact, bool kSplit, class T>
__global__ void __launch_bounds__(kFwWaves * 64, 1) pd_prefill_wide_kernel(const FaParams a) {
    __shared__ __attribute__((aligned(16))) unsigned char lds[kFwLdsBytes];
    wide_workgroup<kFast, kExact, kSplit, T, false, kFwRB>(a, FaWindow{}, lds);
}

// Chunks whose rows see a sliding window and the first `sinks` keys: the row at position p sees key k <= p if p - k < window or
// k < sinks. A query tile streams the tiles that hold a key that one of its rows sees, those of the sinks, then the window's (window + 43
// keys for 256 rows of 6 heads), so a chunk's time goes with tokens x window, whatever lies before; pages that hold nothing
// seen are never addressed. kRB: 16-row blocks of a wave, 4 or 2 (pd_plan.hpp says which call takes which; two wait less for set-up,
// Q and stores, but each conversion then serves half the products). Tiles at the window's two ends and the last of the sinks are masked row by row, the others
// are not. Several sequences' rows lie one after the other; which a workgroup has is looked up on the device, so that a captured
// launch takes any batch of as many rows and sequences.
// What bounds it: for long chunks the tile loop, as in pd_prefill_wide_kernel: 8,192 tokens of 24 / 4 heads over a window of 4,096 620 to 640 us
// (619 GFLOP, 980 TFLOP/s; behind 30,000 keys, where every row sees a whole window, 785 us and 1,050), 2,048 tokens over windows of 512 / 1,024 /
// 2,048 / 4,096 / 8,192 57 / 86 / 144 / 262 / 460; kExact, which takes both halves of the weights through P.V, 791 us and 67 / 104 / 179 / 330 / 572.
// A workgroup's fixed part is about 12 us: block table, first copies, Q and stores. Short
// chunks pay it once and the merge: 64 tokens over 2,048 keys 31 us.
template <bool kFast, bool kExact, bool kSplit, int kRB>
__global__ void __launch_bounds__(kFwWaves * 64, 1) pd_window_kernel(const FaParams a, const FaWindow win) {
    __shared__ __attribute__((aligned(16))) unsigned char lds[kFwWindowLdsBytes];
    wide_workgroup<kFast, kExact, kSplit, _Float16, true, kRB>(a, win, lds);
}

// Log-sum-exp merge of a split windowed launch: a wave per (token, head) row, lane l owning dims 4 l .. 4 l + 3; M = max_s m_s,
// out = sum_s 2^(m_s - M) O_s / sum_s 2^(m_s - M) l_s, 0 for a row that saw no key. Rows outside the sequences, and those of
// sequences without keys, are left alone.
__global__ void __launch_bounds__(256) pd_window_combine_kernel(const FaParams a, const FaWindow win) {
    constexpr int kBatch = 16;
    const int lane = threadIdx.x & 63, head = (int)blockIdx.y;
    const int tok = (int)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    if (tok >= win.num_tokens) return;
    const int64_t base = ((int64_t)tok * a.Hq + head) * a.nsplit;
    // All that the row needs is asked for at once, one trip to memory for up to kBatch splits. (What a row that nobody owns reads lies in
    // the workspace too, whatever it holds.)
    const float4_t* po = reinterpret_cast<const float4_t*>(a.part_o + base * kDim) + lane;
    const float m_mine = lane < a.nsplit ? a.part_m[base + lane] : kNegInf;
    const float l_mine = lane < a.nsplit ? a.part_l[base + lane] : 0.f;
    float4_t o[kBatch];
    auto load = [&](int s0) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < kBatch; ++i)
            if (s0 + i < a.nsplit) o[i] = po[(int64_t)(s0 + i) * (kDim / 4)];
    };
    load(0);
    bool mine = false;
    for (int c = 0; c < win.num_seqs; c += 64) {
        const int i = min(c + lane, win.num_seqs - 1);
        const int first = win.query_start[i], end = win.query_start[i + 1], len = a.seq_lens[i];
        mine = mine | ((tok >= first) & (tok < end) & (len > 0));
    }
    if (__ballot(mine) == 0) return;
    float M = m_mine;
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) M = fmaxf(M, __shfl_xor(M, o, 64));
    const float w_mine = m_mine != kNegInf ? exp2f(m_mine - M) : 0.f;
    float L = w_mine * l_mine;
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) L += __shfl_xor(L, o, 64);
    float4_t acc = (float4_t)0.f;
    for (int s0 = 0; s0 < a.nsplit; s0 += kBatch) {
        if (s0 > 0) load(s0);
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            if (s0 + i >= a.nsplit) break;
            const float wi = __shfl(w_mine, s0 + i, 64);
            acc += wi != 0.f ? wi * o[i] : (float4_t)0.f;
        }
    }
    const float inv = L > 0.f ? 1.f / L : 0.f;
    _Float16* orow = static_cast<_Float16*>(a.out) + (int64_t)tok * a.o_st + (int64_t)head * a.o_sh;
    store_out4<_Float16>(orow + 4 * lane, acc * inv);
}

// ---------------------------------------------------------------------------------------
// host side

template <bool kSplit, class T>
static void launch_wide(const FaParams& p, dim3 grid, hipStream_t stream, bool fast, bool exact) {
    const dim3 block(kFwWaves * 64);
    if (fast && !exact)
        hipLaunchKernelGGL((pd_prefill_wide_kernel<true, false, kSplit, T>), grid, block, 0, stream, p);
    else if (!exact)
        hipLaunchKernelGGL((pd_prefill_wide_kernel<false, false, kSplit, T>), grid, block, 0, stream, p);
    else if (fast)
        hipLaunchKernelGGL((pd_prefill_wide_kernel<true, true, kSplit, T>), grid, block, 0, stream, p);
    else
        hipLaunchKernelGGL((pd_prefill_wide_kernel<false, true, kSplit, T>), grid, block, 0, stream, p);
}

hipError_t launch_prefill_wide(const FaParams& p, int batch, int heads_kv, int dtype, hipStream_t stream, bool exact) {
    const int64_t qtiles = ((int64_t)p.Sq * p.G + kFwRows - 1) / kFwRows;
    const dim3 grid((unsigned)(qtiles * p.nsplit), heads_kv, batch);
    const bool fast = fast_block_table(p.block_size, p.k_ss);
    if (dtype == PD_DTYPE_FP16) {
        if (p.nsplit == 1)
            launch_wide<false, _Float16>(p, grid, stream, fast, exact);
        else
            launch_wide<true, _Float16>(p, grid, stream, fast, exact);
    } else {
        if (p.nsplit == 1)
            launch_wide<false, float>(p, grid, stream, fast, exact);
        else
            launch_wide<true, float>(p, grid, stream, fast, exact);
    }
    return hipGetLastError();
}

template <bool kSplit, int kRB>
static void launch_window_rows(const FaParams& p, const FaWindow& w, dim3 grid, hipStream_t stream, bool fast, bool exact) {
    const dim3 block(kFwWaves * 64);
    if (fast && !exact)
        hipLaunchKernelGGL((pd_window_kernel<true, false, kSplit, kRB>), grid, block, 0, stream, p, w);
    else if (!exact)
        hipLaunchKernelGGL((pd_window_kernel<false, false, kSplit, kRB>), grid, block, 0, stream, p, w);
    else if (fast)
        hipLaunchKernelGGL((pd_window_kernel<true, true, kSplit, kRB>), grid, block, 0, stream, p, w);
    else
        hipLaunchKernelGGL((pd_window_kernel<false, true, kSplit, kRB>), grid, block, 0, stream, p, w);
}

hipError_t launch_window(const FaParams& p, const FaWindow& w, int rows, int heads_kv, hipStream_t stream, bool exact) {
    const dim3 grid((unsigned)(window_tiles(w.num_tokens, w.num_seqs, p.G, rows) * p.nsplit), heads_kv);
    const bool fast = fast_block_table(p.block_size, p.k_ss), narrow = rows != kFwRows;
    if (p.nsplit == 1) {
        narrow ? launch_window_rows<false, 2>(p, w, grid, stream, fast, exact) : launch_window_rows<false, 4>(p, w, grid, stream, fast, exact);
        return hipGetLastError();
    }
    narrow ? launch_window_rows<true, 2>(p, w, grid, stream, fast, exact) : launch_window_rows<true, 4>(p, w, grid, stream, fast, exact);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(pd_window_combine_kernel, dim3((unsigned)((w.num_tokens + 3) / 4), p.Hq), dim3(256), 0, stream, p, w);
    return hipGetLastError();
}

}  // namespace pd
