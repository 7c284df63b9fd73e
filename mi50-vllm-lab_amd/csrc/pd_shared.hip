// Decode attention of a batch whose sequences share their first `prefix` keys. The prefix is read once for all rows of
// the batch instead of once per sequence; each sequence's own keys are read once for it; the parts are joined by their
// log-sum-exp.
//
// One launch of a workgroup per CU takes both, so that neither waits for the other: the first wp workgroups take
// pieces of the prefix, the others deal the own key tiles of all (sequence, kv head) among them as pd_balanced_kernel does.
// wp and the number of pieces are worked out on the device from the lengths (every workgroup, the same numbers), by rating
// each number of pieces: one lane, one number.
//   prefix   tiles of up to 128 or 256 (token of the batch, query head of a kv head) rows. A piece is a run of the prefix's key
//            tiles; it fills one segment of its rows.
//   own      the rows of one sequence and kv head over its keys [prefix, seq_len); segments behind the prefix's.
// Both in the same workgroup form (pd_shared_body.hpp).
// Segments of a row: [0, ns) the prefix's pieces, [ns, ns + n) the own ones; the last one's place holds both numbers, a note that
// spares marking the others empty and tells the join which to leave out: a sequence that does not hold the prefix and its
// query tokens behind it (seq_len - q_len < prefix) takes all of its keys as its own.
// The prefix's blocks are those of the first sequence that holds it.
//
// P' = p v_scale enters P.V as fp16 hi + lo, as in the decode: rounded once it would cost an error of about the final fp16 rounding's
// size (2.9e-4 against 64 bits, 2-norm, where that rounding alone makes 2.1e-4). The 16 more MFMAs per row block, of 48 a
// tile, cost 19 % of the largest batch (128 sequences over 61,440 keys 254 us without, 303 with) and nothing where memory or set-up bounds.
//
// What bounds it (gfx950, both launches, us; 24 / 4 heads unless said): 128 sequences of 64 to 2,048 keys behind 61,440 shared ones 303.
// The prefix alone takes 265 and its join 14: with both terms of P' 1,090 TFLOP/s of MFMAs, 94 % of the rate of a large matrix
// product. The own keys alone take 65 (4.7 TB/s: bound by memory); a CU streams at most 20 bytes a ns, so the deal counts
// 1 us for an own tile and both kinds of work finish together. 32 sequences over 8,192: 37, 12 of them set-up of the pieces, their
// partials (12 MB) and the join. 4 over 2,048: 13.4, five dependent trips to memory and a second launch.
#include "pd_shared_body.hpp"
#include "pth_dec.h"

namespace pd {

// Costs that the deal weighs, in 0.1 us: a key tile of an own workgroup with one wave in rows (20 bytes a ns) or four, of a prefix
// workgroup with one or two row blocks per wave, a prefix piece's set-up and end. Fitted to 46 batches of 10 to 86 sequences
// (13 instead of 15 for the prefix 2 % slower on average and up to 10, 10 instead of 13 for four waves up to 25); set-up
// of 60 to 100 and 250 to 400 rows below change no batch by more than 4 %.
constexpr unsigned kShTile = 10, kShTileFour = 13;
constexpr unsigned kShPrefixTile1 = 15, kShPrefixTile2 = 25;
constexpr unsigned kShPrefixSegment = 80;
constexpr unsigned kShMergeRows = 400;  // (token, head) rows whose segments cost 0.1 us to write and read again
constexpr unsigned kShOwnUnits = 12;    // set-up and merge of an own segment, in tiles (pd_balanced_kernel's line)
constexpr unsigned kShSnap = 6;         // a share's end moves to an item's that is this many units away (pd_balanced_kernel's too)

// OW: waves in rows of the own keys' workgroups (one row block each); PB: row blocks of the prefix's waves.
template <int OW, bool kFast, int PB>
__global__ void __launch_bounds__(kSwThreads, 1) pd_shared_kernel(const SharedParams sp) {
    __shared__ __attribute__((aligned(16))) unsigned char lds[kSwLds];
    constexpr int NB = 8 * PB;  // row blocks of a prefix tile
    const PartialParams& a = sp.p;
    const int lane = threadIdx.x & 63;
    const unsigned Hkv = (unsigned)(a.Hq / a.G), nwg = gridDim.x, wg = blockIdx.x;
    const int segs = a.nsplit - 1;  // and the note

    // ---- the batch: own tiles of each sequence, the first that holds the prefix ----
    auto own_lo = [&](int q_len, int len) __attribute__((always_inline)) { return len - q_len >= sp.prefix ? sp.prefix : 0; };
    auto tiles_of = [&](int i) __attribute__((always_inline)) -> unsigned {
        const int c = min(i, a.num_seqs - 1);
        const int q_len = a.qsl[c + 1] - a.qsl[c], len = a.seq_lens[c];
        return i < a.num_seqs && q_len > 0 && len > 0 ? (unsigned)((len - 1) / kTile - own_lo(q_len, len) / kTile + 1) : 0u;
    };
    auto holds = [&](int i) __attribute__((always_inline)) -> bool {
        const int c = min(i, a.num_seqs - 1);
        const int q_len = a.qsl[c + 1] - a.qsl[c], len = a.seq_lens[c];
        return i < a.num_seqs && q_len > 0 && len - q_len >= sp.prefix;
    };
    auto units_of = [&](unsigned t) __attribute__((always_inline)) { return t ? t + kShOwnUnits : 0u; };
    const unsigned t0 = tiles_of(lane), incl0 = wave_scan(units_of(t0));
    unsigned total = (unsigned)__builtin_amdgcn_readlane((int)incl0, 63), longest = wave_umax(t0);
    uint64_t who = __ballot(holds(lane));
    int first_holder = who ? __builtin_ctzll(who) : -1;
    for (int c = 64; c < a.num_seqs; c += 64) {
        const unsigned t = tiles_of(c + lane);
        total += (unsigned)__builtin_amdgcn_readlane((int)wave_scan(units_of(t)), 63);
        longest = max(longest, wave_umax(t));
        if (first_holder < 0) {
            who = __ballot(holds(c + lane));
            if (who) first_holder = c + __builtin_ctzll(who);
        }
    }
    total *= Hkv;
    const int T = max(0, min(sp.num_tokens, a.qsl[a.num_seqs]));
    // rows of a kv head, their tiles, and the rows of a tile: equal shares in whole waves
    const unsigned prows = (unsigned)(T * a.G), nrt = (prows + 16 * NB - 1) / (16 * NB);
    const unsigned trows = nrt ? ((prows + nrt - 1) / nrt + 16 * PB - 1) / (16 * PB) * (16 * PB) : 0u;
    const unsigned ptiles = first_holder >= 0 && sp.prefix > 0 ? (unsigned)((sp.prefix - 1) / kTile + 1) : 0u;
    const unsigned items = ptiles ? nrt * Hkv : 0u;

    // ---- how many workgroups take the prefix, and in how many pieces: lane i rates i + 1 pieces in one round of
    //      workgroups, the last 16 lanes one piece per item in 2 .. 17 rounds ----
    unsigned wp = 0, ns = 0;
    if (items) {
        constexpr unsigned kLanes = 48;
        constexpr unsigned tile = PB == 1 ? kShPrefixTile1 : kShPrefixTile2, seg = kShPrefixSegment;
        const unsigned rounds = (unsigned)lane < kLanes ? 1u : (unsigned)lane - kLanes + 2u;
        const unsigned pieces = rounds == 1 ? (unsigned)lane + 1u : 1u;
        const unsigned w = (items * pieces + rounds - 1) / rounds;
        const bool own = total > 0;
        const bool can = w + (own ? 1u : 0u) <= nwg && pieces <= (unsigned)(segs - 2) && pieces <= ptiles;
        const unsigned prefix_us = rounds * (seg + (ptiles + pieces - 1) / pieces * tile) + (unsigned)(T * a.Hq) * pieces / kShMergeRows;
        const unsigned share = own && can ? max((total + nwg - w - 1) / (nwg - w), longest / (unsigned)(segs - (int)pieces - 1)) : 0u;
        const unsigned own_us = share * (OW == 1 ? kShTile : kShTileFour);
        const unsigned cost = can ? min(max(prefix_us, own_us), 0x3ffffffu) : 0x3ffffffu;
        // the cheapest (the lowest lane of equal ones); more items than 17 rounds take: as many rounds as it needs
        const unsigned best = ~wave_umax(~((cost << 6) | (unsigned)lane)) & 63u;
        if ((unsigned)__builtin_amdgcn_readlane((int)cost, (int)best) == 0x3ffffffu) {
            ns = 1;
            wp = own ? max(1u, nwg - nwg / 8) : nwg;
            if (wp >= nwg && own) wp = nwg > 1 ? nwg - 1 : 1;
        } else {
            ns = (unsigned)__builtin_amdgcn_readlane((int)pieces, (int)best);
            wp = (unsigned)__builtin_amdgcn_readlane((int)w, (int)best);
        }
    }

    // ---- the prefix ----
    if (wg < wp) {
        for (unsigned x = wg; x < items * ns; x += wp) {
            if (x != wg) __syncthreads();  // the blocks of the piece before have been read
            const unsigned rt = x % nrt, gp = x / nrt, piece = gp % ns, g = gp / ns;
            const unsigned first = piece * ptiles / ns, last = (piece + 1) * ptiles / ns;
            SharedWork wk;
            wk.g = (int)g;
            wk.b = first_holder;
            wk.q0 = 0;
            wk.pos0 = 1 << 30;  // every key of the prefix comes before every query token
            wk.lo = 0;
            wk.hi = sp.prefix;
            wk.row0 = (int)(rt * trows);
            wk.nrow = min((int)trows, (int)prows - wk.row0);
            wk.t0 = (int)first;
            wk.t1 = (int)last;
            wk.seg = (int)piece;
            shared_body<PB, 8, kFast>(sp, wk, lds);
        }
        return;
    }

    // ---- the own keys: pd_balanced_kernel's deal over the other workgroups ----
    if (total == 0) return;
    const unsigned ow = wg - wp, on = nwg - wp, oitems = (unsigned)a.num_seqs * Hkv, cap = (unsigned)(segs - (int)ns);
    const unsigned share = max(max((total + on - 1) / on, (longest + cap - 2) / (cap - 1)), 2u);
    const unsigned nso = min(on / oitems, cap);
    const bool aligned = nso >= 1 && (longest + nso - 1) / nso <= share;
    const unsigned snap = min(kShSnap, share / 8), lead = kShOwnUnits + snap;
    unsigned at_seq, at_start, at_tiles;
    auto locate = [&](unsigned pos) __attribute__((always_inline)) {
        int lane = threadIdx.x;
        asm volatile("" : "+v"(lane));  // (keeps the compiler from holding addresses in registers through the workgroups' bodies)
        lane &= 63;
        unsigned before = 0;
        for (int c = 0;; c += 64) {
            const unsigned t = tiles_of(c + lane);
            const unsigned incl = wave_scan(units_of(t));
            const int k = __popcll(__ballot(Hkv * (before + incl) <= pos));
            if (k < 64) {
                at_seq = (unsigned)(c + k);
                at_tiles = (unsigned)__builtin_amdgcn_readlane((int)t, k);
                at_start = Hkv * (before + (unsigned)__builtin_amdgcn_readlane((int)incl, k) - units_of(at_tiles));
                return;
            }
            before += (unsigned)__builtin_amdgcn_readlane((int)incl, 63);
        }
    };
    auto bound = [&](unsigned x) __attribute__((always_inline)) -> unsigned {
        const unsigned raw = (unsigned)min((uint64_t)x * share, (uint64_t)total);
        if (raw == 0 || raw == total) return raw;
        locate(raw);
        const unsigned units = units_of(at_tiles), off = (raw - at_start) % units;
        if (off <= lead) return raw - off;
        return units - off <= snap ? raw + (units - off) : raw;
    };
    unsigned pos = 0, end = 0;
    if (!aligned) {
        pos = bound(ow);
        end = bound(ow + 1);
        if (pos >= end) return;
    } else if (ow >= oitems * nso) {
        return;
    }
    while (true) {
        unsigned first, last, seg;
        SharedWork wk;
        if (aligned) {
            const unsigned item = ow / nso;
            seg = ow - item * nso;
            wk.b = (int)(item / Hkv);
            wk.g = (int)(item - (unsigned)wk.b * Hkv);
        } else {
            locate(pos);
            const unsigned units = units_of(at_tiles), g = (pos - at_start) / units, item = at_start + g * units;
            first = pos - item <= lead ? 0 : pos - item - kShOwnUnits;
            last = end - item >= units ? at_tiles : end - item - kShOwnUnits;
            seg = ow - min(item + lead, item + units - 1) / share;
            wk.b = (int)at_seq;
            wk.g = (int)g;
        }
        wk.q0 = ((const_int_ptr)(uintptr_t)a.qsl)[wk.b];
        const int q_end = ((const_int_ptr)(uintptr_t)a.qsl)[wk.b + 1];
        wk.hi = ((const_int_ptr)(uintptr_t)a.seq_lens)[wk.b];
        asm volatile("" ::"s"(wk.q0), "s"(q_end), "s"(wk.hi));
        const int q_len = q_end - wk.q0;
        wk.lo = own_lo(q_len, wk.hi);
        wk.pos0 = wk.hi - q_len;
        wk.row0 = 0;
        wk.nrow = min(q_len, a.qmax) * a.G;
        const int t_first = wk.lo / kTile;
        const unsigned ntiles = (unsigned)((wk.hi - 1) / kTile - t_first + 1);
        if (aligned) {
            if (q_len <= 0 || wk.hi <= 0) return;
            const unsigned per = (ntiles + nso - 1) / nso;
            first = seg * per;
            last = min(ntiles, first + per);
            if (first >= last) return;
        }
        wk.seg = (int)(ns + seg);
        wk.t0 = t_first + (int)first;
        wk.t1 = t_first + (int)last;
        shared_body<1, OW, kFast>(sp, wk, lds);
        if (last == ntiles && (int)threadIdx.x < wk.nrow) {  // the item's last workgroup knows how many there are: the note
            const int r = (int)threadIdx.x, i = r / a.G, hh = r - i * a.G;
            a.part_m[((int64_t)(wk.q0 + i) * a.Hq + (wk.g * a.G + hh)) * a.nseg + segs] = __builtin_bit_cast(float, ns | (ns + seg + 1) << 8);
        }
        if (aligned || last < ntiles) return;
        pos = (first ? pos - first - kShOwnUnits : pos) + units_of(ntiles);
        if (pos >= end) return;
        __syncthreads();
    }
}

// Joins the segments of each (token, head) row: M = max m, out = sum 2^(m - M) O / sum 2^(m - M) l over the segments that hold
// anything, without the prefix's where the row's sequence does not hold it. kWaves waves of a workgroup share a row (each
// takes every kWaves-th live segment; lane l dims 4 l .. 4 l + 3).
template <int kRowWaves>
__global__ void __launch_bounds__(256) pd_shared_combine_kernel(const SharedParams sp) {
    constexpr int kBatch = 4;
    __shared__ __attribute__((aligned(16))) float4_t sums[kRowWaves > 1 ? 4 : 1][64];
    const PartialParams& a = sp.p;
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t row = (int64_t)blockIdx.x * (4 / kRowWaves) + w / kRowWaves;
    const int part = w % kRowWaves, segs = a.nsplit - 1;
    if (row >= (int64_t)sp.num_tokens * a.Hq) return;  // (with several waves per row: the whole workgroup)
    const int tok = (int)(row / a.Hq), head = (int)(row - (int64_t)tok * a.Hq);
    // the segments' m and l, requested before the lookup of the sequence
    const float m_ld = a.part_m[row * a.nseg + min(lane, segs)], l_ld = a.part_l[row * a.nseg + min(lane, segs)];
    int b = 0;
    for (int i0 = 0; i0 < a.num_seqs; i0 += 64) {
        const int i = i0 + lane + 1;
        b += __popcll(__ballot(i <= a.num_seqs && a.qsl[min(i, a.num_seqs)] <= tok));
    }
    const int bq = __builtin_amdgcn_readfirstlane(min(b, a.num_seqs - 1));
    const int q_b = ((const_int_ptr)(uintptr_t)a.qsl)[bq], q_end = ((const_int_ptr)(uintptr_t)a.qsl)[bq + 1];
    const int len = ((const_int_ptr)(uintptr_t)a.seq_lens)[bq];
    if (!(b < a.num_seqs && tok >= q_b && len > 0 && tok - q_b < a.qmax)) return;  // (uniform over the row's waves)
    const int note = __builtin_amdgcn_readlane(__builtin_bit_cast(int, m_ld), segs);
    const int from = len - (q_end - q_b) >= sp.prefix ? 0 : note & 0xff;
    const bool live = lane >= from && lane < note >> 8 && m_ld != kNegInf;
    uint64_t mask = __ballot(live);
    float M = live ? m_ld : kNegInf;
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) M = fmaxf(M, __shfl_xor(M, o, 64));
    const float f = live ? __builtin_amdgcn_exp2f(m_ld - M) : 0.f;
    float L = f * (live ? l_ld : 0.f);
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) L += __shfl_xor(L, o, 64);
    float4_t acc = (float4_t)0.f;
    const float4_t* po = reinterpret_cast<const float4_t*>(a.part_o + row * a.nseg * kDim) + lane;
    for (int i = 0; i < part && mask; ++i) mask &= mask - 1;
    while (mask) {
        float4_t o[kBatch];
        float wt[kBatch];
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
            const int s = mask ? __builtin_ctzll(mask) : 0;
            wt[k] = mask ? __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, f), s)) : 0.f;
            o[k] = (float4_t)0.f;
            if (mask) o[k] = po[(int64_t)s * (kDim / 4)];
#pragma unroll
            for (int i = 0; i < kRowWaves; ++i) mask &= mask - 1;
        }
#pragma unroll
        for (int k = 0; k < kBatch; ++k) acc += wt[k] * o[k];
    }
    if constexpr (kRowWaves > 1) {
        sums[w][lane] = acc;
        __syncthreads();
        if (part != 0) return;
#pragma unroll
        for (int i = 1; i < kRowWaves; ++i) acc += sums[w + i][lane];
    }
    const float inv = L > 0.f ? 1.f / L : 0.f;
    typedef _Float16 half4_t __attribute__((ext_vector_type(4)));
    const half4_t h = {(_Float16)(acc.x * inv), (_Float16)(acc.y * inv), (_Float16)(acc.z * inv), (_Float16)(acc.w * inv)};
    __builtin_memcpy(sp.out + (int64_t)tok * sp.o_st + (int64_t)head * sp.o_sh + 4 * lane, &h, 8);
    if (sp.lse && lane == 0) sp.lse[row] = L > 0.f ? (M + __builtin_amdgcn_logf(L)) * 0.6931471805599453f : kNegInf;
}

// ---------------------------------------------------------------------------------------
// host side

template <bool kFast, int PB>
static void launch_shared_rows(const SharedParams& s, int rows, int wgs, hipStream_t stream) {
    if (rows <= 16)
        hipLaunchKernelGGL((pd_shared_kernel<1, kFast, PB>), dim3(wgs), dim3(kSwThreads), 0, stream, s);
    else
        hipLaunchKernelGGL((pd_shared_kernel<4, kFast, PB>), dim3(wgs), dim3(kSwThreads), 0, stream, s);
}

// Whether the prefix's waves take two row blocks, for `rows` rows of a kv head. Two read and widen every key half as often; one
// makes smaller pieces and tiles. us with one and two, 24 / 4 heads: 192 rows over 8,192 keys 37.6 and 39.0, over 61,440 109.6 and 111;
// 258 over 32,768 93.7 and 104; 384 over 16,384 69.8 and 75.8, over 61,440 169 and 179; 510 over 16,384 89.5 and 89.6, over 32,768
// 136 and 132, over 61,440 224 and 200; 768 over 8,192 66.9 and 72.5, over 16,384 99.2 and 99.3, over 32,768 181 and 161, over 61,440
// 309 and 275; 1,020 over 8,192 108 and 115, over 32,768 256 and 232. (For up to 64 rows the own keys' form, tiles in LDS that four waves
// share, gains 6 % over 32,768 keys and nothing below; it is not here.)
static bool two_row_blocks(int64_t rows, int prefix) {
    return rows > 384 && prefix > 16384;
}

hipError_t launch_shared(const LaunchArgs& x, int prefix, int bt32, hipStream_t stream) {
    SharedParams s = {};
    PartialParams& p = s.p;
    p.q = static_cast<const _Float16*>(x.q);
    p.q_st = x.q_st;
    p.kc = static_cast<const int8_t*>(x.kc);
    p.k_sb = x.k_sb;
    p.k_ss = x.k_ss;
    p.k_sh = x.k_sh;
    p.block_table = x.block_table;
    p.bt_stride = x.bt_stride;
    p.seq_lens = x.seq_lens;
    p.qsl = x.qsl;
    p.block_size = x.block_size;
    p.scale_log2 = x.scale * 1.4426950408889634f;
    p.part_o = x.part_o;
    p.part_m = x.part_m;
    p.part_l = x.part_l;
    p.nseg = x.nseg;
    p.nsplit = x.nseg < 64 ? x.nseg : 64;  // (the join holds a segment per lane)
    p.G = x.heads_q / x.heads_kv;
    p.qmax = x.qmax;
    p.Hq = x.heads_q;
    p.causal = 1;
    p.bs_shift = (x.block_size & (x.block_size - 1)) == 0 ? __builtin_ctz((unsigned)x.block_size) : -1;
    p.num_seqs = x.num_seqs;
    p.rslices = 1;
    s.num_tokens = x.num_tokens;
    s.prefix = prefix;
    s.bt32 = bt32;
    s.out = static_cast<_Float16*>(x.out);
    s.o_st = x.o_st;
    s.o_sh = x.o_sh;
    s.lse = x.lse;
    const int known = compute_units(stream), cus = known > 1 ? known : 256;
    const bool fast = fast_block_table(x.block_size, x.k_ss);
    const int rows_own = x.qmax * p.G;
    const bool two = fast && two_row_blocks((int64_t)x.num_tokens * p.G, prefix);
    two ? launch_shared_rows<true, 2>(s, rows_own, cus, stream)
        : fast ? launch_shared_rows<true, 1>(s, rows_own, cus, stream) : launch_shared_rows<false, 1>(s, rows_own, cus, stream);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    // four waves share a row where rows are few: 96 rows 13.8 us (both launches), one wave 16.5; 504 20.4 and 21; 768 39 both; 1,056 50 both
    const int64_t rows = (int64_t)x.num_tokens * x.heads_q;
    if (rows <= 768)
        hipLaunchKernelGGL((pd_shared_combine_kernel<4>), dim3((unsigned)rows), dim3(256), 0, stream, s);
    else
        hipLaunchKernelGGL((pd_shared_combine_kernel<1>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, stream, s);
    return hipGetLastError();
}

}  // namespace pd
