// Decode attention of a batch whose sequences share their first `prefix` keys. The prefix is read once for all rows of
// the batch instead of once per sequence; each sequence's own keys are read once for it; the parts are joined by their
// log-sum-exp.
//
// One launch of a workgroup per CU takes both, so that neither waits for the other: the first wp workgroups take
// pieces of the prefix, the others deal the own key tiles of all (sequence, kv head) among them as pd_balanced_kernel does.
// wp and the number of pieces are worked out on the device from the lengths (every workgroup, the same numbers), by rating
// each number of pieces: one lane, one number.
//   prefix   up to 32 rows of a kv head (tokens of the batch x its query heads) are one group of the decode's workgroup
//            (pd_partial.hpp) over a sequence made of the whole batch; more are tiles of 192 rows in the
//            prefill's (pd_prefill_body.hpp), where all of the workgroup's waves share one widening of each tile. A piece
//            is a run of the prefix's key tiles; it fills one segment of its rows.
//   own      the decode's workgroup over keys [prefix, seq_len) of one sequence; segments behind the prefix's. More than 32
//            rows of a sequence and kv head are two slices, which read the keys twice (three row blocks do not fit the
//            registers beside the deal).
// Segments of a row: [0, ns) the prefix's pieces, [ns, ..) the own ones, the rest up to the last marked empty; the last one's
// place holds ns, which the join needs: a sequence that does not hold the prefix and its query tokens behind it
// (seq_len - q_len < prefix) takes all of its keys as its own and leaves the prefix's segments out.
// The prefix's blocks are those of the first sequence that holds it.
//
// The 192-row tiles round P' = p v_scale once to fp16 as the default prefill does (11 bits: an error of about the final
// fp16 rounding's size; hi + lo would double their P.V products), the decode's workgroups carry hi + lo.
#include "pd_partial.hpp"
#include "pd_prefill_body.hpp"
#include "pth_dec.h"

namespace pd {

// Costs that the deal weighs, in 0.1 us: a workgroup's key tile and its set-up and merge.
constexpr unsigned kShTile = 8, kShSegment = 100;        // decode workgroup
constexpr unsigned kShWideTile = 18, kShWideSegment = 160;  // 192-row workgroup
constexpr unsigned kShMergeRows = 190;                    // (token, head) rows whose segments cost 0.1 us to write and read again
constexpr unsigned kShOwnUnits = 12;                      // set-up and merge of an own segment, in tiles (pd_balanced_kernel's line)
constexpr unsigned kShSnap = 6;

// kWide: the prefix in 192-row tiles; NRB: row blocks of the decode workgroups (both parts without kWide).
template <int NRB, bool kFast, bool kWide>
__global__ void __launch_bounds__(kThreads, 1) pd_shared_kernel(const SharedParams sp) {
    constexpr int kOwnLds = PartialLds<NRB, kFast>::kBytes;
    __shared__ __attribute__((aligned(16))) unsigned char lds[kWide && kFaLdsBytes > kOwnLds ? kFaLdsBytes : kOwnLds];
    const PartialParams& a = sp.p;
    const int lane = threadIdx.x & 63;
    const unsigned Hkv = (unsigned)(a.Hq / a.G), nwg = gridDim.x, wg = blockIdx.x;
    const int segs = a.nsplit - 1;  // and the note
    const unsigned slices = NRB == 2 && a.qmax * a.G > 32 ? 2u : 1u, groups = Hkv * slices;  // own items of a sequence

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
    total *= groups;
    const int T = max(0, min(sp.num_tokens, a.qsl[a.num_seqs]));
    const int tok_tile = kWide ? kFaRows / a.G : T;                   // query tokens of a prefix item
    const unsigned nrt = T > 0 ? (unsigned)((T + tok_tile - 1) / tok_tile) : 0u;
    const unsigned ptiles = first_holder >= 0 && sp.prefix > 0 ? (unsigned)((sp.prefix - 1) / kTile + 1) : 0u;
    const unsigned items = ptiles ? nrt * Hkv : 0u;

    // ---- how many workgroups take the prefix, and in how many pieces: lane i rates i + 1 pieces in one round of
    //      workgroups, the last 16 lanes one piece per item in 2 .. 17 rounds ----
    unsigned wp = 0, ns = 0;
    if (items) {
        constexpr unsigned kLanes = 48;
        const unsigned tile = kWide ? kShWideTile : kShTile;
        const unsigned seg = kWide ? kShWideSegment : kShSegment;
        const unsigned rounds = (unsigned)lane < kLanes ? 1u : (unsigned)lane - kLanes + 2u;
        const unsigned pieces = rounds == 1 ? (unsigned)lane + 1u : 1u;
        const unsigned w = (items * pieces + rounds - 1) / rounds;
        const bool own = total > 0;
        const bool can = w + (own ? 1u : 0u) <= nwg && pieces <= (unsigned)(segs - 2) && pieces <= ptiles;
        const unsigned prefix_us = rounds * (seg + (ptiles + pieces - 1) / pieces * tile) + (unsigned)(T * a.Hq) * pieces / kShMergeRows;
        const unsigned share = own && can ? max((total + nwg - w - 1) / (nwg - w), longest / (unsigned)(segs - (int)pieces - 1)) : 0u;
        const unsigned own_us = share * (kShTile) * 9 / 8;
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
            if constexpr (kWide) {
                FaParams f = {};
                f.q = a.q;
                f.q_sh = kDim;
                f.q_st = a.q_st;
                f.kc = a.kc;
                f.k_sb = a.k_sb;
                f.k_ss = a.k_ss;
                f.k_sh = a.k_sh;
                f.block_table = a.block_table;
                f.bt_stride = a.bt_stride;
                f.Hq = a.Hq;
                f.G = a.G;
                f.tok_per_wg = tok_tile;
                f.block_size = a.block_size;
                f.bs_shift = a.bs_shift;
                f.bt32 = sp.bt32;
                f.scale_log2 = a.scale_log2;
                f.nsplit = a.nseg;
                f.part_o = a.part_o;
                f.part_m = a.part_m;
                f.part_l = a.part_l;
                FaWork wk;
                wk.b = first_holder;
                wk.g = (int)g;
                wk.tq0 = (int)rt * tok_tile;
                wk.ntok = min(tok_tile, T - wk.tq0);
                wk.seq_len = sp.prefix;
                wk.qabs = 1 << 30;  // every key of the prefix is before every query token
                wk.qrow0 = 0;
                wk.orow0 = 0;
                wk.t0 = (int)first;
                wk.t1 = (int)last;
                wk.part = (int)piece;
                prefill_body<kFast, false, 3, _Float16>(f, wk, lds);
            } else {
                Work wk;
                wk.g = (int)g;
                wk.b = first_holder;
                wk.row0 = 0;
                wk.q0 = 0;
                wk.q_len = T;
                wk.ql = T;
                wk.seq_len = sp.prefix;
                wk.ctx0 = 1 << 30;
                wk.lo = 0;
                wk.seg = (int)piece;
                wk.tb = (int)first;
                wk.te = (int)last;
                wk.t_first = 0;
                wk.ntiles = (int)ptiles;
                wk.W = 0;
                wk.interleave = false;
                partial_body<NRB, kFast, true>(a, wk, lds);
            }
        }
        return;
    }

    // ---- the own keys: pd_balanced_kernel's deal over the other workgroups ----
    if (total == 0) return;
    const unsigned ow = wg - wp, on = nwg - wp, oitems = (unsigned)a.num_seqs * groups, cap = (unsigned)(segs - (int)ns);
    const unsigned share = max(max((total + on - 1) / on, (longest + cap - 2) / (cap - 1)), 2u);
    const unsigned nso = min(on / oitems, cap);
    const bool aligned = nso >= 1 && (longest + nso - 1) / nso <= share;
    const unsigned snap = min(kShSnap, share / 8), lead = kShOwnUnits + snap;
    unsigned at_seq, at_start, at_tiles;
    auto locate = [&](unsigned pos) __attribute__((always_inline)) {
        unsigned before = 0;
        for (int c = 0;; c += 64) {
            const unsigned t = c == 0 ? t0 : tiles_of(c + lane);
            const unsigned incl = c == 0 ? incl0 : wave_scan(units_of(t));
            const int k = __popcll(__ballot(groups * (before + incl) <= pos));
            if (k < 64) {
                at_seq = (unsigned)(c + k);
                at_tiles = (unsigned)__builtin_amdgcn_readlane((int)t, k);
                at_start = groups * (before + (unsigned)__builtin_amdgcn_readlane((int)incl, k) - units_of(at_tiles));
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
        Work wk;
        if (aligned) {
            const unsigned item = ow / nso;
            seg = ow - item * nso;
            wk.b = (int)(item / groups);
            wk.g = (int)(item - (unsigned)wk.b * groups);
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
        wk.seq_len = ((const_int_ptr)(uintptr_t)a.seq_lens)[wk.b];
        asm volatile("" ::"s"(wk.q0), "s"(q_end), "s"(wk.seq_len));
        wk.q_len = q_end - wk.q0;
        wk.lo = own_lo(wk.q_len, wk.seq_len);
        wk.ctx0 = wk.seq_len - wk.q_len;
        wk.ql = min(wk.q_len, a.qmax);
        wk.t_first = wk.lo / kTile;
        wk.ntiles = (wk.seq_len - 1) / kTile - wk.t_first + 1;
        if (aligned) {
            if (wk.q_len <= 0 || wk.seq_len <= 0) return;
            const unsigned per = ((unsigned)wk.ntiles + nso - 1) / nso;
            first = seg * per;
            last = min((unsigned)wk.ntiles, first + per);
            if (first >= last) return;
        }
        wk.row0 = slices > 1 ? 32 * (wk.g & 1) : 0;
        wk.g = slices > 1 ? wk.g >> 1 : wk.g;
        wk.seg = (int)(ns + seg);
        wk.tb = wk.t_first + (int)first;
        wk.te = wk.t_first + (int)last;
        wk.W = 0;
        wk.interleave = false;
        const int R = min(16 * NRB, wk.ql * a.G - wk.row0);
        if (R > 0) partial_body<NRB, kFast, true>(a, wk, lds);  // (a slice past the sequence's rows has none)
        if (last == (unsigned)wk.ntiles) {  // the item's last workgroup: no other segments, and the note
            const int spare = segs - wk.seg;
            for (int k = threadIdx.x; k < R * spare; k += kThreads) {
                const int r = k / spare, i = (wk.row0 + r) / a.G, hh = wk.row0 + r - i * a.G, s = wk.seg + 1 + (k - r * spare);
                const int64_t pr = ((int64_t)(wk.q0 + i) * a.Hq + (wk.g * a.G + hh)) * a.nseg + s;
                a.part_m[pr] = s == segs ? __builtin_bit_cast(float, ns) : kNegInf;
                a.part_l[pr] = 0.f;
            }
        }
        if (aligned || last < (unsigned)wk.ntiles) return;
        pos = (first ? pos - first - kShOwnUnits : pos) + units_of((unsigned)wk.ntiles);
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
    const int ns = __builtin_amdgcn_readlane(__builtin_bit_cast(int, m_ld), segs);
    const int from = len - (q_end - q_b) >= sp.prefix ? 0 : ns;
    const bool live = lane >= from && lane < segs && m_ld != kNegInf;
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

template <bool kFast, bool kWide>
static void launch_shared_rows(const SharedParams& s, int rows, int wgs, hipStream_t stream) {
    if (rows <= 16)
        hipLaunchKernelGGL((pd_shared_kernel<1, kFast, kWide>), dim3(wgs), dim3(kThreads), 0, stream, s);
    else
        hipLaunchKernelGGL((pd_shared_kernel<2, kFast, kWide>), dim3(wgs), dim3(kThreads), 0, stream, s);
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
    const int64_t all = (int64_t)x.num_tokens * p.G;  // rows of a kv head
    const int own = x.qmax * p.G;
    if (all <= 32)
        fast ? launch_shared_rows<true, false>(s, (int)all, cus, stream) : launch_shared_rows<false, false>(s, (int)all, cus, stream);
    else
        fast ? launch_shared_rows<true, true>(s, own, cus, stream) : launch_shared_rows<false, true>(s, own, cus, stream);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    const int64_t rows = (int64_t)x.num_tokens * x.heads_q;
    if (rows <= 1024)
        hipLaunchKernelGGL((pd_shared_combine_kernel<4>), dim3((unsigned)rows), dim3(256), 0, stream, s);
    else
        hipLaunchKernelGGL((pd_shared_combine_kernel<1>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, stream, s);
    return hipGetLastError();
}

}  // namespace pd
