// Eviction from the cache by running attention weights: per (sequence, kv head) the last `recent` keys and the
// keep - recent others with the largest weights stay (equal weights: the lowest key first; NaN counts as the largest), in the
// order of their positions. pd_evict_select_kernel finds them and writes their numbers; pd_evict_copy_kernel copies their
// weights and 520-byte rows, the rows into the blocks of another table, so blocks that several sequences share stay as they
// are and no row is read after it was written over.
//
// The select is one workgroup per (sequence, kv head). A weight's bits become an unsigned number of the same order; the
// range [lo, hi] of numbers that holds the smallest weight to keep is narrowed by histograms of 2,048 parts, 11 bits at a time,
// until it is one value or is kept whole; once few keys lie in it they go on as a list. Then each wave's kept keys are
// counted (the list knows them by wave), the counts are summed over the waves, and each wave writes its kept keys in
// order: their places are known without a barrier. Rows of up to 65,536 keys are read once, all loads in flight together, and
// stay in registers (kPer a lane) through all passes; longer ones are read again in every pass. A pass over a row costs its
// CU 4 waves x kPer x its instructions on each SIMD: keys of weight 0, which sums that no row has added to
// share, and lanes that agree on a part do not queue for one counter.
//
// What bounds it, us: 8 sequences of 1,000 to 6,000 keys (4 kv heads, 2,048 kept) select 7.3 to 8.7, latency of its passes, and copy 9.6, 68 MB
// at 7 TB/s from and to caches; one of 61,440 (2 heads, 8,000 kept) select 32, the instructions of the one CU that a row
// has, and copy 6. One of 131,072, read again in every pass, 83 in all (16,000 kept: 87).
#include "pd_tile.hpp"
#include "pth_dec.h"

namespace pd {

constexpr int kEvWaves = 16;
constexpr int kEvThreads = 64 * kEvWaves;
constexpr int kEvBins = 2048;
constexpr int kEvList = 4 * kEvThreads;

// Order of the weights as unsigned numbers: -0 as 0, NaN above all.
__device__ __forceinline__ unsigned weight_order(float x) {
    if (x != x) return 0xffffffffu;
    const unsigned u = __builtin_bit_cast(unsigned, x + 0.f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// kPer: keys of a lane; kOnce: the row has at most kPer x kEvThreads candidates and is read once.
template <int kPer, bool kOnce>
__global__ void __launch_bounds__(kEvThreads) pd_evict_select_kernel(const EvictParams a) {
    __shared__ unsigned hist[kEvBins];
    __shared__ unsigned part[2][kEvWaves];
    __shared__ unsigned found[4];
    __shared__ unsigned list[kEvList];
    __shared__ unsigned char list_wave[kEvList];
    const int g = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, l = tid & 63;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = max(0, min(a.seq_lens[b], a.max_keys)), keep = a.keep;
    const float* wsrc = a.weights + (int64_t)b * a.w_sb + (int64_t)g * a.w_sh;
    int* kept = a.kept + ((int64_t)b * a.Hkv + g) * keep;
    if (g == 0 && tid == 0) a.new_lens[b] = min(n, keep);
    if (n <= keep) {  // everything stays
        for (int j = tid; j < keep; j += kEvThreads) kept[j] = j < n ? j : -1;
        return;
    }
    const int recent = min(a.recent, keep), nc = n - recent;  // candidates [0, nc)
    const unsigned want = (unsigned)(keep - recent);           // of which so many stay
    for (int j = tid; j < recent; j += kEvThreads) kept[want + j] = nc + j;
    if (want == 0) return;

    // This wave's run of keys [t0, t1), 64 x kPer of them at a time: lane l has t + 64 i. Past the end 0, which no weight is.
    const int per = ((nc + kEvWaves - 1) / kEvWaves + 63) / 64 * 64;
    const int t0 = min(nc, w * per), t1 = min(nc, t0 + per);
    unsigned u[kPer];
    auto load = [&](int t) __attribute__((always_inline)) {
        const float* x = wsrc + t + l;
        const int lanes = t1 - t - l;  // keys from this lane's first on
#pragma unroll
        for (int i = 0; i < kPer; ++i) u[i] = 64 * i < lanes ? __builtin_bit_cast(unsigned, x[64 * i]) : 0u;
        int again = lanes;  // (a value of its own: kPer comparisons kept from the loads do not fit the scalar registers)
        asm volatile("" : "+v"(again));
#pragma unroll
        for (int i = 0; i < kPer; ++i) u[i] = 64 * i < again ? weight_order(__builtin_bit_cast(float, u[i])) : 0u;
    };
    // f(t, u of key t + l) over the run, in order; whole waves
    auto each = [&](auto f) __attribute__((always_inline)) {
        if constexpr (kOnce) {
            int chunks = (t1 - t0 + 63) / 64;
            asm volatile("" : "+s"(chunks));  // (kPer comparisons kept from pass to pass do not fit the scalar registers)
#pragma unroll
            for (int i = 0; i < kPer; ++i)
                if (i < chunks) f(t0 + 64 * i, u[i]);
        } else {
            for (int t = t0; t < t1; t += 64 * kPer) {
                load(t);
                const int chunks = (t1 - t + 63) / 64;
#pragma unroll
                for (int i = 0; i < kPer; ++i)
                    if (i < chunks) f(t + 64 * i, u[i]);
            }
        }
    };
    if constexpr (kOnce) load(t0);

    constexpr unsigned kZero = 0x80000000u;  // weight_order(0)
    // Adds the keys x of a wave (`in`: lanes that count) to their parts.
    auto count_into = [&](unsigned bin, bool in) __attribute__((always_inline)) {
        const uint64_t who = __ballot(in);
        if (who == 0) return;
        const unsigned lead = (unsigned)__builtin_amdgcn_readlane((int)bin, __builtin_ctzll(who));
        if (__ballot(in && bin == lead) == who) {
            if (l == 0) atomicAdd(&hist[lead], (unsigned)__popcll(who));
        } else if (in) {
            atomicAdd(&hist[bin], 1u);
        }
    };
    // The part, from the top, in which the count reaches `left` (thread i has parts 2,047 - 2 i and the one below), its keys and
    // those of the parts above it.
    auto find_part = [&](unsigned left, unsigned& bin, unsigned& above, unsigned& inside) __attribute__((always_inline)) {
        __syncthreads();
        const unsigned h0 = hist[kEvBins - 1 - 2 * tid], h1 = hist[kEvBins - 2 - 2 * tid];
        unsigned upto = wave_scan(h0 + h1);
        if (l == 63) part[0][w] = upto;
        __syncthreads();
        hist[kEvBins - 1 - 2 * tid] = 0;  // for the next pass
        hist[kEvBins - 2 - 2 * tid] = 0;
#pragma unroll
        for (int i = 0; i < kEvWaves; ++i) upto += i < w ? part[0][i] : 0u;
        if (upto >= left && upto - h0 - h1 < left) {
            const bool upper = upto - h1 >= left;
            found[0] = (unsigned)(upper ? kEvBins - 1 - 2 * tid : kEvBins - 2 - 2 * tid);
            found[1] = upper ? upto - h0 - h1 : upto - h1;
            found[2] = upper ? h0 : h1;
        }
        __syncthreads();
        bin = found[0];
        above = found[1];
        inside = found[2];
    };
    hist[tid] = 0;
    hist[tid + kEvThreads] = 0;
    if (tid == 0) found[3] = 0;
    __syncthreads();

    // ---- narrow: `left` of the `inside` keys in [lo, hi] stay, and all above hi; `bits` of a number are not yet decided ----
    unsigned lo = 0, hi = 0xffffffffu, left = want, inside = (unsigned)nc;
    int bits = 32;
    unsigned zeros = 0;
    each([&](int, unsigned x) __attribute__((always_inline)) {
        zeros += x == kZero ? 1u : 0u;
        count_into(x >> 21, x != kZero && x != 0u);
    });
    zeros = wave_scan(zeros);
    if (l == 63 && zeros) atomicAdd(&hist[kZero >> 21], zeros);
    while (true) {
        const int shift = bits > 11 ? bits - 11 : 0;
        unsigned bin, above;
        find_part(left, bin, above, inside);
        left -= above;
        lo += bin << shift;
        hi = lo + ((1u << shift) - 1u);
        bits = shift;
        if (bits == 0 || inside == left || inside <= kEvList) break;
        const int next = bits > 11 ? bits - 11 : 0;
        each([&](int, unsigned x) __attribute__((always_inline)) { count_into((x - lo) >> next, x >= lo && x <= hi); });
    }
    // ---- how many keys of each wave's run lie above hi, how many in [lo, hi] (all of those or the first `left` stay) ----
    unsigned above = 0, in = 0;
    if (bits != 0 && inside != left) {  // (uniform) few keys: the rest of the bits as a list
        each([&](int, unsigned x) __attribute__((always_inline)) {
            above += x > hi ? 1u : 0u;
            if (x >= lo && x <= hi) {
                const unsigned at = atomicAdd(&found[3], 1u);
                list[at] = x;
                list_wave[at] = (unsigned char)w;
            }
        });
        const int mine = ((int)inside - tid + kEvThreads - 1) / kEvThreads;  // entries tid, tid + 1,024, ..
        while (bits > 0 && inside != left) {
            __syncthreads();
            const int shift = bits > 11 ? bits - 11 : 0;
            for (int i = 0; i < mine; ++i) {
                const unsigned x = list[tid + i * kEvThreads];
                if (x >= lo && x <= hi) atomicAdd(&hist[(x - lo) >> shift], 1u);
            }
            unsigned bin, over;
            find_part(left, bin, over, inside);
            left -= over;
            lo += bin << shift;
            hi = lo + ((1u << shift) - 1u);
            bits = shift;
        }
        above = wave_scan(above);
        if (l == 63) {
            part[0][w] = above;
            part[1][w] = 0;
        }
        __syncthreads();
        for (int i = 0; i < mine; ++i) {
            const unsigned x = list[tid + i * kEvThreads], v = list_wave[tid + i * kEvThreads];
            if (x > hi) atomicAdd(&part[0][v], 1u);
            if (x >= lo && x <= hi) atomicAdd(&part[1][v], 1u);
        }
    } else {
        each([&](int, unsigned x) __attribute__((always_inline)) {
            above += x > hi ? 1u : 0u;
            in += x >= lo ? 1u : 0u;
        });
        above = wave_scan(above);
        in = wave_scan(in);
        if (l == 63) {
            part[0][w] = above;
            part[1][w] = in - above;
        }
    }
    __syncthreads();
    unsigned in_before = 0, at = 0;  // of the waves before: keys in [lo, hi], kept keys
    for (int i = 0; i < w; ++i) {
        const unsigned take = min(part[1][i], left - min(left, in_before));
        in_before += part[1][i];
        at += part[0][i] + take;
    }
    auto rank = [](uint64_t mask) __attribute__((always_inline)) {  // lanes of the mask before this one
        return __builtin_amdgcn_mbcnt_hi((unsigned)(mask >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)mask, 0u));
    };
    each([&](int t, unsigned x) __attribute__((always_inline)) {
        uint64_t stays = __ballot(x > hi);
        const uint64_t ins = __ballot(x >= lo) & ~stays;
        if (ins != 0) {  // (the first `left` of the range, counted over the row)
            stays = __ballot(x > hi || (x >= lo && in_before + rank(ins) < left));
            in_before += __popcll(ins);
        }
        if (stays >> l & 1) kept[at + rank(stays)] = t + l;
        at += __popcll(stays);
    });
}

// Weights and rows of the kept keys; zeros behind their weights. A row is 65 units of 8 bytes: a workgroup copies kEvCopyRows rows of
// one (sequence, kv head), unit after unit over its lanes, all of a lane's loads before its stores.
constexpr int kEvCopyRows = 32;
constexpr int kEvUnits = 65;
constexpr int kEvLoads = (kEvCopyRows * kEvUnits + 255) / 256;

__global__ void __launch_bounds__(256) pd_evict_copy_kernel(const EvictParams a) {
    __shared__ int64_t from[kEvCopyRows], to[kEvCopyRows];
    const int g = blockIdx.y, b = blockIdx.z, j0 = blockIdx.x * kEvCopyRows, tid = threadIdx.x;
    const int n = max(0, min(min(a.seq_lens[b], a.max_keys), a.keep));
    float* wdst = a.new_weights + (int64_t)b * a.n_sb + (int64_t)g * a.n_sh;
    for (int64_t j = n + (int64_t)blockIdx.x * 256 + tid; j < a.new_keys; j += (int64_t)256 * gridDim.x) wdst[j] = 0.f;
    const int rows = min(kEvCopyRows, n - j0);
    if (rows <= 0) return;
    if (tid < rows) {
        const int j = j0 + tid, t = a.kept[((int64_t)b * a.Hkv + g) * a.keep + j];
        const int fb = t / a.block_size, tb = j / a.block_size;
        from[tid] = (int64_t)a.block_table[b * a.bt_stride + fb] * a.k_sb + (int64_t)(t - fb * a.block_size) * a.k_ss;
        to[tid] = (int64_t)a.new_table[b * a.nt_stride + tb] * a.k_sb + (int64_t)(j - tb * a.block_size) * a.k_ss;
        wdst[j] = a.weights[(int64_t)b * a.w_sb + (int64_t)g * a.w_sh + t];
    }
    __syncthreads();
    int8_t* base = a.kc + (int64_t)g * a.k_sh;
    uint64_t x[kEvLoads];
#pragma unroll
    for (int i = 0; i < kEvLoads; ++i) {
        const int u = min(tid + 256 * i, rows * kEvUnits - 1), r = u / kEvUnits;
        x[i] = *reinterpret_cast<const uint64_t*>(base + from[r] + 8 * (u - r * kEvUnits));
    }
#pragma unroll
    for (int i = 0; i < kEvLoads; ++i) {
        const int u = tid + 256 * i, r = u / kEvUnits;
        if (u < rows * kEvUnits) *reinterpret_cast<uint64_t*>(base + to[r] + 8 * (u - r * kEvUnits)) = x[i];
    }
}

// ---------------------------------------------------------------------------------------
// host side

hipError_t launch_evict(const EvictParams& p, int num_seqs, hipStream_t stream) {
    // registers for the longest row that the table and the weights can hold: sequences of up to 6,000 keys, both launches, 19.0 us with 8
    // a lane, 20.6 with 24, 24.8 with 64; one of 61,440 keys 37.3 with 64 and 45.7 read again in every pass
    const dim3 rows(p.Hkv, num_seqs), block(kEvThreads);
    if (p.max_keys <= 8 * kEvThreads)
        hipLaunchKernelGGL((pd_evict_select_kernel<8, true>), rows, block, 0, stream, p);
    else if (p.max_keys <= 24 * kEvThreads)
        hipLaunchKernelGGL((pd_evict_select_kernel<24, true>), rows, block, 0, stream, p);
    else if (p.max_keys <= 64 * kEvThreads)
        hipLaunchKernelGGL((pd_evict_select_kernel<64, true>), rows, block, 0, stream, p);
    else
        hipLaunchKernelGGL((pd_evict_select_kernel<32, false>), rows, block, 0, stream, p);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    const dim3 grid((p.keep + kEvCopyRows - 1) / kEvCopyRows, p.Hkv, num_seqs);
    hipLaunchKernelGGL(pd_evict_copy_kernel, grid, dim3(256), 0, stream, p);
    return hipGetLastError();
}

}  // namespace pd
