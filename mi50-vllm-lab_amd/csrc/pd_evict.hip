// Eviction from the cache by running attention weights: per (sequence, kv head) the last `recent` keys and the
// keep - recent others with the largest weights stay (equal weights: the lowest key first; NaN counts as the largest), in the
// order of their positions. pd_evict_select_kernel finds them and writes their numbers and weights; pd_evict_copy_kernel
// copies their 520-byte rows into the blocks of another table, so blocks that several sequences share stay as they are
// and no row is read after it was written over.
//
// The select is one workgroup per (sequence, kv head). A weight's bits become an unsigned number of the same order; the
// range [lo, hi] that holds the smallest weight to keep is narrowed from [min, max] by histograms of 2,048 equal parts
// (each pass divides it by 2,048: three at the most, and the parts follow the data, so few lanes meet in one counter), until
// the part is one value or is kept whole. Then each wave counts its own run of keys, the counts are summed over the
// waves, and each wave writes its kept keys in order: their places are known without a barrier.
#include "pd_tile.hpp"
#include "pth_dec.h"

namespace pd {

constexpr int kEvWaves = 16;
constexpr int kEvThreads = 64 * kEvWaves;
constexpr int kEvBins = 2048;

// Order of the weights as unsigned numbers: -0 as 0, NaN above all.
__device__ __forceinline__ unsigned weight_order(float x) {
    if (x != x) return 0xffffffffu;
    const unsigned u = __builtin_bit_cast(unsigned, x + 0.f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__global__ void __launch_bounds__(kEvThreads) pd_evict_select_kernel(const EvictParams a) {
    __shared__ unsigned hist[kEvBins];
    __shared__ unsigned part[2][kEvWaves];
    __shared__ unsigned found[2];
    const int g = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, l = tid & 63;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = max(0, min(a.seq_lens[b], a.max_keys)), keep = a.keep;
    const float* wsrc = a.weights + (int64_t)b * a.w_sb + (int64_t)g * a.w_sh;
    float* wdst = a.new_weights + (int64_t)b * a.n_sb + (int64_t)g * a.n_sh;
    int* kept = a.kept + ((int64_t)b * a.Hkv + g) * keep;
    if (g == 0 && tid == 0) a.new_lens[b] = min(n, keep);
    for (int j = min(n, keep) + tid; j < a.new_keys; j += kEvThreads) wdst[j] = 0.f;
    if (n <= keep) {  // everything stays
        for (int j = tid; j < keep; j += kEvThreads) {
            kept[j] = j < n ? j : -1;
            if (j < n) wdst[j] = wsrc[j];
        }
        return;
    }
    const int recent = min(a.recent, keep), nc = n - recent;  // candidates [0, nc)
    const unsigned want = (unsigned)(keep - recent);           // of which so many stay
    for (int j = tid; j < recent; j += kEvThreads) {
        kept[want + j] = nc + j;
        wdst[want + j] = wsrc[nc + j];
    }
    if (want == 0) return;

    // ---- [lo, hi]: smallest and largest candidate ----
    unsigned lo = 0xffffffffu, hi = 0;
    for (int t = tid; t < nc; t += kEvThreads) {
        const unsigned u = weight_order(wsrc[t]);
        lo = min(lo, u);
        hi = max(hi, u);
    }
    lo = ~wave_umax(~lo);
    hi = wave_umax(hi);
    if (l == 0) {
        part[0][w] = lo;
        part[1][w] = hi;
    }
    __syncthreads();
    for (int i = 0; i < kEvWaves; ++i) {
        lo = min(lo, part[0][i]);
        hi = max(hi, part[1][i]);
    }
    // ---- narrow: `left` of the keys in [lo, hi] stay, and all above hi ----
    unsigned left = want;
    while (hi > lo) {
        const int bits = 32 - __builtin_clz(hi - lo);  // of the distance
        const int shift = bits > 11 ? bits - 11 : 0;
        for (int i = tid; i < kEvBins; i += kEvThreads) hist[i] = 0;
        __syncthreads();
        for (int t = tid; t < nc; t += kEvThreads) {
            const unsigned u = weight_order(wsrc[t]);
            if (u >= lo && u <= hi) atomicAdd(&hist[(u - lo) >> shift], 1u);
        }
        __syncthreads();
        if (w == 0) {  // the part, from the top, in which the count reaches `left`: 32 parts per lane
            unsigned mine = 0;
            for (int i = 0; i < 32; ++i) mine += hist[kEvBins - 1 - (32 * l + i)];
            const unsigned upto = wave_scan(mine);
            if (upto >= left && upto - mine < left) {
                unsigned above = upto - mine;
                int i = 0;
                while (above + hist[kEvBins - 1 - (32 * l + i)] < left) above += hist[kEvBins - 1 - (32 * l + i++)];
                found[0] = (unsigned)(kEvBins - 1 - (32 * l + i));
                found[1] = above;
            }
        }
        __syncthreads();
        const unsigned bin = found[0], inside = hist[bin];
        left -= found[1];
        lo += bin << shift;
        if (((hi - lo) >> shift) != 0) hi = lo + ((1u << shift) - 1u);
        if (inside == left) break;  // the whole part stays
        __syncthreads();             // hist and found are written again
    }

    // ---- each wave's run of keys: how many lie above hi, how many in [lo, hi] ----
    const int per = ((nc + kEvWaves - 1) / kEvWaves + 63) / 64 * 64;
    const int t0 = min(nc, w * per), t1 = min(nc, t0 + per);
    unsigned above = 0, in = 0;
    for (int t = t0; t < t1; t += 64) {
        const bool live = t + l < t1;
        const unsigned u = live ? weight_order(wsrc[t + l]) : 0;
        above += __popcll(__ballot(live && u > hi));
        in += __popcll(__ballot(live && u >= lo && u <= hi));
    }
    __syncthreads();
    if (l == 0) {
        part[0][w] = above;
        part[1][w] = in;
    }
    __syncthreads();
    unsigned in_before = 0, at = 0;  // of the waves before: keys in [lo, hi], kept keys
    for (int i = 0; i < w; ++i) {
        const unsigned take = min(part[1][i], left - min(left, in_before));
        in_before += part[1][i];
        at += part[0][i] + take;
    }
    const uint64_t below = ((uint64_t)1 << l) - 1;
    for (int t = t0; t < t1; t += 64) {
        const bool live = t + l < t1;
        const float x = live ? wsrc[t + l] : 0.f;
        const unsigned u = live ? weight_order(x) : 0;
        const bool inside = live && u >= lo && u <= hi;
        const uint64_t ins = __ballot(inside);
        const bool stay = (live && u > hi) || (inside && in_before + __popcll(ins & below) < left);
        const uint64_t stays = __ballot(stay);
        if (stay) {
            const unsigned j = at + __popcll(stays & below);
            kept[j] = t + l;
            wdst[j] = x;
        }
        in_before += __popcll(ins);
        at += __popcll(stays);
    }
}

// Rows of the cache, 65 units of 8 bytes each: a workgroup copies kEvCopyRows rows of one (sequence, kv head), unit after
// unit over its lanes.
constexpr int kEvCopyRows = 64;
constexpr int kEvUnits = 65;

__global__ void __launch_bounds__(256) pd_evict_copy_kernel(const EvictParams a) {
    __shared__ int64_t from[kEvCopyRows], to[kEvCopyRows];
    const int g = blockIdx.y, b = blockIdx.z, j0 = blockIdx.x * kEvCopyRows, tid = threadIdx.x;
    const int n = max(0, min(min(a.seq_lens[b], a.max_keys), a.keep)), rows = min(kEvCopyRows, n - j0);
    if (rows <= 0) return;
    if (tid < rows) {
        const int j = j0 + tid, t = a.kept[((int64_t)b * a.Hkv + g) * a.keep + j];
        const int fb = t / a.block_size, tb = j / a.block_size;
        from[tid] = (int64_t)a.block_table[b * a.bt_stride + fb] * a.k_sb + (int64_t)(t - fb * a.block_size) * a.k_ss;
        to[tid] = (int64_t)a.new_table[b * a.nt_stride + tb] * a.k_sb + (int64_t)(j - tb * a.block_size) * a.k_ss;
    }
    __syncthreads();
    int8_t* base = a.kc + (int64_t)g * a.k_sh;
    for (int u = tid; u < rows * kEvUnits; u += 256) {
        const int r = u / kEvUnits, c = 8 * (u - r * kEvUnits);
        *reinterpret_cast<uint64_t*>(base + to[r] + c) = *reinterpret_cast<const uint64_t*>(base + from[r] + c);
    }
}

// ---------------------------------------------------------------------------------------
// host side

hipError_t launch_evict(const EvictParams& p, int num_seqs, hipStream_t stream) {
    hipLaunchKernelGGL(pd_evict_select_kernel, dim3(p.Hkv, num_seqs), dim3(kEvThreads), 0, stream, p);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    const dim3 grid((p.keep + kEvCopyRows - 1) / kEvCopyRows, p.Hkv, num_seqs);
    hipLaunchKernelGGL(pd_evict_copy_kernel, grid, dim3(256), 0, stream, p);
    return hipGetLastError();
}

}  // namespace pd
