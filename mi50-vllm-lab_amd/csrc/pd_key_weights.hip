// Running attention weights of the cached keys: for a decode step's query rows and the logarithms of their softmax
// sums (the decode operators' lse), weights[b, g, t] += sum over the rows r of kv head g that see key t of
// e^(scale ksc_t (q_r . k_t) - lse_r), the weight that the step gave key t. Summed over steps it says which keys a sequence
// attends to; evict keeps those.
//
// A wave takes blocks of 16 keys: S = K Q^T on v_mfma_f32_16x16x32_f16 with A = 16 keys x 32 dims of K (int8 widened to fp16
// exactly, straight from global memory: a lane's operand is 16 consecutive bytes of one row) and B = Q^T
// in registers, the accumulators giving each lane 4 keys of one query row. The exponentials are summed over the row
// blocks in the lane and over the 16 rows of a block by DPP rotations, so every weight is formed by one lane in a fixed
// order: no atomics, the same result every time. Scores, exponentials and sums are fp32.
//
// What bounds it: memory. A row's 260 bytes of K and scale touch three 128-byte lines, 388 bytes: 61,440 keys of 4 heads 21.6 us for 95 MB of
// lines, 4.4 TB/s; 16 sequences of 500 to 8,192 keys 19.0.
#include "pd_tile.hpp"
#include "pth_dec.h"

namespace pd {

constexpr int kKwKeys = 16;   // keys of a block
constexpr int kKwWaves = 4;

// Sum over the 16 lanes of a DPP row, in every lane (rotations by 8, 4, 2, 1).
__device__ __forceinline__ float row16_sum(float v) {
    auto ror = [](float x, auto ctrl) {
        return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), decltype(ctrl)::value, 0xf, 0xf, false));
    };
    v += ror(v, std::integral_constant<int, 0x128>{});
    v += ror(v, std::integral_constant<int, 0x124>{});
    v += ror(v, std::integral_constant<int, 0x122>{});
    return v + ror(v, std::integral_constant<int, 0x121>{});
}

template <int NRB>
__global__ void __launch_bounds__(64 * kKwWaves) pd_key_weights_kernel(const KeyWeightsParams a) {
    const int g = blockIdx.y, b = blockIdx.z;
    const int l = threadIdx.x & 63, lg = l >> 4, li = l & 15;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int q0 = a.qsl[b], q_len = a.qsl[b + 1] - q0;
    const int seq_len = a.seq_lens[b];
    if (q_len <= 0 || seq_len <= 0) return;
    const int G = a.G, R = min(16 * NRB, min(q_len, a.qmax) * G), ctx0 = seq_len - q_len;
    const int nblk = (min(seq_len, a.max_keys) + kKwKeys - 1) / kKwKeys, stride = gridDim.x * kKwWaves;
    const int first = blockIdx.x * kKwWaves + w;
    if (first >= nblk) return;

    const int8_t* gbase = a.kc + (int64_t)g * a.k_sh;
    const int* bt = a.block_table + (int64_t)b * a.bt_stride;
    float* wrow = a.weights + (int64_t)b * a.w_sb + (int64_t)g * a.w_sh;
    // Three stages of a block, each a memory round trip, run one behind the other: the page of this lane's key, the operand
    // bytes of its row (keys past the last are the last), the products.
    auto key_of = [&](int n) __attribute__((always_inline)) { return min(n * kKwKeys + li, seq_len - 1); };
    auto slot_of = [&](int key) __attribute__((always_inline)) { return a.bs_shift >= 0 ? key >> a.bs_shift : key / a.block_size; };
    auto page_of = [&](int n) __attribute__((always_inline)) { return n < nblk ? bt[slot_of(key_of(n))] : 0; };
    struct Block {
        uint4_t k[4];
        float ks;
    };
    auto fetch = [&](int n, int page) __attribute__((always_inline)) {
        const int key = key_of(n);
        const int8_t* row = gbase + (int64_t)page * a.k_sb + (int64_t)(key - slot_of(key) * a.block_size) * a.k_ss;
        Block x;
#pragma unroll
        for (int c = 0; c < 4; ++c) __builtin_memcpy(&x.k[c], __builtin_assume_aligned(row + 64 * c + 16 * lg, 8), 16);
        x.ks = *reinterpret_cast<const float*>(row + kDim);
        return x;
    };
    const int page0 = page_of(first), page1 = page_of(first + stride);
    int page2 = page_of(first + 2 * stride);

    // ---- Q^T: lane (lg, li) holds row 16 rb + li, dims 64 (st / 2) + 16 lg + 8 (st % 2) + [0, 8) ----
    half8_t qop[NRB][8];
    float nlse[NRB];  // -lse in log2 units
    int rpos[NRB];    // the last key that counts for the row: none where its sum was 0 or it is past the last row
    bool valid[NRB];
#pragma unroll
    for (int rb = 0; rb < NRB; ++rb) {
        const int r = 16 * rb + li;
        valid[rb] = r < R;
        const int qi = valid[rb] ? r / G : 0, qh = valid[rb] ? r - qi * G : 0;
        const _Float16* qrow = a.q + (int64_t)(q0 + qi) * a.q_st + (int64_t)(g * G + qh) * kDim;
#pragma unroll
        for (int st = 0; st < 8; ++st)
            __builtin_memcpy(&qop[rb][st], __builtin_assume_aligned(qrow + 64 * (st >> 1) + 16 * lg + 8 * (st & 1), 4), 16);
        nlse[rb] = a.lse[(int64_t)(q0 + qi) * a.Hq + g * G + qh];
        rpos[rb] = ctx0 + qi;
    }
    Block cur = fetch(first, page0), next = cur;
    if (first + stride < nblk) next = fetch(first + stride, page1);
#pragma unroll
    for (int rb = 0; rb < NRB; ++rb) {
#pragma unroll
        for (int st = 0; st < 8; ++st) qop[rb][st] = valid[rb] ? qop[rb][st] : (half8_t)(_Float16)0.0f;
        rpos[rb] = valid[rb] && nlse[rb] != kNegInf ? rpos[rb] : -1;
        nlse[rb] *= -1.4426950408889634f;
    }
    for (int n = first; n < nblk; n += stride) {
        Block later = next;
        if (n + 2 * stride < nblk) later = fetch(n + 2 * stride, page2);
        page2 = page_of(n + 3 * stride);
        float4_t s[NRB];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
#pragma unroll
            for (int hh = 0; hh < 2; ++hh) {
                const half8_t kf = hh == 0 ? widen_i8x8_exact(cur.k[c].x, cur.k[c].y) : widen_i8x8_exact(cur.k[c].z, cur.k[c].w);
#pragma unroll
                for (int rb = 0; rb < NRB; ++rb)
                    s[rb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qop[rb][2 * c + hh], (c | hh) ? s[rb] : (float4_t)0.f, 0, 0, 0);
            }
        }
        const int key0 = n * kKwKeys + 4 * lg;
        float sum[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float ks = __shfl(cur.ks, 4 * lg + j, 64) * a.scale_log2;  // (lane 4 lg + j of the first row holds key 4 lg + j)
            float acc = 0.f;
#pragma unroll
            for (int rb = 0; rb < NRB; ++rb) {
                const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[rb][j], ks, nlse[rb]));
                acc += key0 + j <= rpos[rb] ? p : 0.f;
            }
            sum[j] = row16_sum(acc);
        }
        const float mine = li == 0 ? sum[0] : li == 1 ? sum[1] : li == 2 ? sum[2] : sum[3];
        if (li < 4 && key0 + li < min(seq_len, a.max_keys)) wrow[key0 + li] += mine;
        cur = next;
        next = later;
    }
}

// ---------------------------------------------------------------------------------------
// host side

hipError_t launch_key_weights(const KeyWeightsParams& p, int num_seqs, int heads_kv, hipStream_t stream) {
    const int rows = p.qmax * p.G, nrb = (rows + 15) / 16;
    const int known = compute_units(stream);
    const int64_t cus = known > 0 ? known : 256;
    // as many workgroups as run at once: 4, 3 or 2 per CU by the registers of 1 to 3 row blocks. us with 2, 3, 4 and 6 per CU: 16 sequences
    // of 500 to 8,192 keys (one block) 22.7, 18.9, 18.6, 17.8; 4 tokens over 61,440 (two) 21.3, 20.9, 23.3, 22.8
    int64_t splits = (5 - nrb) * cus / ((int64_t)num_seqs * heads_kv);
    const int64_t most = (p.table_keys + kKwKeys * kKwWaves - 1) / (kKwKeys * kKwWaves);
    splits = splits < 1 ? 1 : splits;
    if (most >= 1 && splits > most) splits = most;
    const dim3 grid((unsigned)splits, heads_kv, num_seqs), block(64 * kKwWaves);
    if (nrb == 1)
        hipLaunchKernelGGL((pd_key_weights_kernel<1>), grid, block, 0, stream, p);
    else if (nrb == 2)
        hipLaunchKernelGGL((pd_key_weights_kernel<2>), grid, block, 0, stream, p);
    else
        hipLaunchKernelGGL((pd_key_weights_kernel<3>), grid, block, 0, stream, p);
    return hipGetLastError();
}

}  // namespace pd
