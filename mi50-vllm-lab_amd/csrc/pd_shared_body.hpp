// The workgroup of the shared-prefix decode (pd_shared.hip): a run of key tiles against rows of one kv head. Eight waves, two
// per SIMD, in KW key groups of RW row groups: wave (k, r) takes every KW-th tile of the run for RB blocks of 16 rows, and the
// key groups' states are merged through LDS at the end. A wave holds Q and O of its rows in registers; S^T = K Q^T leaves a lane
// the weights that it needs as an operand of O^T += V^T P^T, so nothing is exchanged between waves in a tile and a row's
// running max belongs to one wave. Per tile a wave has 16 RB MFMAs for the scores, as many for each term of P', a softmax
// of 8 RB scores per lane, and the widening of int8 to fp16 operands (256 conversions for all of a tile), which is what the three forms
// treat differently:
//   RW = 8  (the prefix) each wave widens an eighth of the tile into operands in LDS, a tile ahead, and all read them: 32 conversions
//           and 32 reads of 1 KiB. The two waves of a SIMD do so before and behind their products, so that one converts while
//           the other multiplies. A tile of 256 rows takes 2.4 us (2.0 with one term of P'; then 2.9 with every wave widening all
//           of it for itself, VALU busy 61 % and MFMA 31 % of the time, nothing of it at once, and 2.9, two tiles of 128, with the
//           scores' keys and the values' dims split over the waves and P' exchanged through LDS).
//   RW = 1  (own keys, <= 16 rows) a wave's tiles are its own: no barrier, every byte is widened once, K goes straight to
//           registers, as its operands lie as the rows do.
//   RW = 4  (own keys, up to 48 rows) as RW = 1 on tiles in LDS that four waves share; 7 sequences of 3 x 6 rows 20.0 us, with two row
//           blocks per wave and four key groups 21.9.
// Tiles come by DMA into rings of kRing slots per key group, copied by the group's own waves; RW > 1: one barrier per tile.
// P' = p v_scale enters P.V as fp16 hi + lo (see pd_shared.hip).
#pragma once

#include "pd_tile.hpp"

namespace pd {

constexpr int kSwWaves = 8;
constexpr int kSwThreads = 64 * kSwWaves;
// A slot: the K and V images of pd_tile.hpp (V from byte 260 of the row, so its 16 blocks hold whole dim blocks), then
// the tile's scales: k_scale [32], v_scale [32].
constexpr int kSwImgS = 16 * kBlk;
constexpr int kSwSlot = kSwImgS + 256;
constexpr int kSwSlots = 8;        // of the key groups' rings
constexpr int kSwOwn = 8 * kBlk + 256;  // a V image and scales
constexpr int kSwWide = 5;         // of the ring beside the fragments
constexpr int kSwFrag = 32 * 1024; // a tile's K and V as MFMA operands: [key block][step] and [dim block], a lane's 16 bytes each
constexpr int kSwTable = 1024;     // 16-key blocks (or pages) of the LDS block table
constexpr int kSwBt = kSwWide * kSwSlot + 2 * kSwFrag;
constexpr int kSwLds = kSwBt + kSwTable * 4;
static_assert(kSwSlots * kSwSlot <= kSwBt && 2 * kSwWaves * kSwOwn <= kSwBt, "");
static_assert(kSwLds <= 160 * 1024, "gfx950 has 160 KiB of LDS per CU");

// What a workgroup computes: rows [row0, row0 + nrow) of kv head g, row r: token q0 + r / G at position pos0 + r / G, head r % G of g;
// keys [lo, hi) of the table of sequence b up to the row's position, of tiles [t0, t1); into segment `seg`.
struct SharedWork {
    int g, b, q0, row0, nrow, pos0, lo, hi, t0, t1, seg;
};

template <int RB, int RW, bool kFast>
__device__ __forceinline__ void shared_body(const SharedParams& sp, const SharedWork& wk, unsigned char* lds) {
    constexpr int KW = kSwWaves / RW, kRing = RW == 8 ? kSwWide : kSwSlots / KW;
    static_assert(KW == 1 || 64 * RB * (KW / 2) * RW * 264 <= kSwBt, "half of the key groups' O fits the slots");
    const PartialParams& a = sp.p;
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));  // (keeps the compiler from holding this function's addresses in registers around its caller's loop)
    const int l = tid & 63, lg = l >> 4, li = l & 15;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = w % RW, k = w / RW;
    const int G = a.G, g = wk.g, t0 = wk.t0, cnt = wk.t1 - wk.t0, hi = wk.hi;
    const int mine = (cnt - k + KW - 1) / KW;                 // tiles of this key group
    const bool rows = 16 * RB * r < wk.nrow;                  // this wave has rows
    lds_u8* L = (lds_u8*)lds;
    const int8_t* gbase = a.kc + (int64_t)g * a.k_sh;

    // ---- block table of the workgroup's keys into LDS: for bs % 16 == 0 the byte offset / 8 of every 16-key block's first
    //      row, else the page numbers ----
    PageTable pt;
    pt.glob = (const_int_ptr)(uintptr_t)(a.block_table + (int64_t)wk.b * a.bt_stride);
    pt.lds = (const lds_int*)(L + kSwBt);
    pt.rows16 = nullptr;
    pt.pfirst = 0;
    {
        const int* bt_glob = a.block_table + (int64_t)wk.b * a.bt_stride;
        lds_int* dst = (lds_int*)(L + kSwBt);
        if constexpr (kFast) {
            const int nblk = 2 * cnt;
            pt.in_lds = sp.bt32 && nblk <= kSwTable;
            if (pt.in_lds) {
                for (int i = tid; i < nblk; i += kSwThreads) {
                    const int kb = (t0 + (i >> 1)) * kTile, klast = min(kb + kTile - 1, hi - 1);
                    const int key0 = min(kb + 16 * (i & 1), klast) & ~15;
                    const int lb = a.bs_shift >= 0 ? key0 >> a.bs_shift : key0 / a.block_size;
                    const int64_t off = (int64_t)bt_glob[lb] * a.k_sb + (int64_t)(key0 - lb * a.block_size) * a.k_ss;
                    dst[i] = (int)(unsigned)((uint64_t)off >> 3);
                }
            }
        } else {
            pt.pfirst = t0 * kTile / a.block_size;
            const int npages = (min(wk.t1 * kTile, hi) - 1) / a.block_size + 1 - pt.pfirst;
            pt.in_lds = npages <= kSwTable;
            if (pt.in_lds)
                for (int i = tid; i < npages; i += kSwThreads) dst[i] = bt_glob[pt.pfirst + i];
        }
    }

    // ---- Q^T of this wave's row blocks: lane (lg, li) holds row 16 (RB r + j) + li, dims 64 (st / 2) + 16 lg + 8 (st % 2) + [0, 8)
    //      in qop[st][j] ----
    half8_t qop[8][RB];
    auto row_at = [&](int x, int& tok, int& hd) __attribute__((always_inline)) {  // row x of the tile (the first if there is none)
        const int at = wk.row0 + (x < wk.nrow ? x : 0);
        tok = at / G;
        hd = at - tok * G;
    };
#pragma unroll
    for (int j = 0; j < RB; ++j) {
        int tok, hd;
        row_at(16 * (RB * r + j) + li, tok, hd);
        const _Float16* qrow = a.q + (int64_t)(wk.q0 + tok) * a.q_st + (int64_t)(g * G + hd) * kDim;
#pragma unroll
        for (int st = 0; st < 8; ++st)
            __builtin_memcpy(&qop[st][j], __builtin_assume_aligned(qrow + 64 * (st >> 1) + 16 * lg + 8 * (st & 1), 4), 16);
    }
#pragma unroll
    for (int j = 0; j < RB; ++j)
#pragma unroll
        for (int st = 0; st < 8; ++st)
            if (16 * (RB * r + j) + li >= wk.nrow) qop[st][j] = (half8_t)(_Float16)0.0f;
    __syncthreads();  // the LDS block table is complete

    // Relative scores carry +kPLog2: p' = 2^(s - m + kPLog2) = 16 p, so P' = p' * v_scale spans the same fp16 range as in
    // the decode kernel; l accumulates p'.
    constexpr float kPLog2 = 4.0f;
    // per row: this lane's sum over its keys, the score offset -m + kPLog2 (kPLog2 while the row has seen no key) and the
    // relative score above which the running max m must be raised (any finite score while fresh)
    float l_run[RB], nm_run[RB], thr_run[RB];
    float4_t oacc[16][RB];  // dims 16 m + 4 lg .. of row li of each block
#pragma unroll
    for (int j = 0; j < RB; ++j) {
        l_run[j] = 0.f;
        nm_run[j] = kPLog2;
        thr_run[j] = kNegInf;
#pragma unroll
        for (int m = 0; m < 16; ++m) oacc[m][j] = (float4_t)0.f;
    }

    // ---- this lane's positions in a slot ----
    int kro[4];  // K operand of 32-dim step pair c: 16 source bytes of key row li of key block 0
#pragma unroll
    for (int c = 0; c < 4; ++c) kro[c] = kImgK + (li >> 2) * kBlk + 256 * (l & 3) + 64 * (c ^ (l & 3)) + 16 * lg;
    // transposed V reads: 8 keys of one dim (lanes 2 i, 2 i + 1 of a 16-lane group name tile row tkey); odd row groups hold
    // dim blocks 0..7 in their second half
    int vro[2];
    {
        const int i = li >> 1;
        const int tkey = i < 4 ? 4 * lg + i : 12 + 4 * lg + i;
        const int at = kImgV + ((tkey & 3) + 4 * (tkey >> 4)) * kBlk + 256 * lg + 8 * (l & 1);
        vro[0] = at + (lg & 1 ? 128 : 0);
        vro[1] = at - (lg & 1 ? 128 : 0);
    }
    const int sro = kSwImgS + 16 * lg;  // k_scale of keys 4 lg + j of key block 0; block 1 64, v_scale 128 bytes on

    float4_t s[2][RB];
    auto max8 = [&](int j) __attribute__((always_inline)) {
        return fmaxf(fmaxf(fmaxf(s[0][j][0], s[0][j][1]), fmaxf(s[0][j][2], s[0][j][3])),
                     fmaxf(fmaxf(s[1][j][0], s[1][j][1]), fmaxf(s[1][j][2], s[1][j][3])));
    };
    // S: the tile's slot; F (RW = 8): this lane's place in its fragments
    auto scores = [&](int kb, const lds_u8* S, const lds_u8* F, const uint4_t* kc) __attribute__((always_inline)) {
        if constexpr (RW == 8) {
            half8_t kf[4];  // three reads ahead
#pragma unroll
            for (int i = 0; i < 3; ++i) kf[i] = *(const lds_half8*)(F + i * 1024);
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                if (i < 13) kf[(i + 3) & 3] = *(const lds_half8*)(F + (i + 3) * 1024);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int j = 0; j < RB; ++j)
                    s[i >> 3][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[i & 3], qop[i & 7][j], i & 7 ? s[i >> 3][j] : (float4_t)0.f, 0, 0, 0);
            }
        } else
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            uint4_t kr[2];
            if constexpr (RW > 1) kr[0] = *(const lds_uint4*)(S + kro[0] + u * 4 * kBlk);
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                if constexpr (RW > 1) {
                    if (c < 3) kr[(c + 1) & 1] = *(const lds_uint4*)(S + kro[c + 1] + u * 4 * kBlk);
                    __builtin_amdgcn_sched_barrier(0);
                } else {
                    kr[c & 1] = kc[4 * u + c];
                }
#pragma unroll
                for (int hh = 0; hh < 2; ++hh) {
                    const half8_t kf = hh == 0 ? widen_i8x8_exact(kr[c & 1].x, kr[c & 1].y) : widen_i8x8_exact(kr[c & 1].z, kr[c & 1].w);
#pragma unroll
                    for (int j = 0; j < RB; ++j)
                        s[u][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qop[2 * c + hh][j], (c | hh) ? s[u][j] : (float4_t)0.f, 0, 0, 0);
                }
            }
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const float4_t ksc = *(const lds_float4*)(S + sro + 64 * u);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float ks = ksc[i] * a.scale_log2;
#pragma unroll
                for (int j = 0; j < RB; ++j) s[u][j][i] = __builtin_fmaf(s[u][j][i], ks, nm_run[j]);
            }
        }
        if (kb < wk.lo || kb + kTile > min(hi, wk.pos0 + 1)) {  // some row does not see all of the tile
            int lim[RB], lr = threadIdx.x;  // last key that the row sees
            asm volatile("" : "+v"(lr));
            const int lg = lr >> 4 & 3;
#pragma unroll
            for (int j = 0; j < RB; ++j) {
                int tok, hd;
                row_at(16 * (RB * r + j) + (lr & 15), tok, hd);
                lim[j] = min(hi - 1, wk.pos0 + tok);
            }
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int t = kb + 16 * u + 4 * lg + i;
#pragma unroll
                    for (int j = 0; j < RB; ++j) s[u][j][i] = t >= wk.lo && t <= lim[j] ? s[u][j][i] : kNegInf;
                }
        }
        float mloc[RB];
        bool need = false;
#pragma unroll
        for (int j = 0; j < RB; ++j) {
            mloc[j] = max8(j);
            need |= mloc[j] > thr_run[j];
        }
        if (__builtin_amdgcn_ballot_w64(need) != 0) {  // rare: raise the running max of the rows that need it
#pragma unroll
            for (int j = 0; j < RB; ++j) {
                const float mrow = xor_max(xor_max(mloc[j], 16), 32) - kPLog2;  // tile max relative to m
                const bool fresh = thr_run[j] == kNegInf;
                const bool up = fresh ? mrow > kNegInf : mrow > kLazy;
                const float shift = up ? mrow : 0.f;
                const float alpha = fresh ? 0.f : __builtin_amdgcn_exp2f(-shift);
                nm_run[j] -= shift;
                if (up) thr_run[j] = kLazy + kPLog2;
                l_run[j] *= alpha;
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int i = 0; i < 4; ++i) s[u][j][i] -= shift;
#pragma unroll
                for (int m = 0; m < 16; ++m) oacc[m][j] *= alpha;
            }
        }
    };
    auto value_scales = [&](int kb, const lds_u8* S, float4_t (&vs)[2]) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < 2; ++u) vs[u] = *(const lds_float4*)(S + sro + 64 * u + 128);
        if (kb < wk.lo || kb + kTile > hi) {  // a scale outside may be garbage, even NaN
            int lr = threadIdx.x;
            asm volatile("" : "+v"(lr));
            const int lg = lr >> 4 & 3;
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int t = kb + 16 * u + 4 * lg + i;
                    vs[u][i] = t >= wk.lo && t < hi ? vs[u][i] : 0.f;
                }
        }
    };
    // ---- p' = 2^s, P' = p' * v_scale in fp16, hi and what hi leaves in lo; O += V^T P'^T ----
    auto weights = [&](int j, float (&p)[8]) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < 8; ++i) p[i] = __builtin_amdgcn_exp2f(s[i >> 2][j][i & 3]);
    };
    auto split = [&](const float (&p)[8], const float4_t (&vs)[2], half8_t& hi8, half8_t& lo8) __attribute__((always_inline)) {
        half2_t x[4], y[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float a0 = p[2 * i] * vs[i >> 1][2 * (i & 1)], a1 = p[2 * i + 1] * vs[i >> 1][2 * (i & 1) + 1];
            x[i] = __builtin_convertvector((float2_t){a0, a1}, half2_t);
            y[i] = __builtin_convertvector((float2_t){a0 - (float)x[i].x, a1 - (float)x[i].y}, half2_t);
        }
        __builtin_memcpy(&hi8, x, 16);
        __builtin_memcpy(&lo8, y, 16);
    };
    auto sum8 = [](const float (&p)[8]) __attribute__((always_inline)) { return ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7])); };
    auto values = [&](int kb, const lds_u8* S, const lds_u8* F) __attribute__((always_inline)) {
        half8_t pf[RB], pl[RB];
        float4_t vs[2];
        value_scales(kb, S, vs);
#pragma unroll
        for (int j = 0; j < RB; ++j) {
            float p[8];
            weights(j, p);
            l_run[j] += sum8(p);
            split(p, vs, pf[j], pl[j]);
        }
        constexpr int kAhead = 3;
        half8_t vb[kAhead + 1];
        if constexpr (RW == 8) {
#pragma unroll
            for (int m = 0; m < kAhead; ++m) vb[m] = *(const lds_half8*)(F + (16 + m) * 1024);
        }
#pragma unroll
        for (int m = 0; m < 16; ++m) {
            half8_t vf;
            if constexpr (RW == 8) {
                if (m + kAhead < 16) vb[(m + kAhead) % (kAhead + 1)] = *(const lds_half8*)(F + (16 + m + kAhead) * 1024);
                __builtin_amdgcn_sched_barrier(0);
                vf = vb[m % (kAhead + 1)];
            } else {
                const int2_t vr = __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_int2*)(S + vro[m >> 3] + 16 * m));
                vf = widen_i8x8_exact((unsigned)vr.x, (unsigned)vr.y);
            }
#pragma unroll
            for (int j = 0; j < RB; ++j) oacc[m][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pf[j], oacc[m][j], 0, 0, 0);
#pragma unroll
            for (int j = 0; j < RB; ++j) oacc[m][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pl[j], oacc[m][j], 0, 0, 0);
        }
    };

    auto tile_loop = [&](auto lds_flag) __attribute__((always_inline)) {
        constexpr bool kLds = decltype(lds_flag)::value;
        // This wave copies blocks r, r + RW, .. of the 8 K and 8 V blocks of its group's tiles and 64 / RW of the 64 scales.
        constexpr int kPer = 8 / RW, kCopies = 2 * kPer + 1;
        const unsigned group = (unsigned)(uintptr_t)L + k * kRing * kSwSlot;
        auto tile_of = [&](int n) __attribute__((always_inline)) { return KW * min(n, mine - 1) + k; };
        auto block_base = [&](int entry, int tile, int ub) __attribute__((always_inline)) -> const int8_t* {
            if constexpr (kLds) {
                return gbase + ((int64_t)(unsigned)__builtin_amdgcn_readfirstlane(entry) << 3);
            } else {
                const int kb = (t0 + tile) * kTile, klast = min(kb + kTile - 1, hi - 1);
                const int key0 = min(kb + 16 * ub, klast) & ~15;
                const int lb = a.bs_shift >= 0 ? key0 >> a.bs_shift : key0 / a.block_size;
                return gbase + (int64_t)pt.glob[lb] * a.k_sb + (int64_t)(key0 - lb * a.block_size) * a.k_ss;
            }
        };
        auto row_base = [&](int tile, int row) __attribute__((always_inline)) -> const int8_t* {
            const int key = min((t0 + tile) * kTile + row, hi - 1);
            const int lb = a.bs_shift >= 0 ? key >> a.bs_shift : key / a.block_size;
            return gbase + pt.get<kLds>(lb) * a.k_sb + (int64_t)(key - lb * a.block_size) * a.k_ss;
        };
        int2_t ent = {0, 0};  // the next tile's table entries
        auto lookup = [&](int n) __attribute__((always_inline)) {
            if constexpr (kFast && kLds) ent = *(const lds_int2*)(L + kSwBt + 8 * tile_of(n));
        };
        const int8_t *base0 = gbase, *base1 = gbase;  // of the tile being copied
        // this lane's bytes of its first K and V block, from the 16-key block's first row, and of its scale: worked out for each
        // tile again (registers are short)
        unsigned kvo, vvo;
        int sco, lc;
        auto locate = [&](int n) __attribute__((always_inline)) {
            lc = threadIdx.x;
            asm volatile("" : "+v"(lc));
            lc &= 63;
            const int lg = lc >> 4, li = lc & 15;
            kvo = (unsigned)(kFast ? (lg + 4 * r) * a.k_ss : 0) + 16u * (unsigned)(li ^ (4 * lg));
            vvo = (unsigned)(kFast ? (4 * lg + r) * a.k_ss : 0) + 260u + 16u * (unsigned)(li ^ (8 * (lg & 1)));
            sco = (kFast ? li * a.k_ss : 0) + (lc < 32 ? 256 : 516);
            if constexpr (kFast) {
                base0 = block_base(ent.x, tile_of(n), 0);
                base1 = block_base(ent.y, tile_of(n), 1);
            }
        };
        auto copy_scales = [&](int n, unsigned to) __attribute__((always_inline)) {
            if (RW == 1 || lc / (64 / RW) == r) {
                const int8_t* src;
                if constexpr (kFast)
                    src = (lc & 16 ? base1 : base0) + sco;
                else
                    src = row_base(tile_of(n), lc & 31) + sco;
                dma4_v(reinterpret_cast<const int*>(src), to);
            }
        };
        auto copy_k = [&](int n, unsigned slot) __attribute__((always_inline)) {
            static_for<0, kPer>([&](auto ic) __attribute__((always_inline)) {
                constexpr int i = decltype(ic)::value;
                const int blk = r + RW * i;  // RW = 8: r, block r / 4 of keys
                if constexpr (kFast) {
                    constexpr int q = RW < 4 ? RW * (i % (4 / RW)) : 0;
                    const int8_t* base = (RW == 8 ? r >= 4 : i >= kPer / 2) ? base1 : base0;
                    dma16_s(base + (RW == 8 ? (int64_t)(r >= 4 ? -16 * a.k_ss : 0) : (int64_t)(4 * q * a.k_ss)), kvo, slot + kImgK + blk * kBlk);
                } else {
                    dma16_v<0>(row_base(tile_of(n), 16 * (blk >> 2) + 4 * (blk & 3) + (lc >> 4)) + kvo, slot + kImgK + blk * kBlk);
                }
            });
            copy_scales(n, slot + kSwImgS);
        };
        auto copy_v = [&](int n, unsigned slot) __attribute__((always_inline)) {
            static_for<0, kPer>([&](auto ic) __attribute__((always_inline)) {
                constexpr int i = decltype(ic)::value;
                const int blk = r + RW * i;
                if constexpr (kFast) {
                    constexpr int q = RW < 4 ? RW * (i % (4 / RW)) : 0;
                    const int8_t* base = (RW == 8 ? r >= 4 : i >= kPer / 2) ? base1 : base0;
                    dma16_s(base + (RW == 8 ? (int64_t)(r >= 4 ? -4 * a.k_ss : 0) : (int64_t)(q * a.k_ss)), vvo, slot + kImgV + blk * kBlk);
                } else {
                    dma16_v<0>(row_base(tile_of(n), 16 * (blk >> 2) + (blk & 3) + 4 * (lc >> 4)) + vvo, slot + kImgV + blk * kBlk);
                }
            });
        };
        if constexpr (RW == 8) {
            unsigned slot_in = 0;  // ring position (bytes) of the next tile to copy
            auto issue = [&](int n) __attribute__((always_inline)) {
                locate(n);
                copy_k(n, group + slot_in);
                copy_v(n, group + slot_in);
                slot_in = slot_in + kSwSlot == kRing * kSwSlot ? 0 : slot_in + kSwSlot;
                lookup(n + 1);
            };
            // This wave's share of a tile's conversion: steps 2 c, 2 c + 1 of key block u and dim blocks 2 w, 2 w + 1
            const int u = w & 1, c = w >> 1;
            int ko = kImgK + (4 * u + (li >> 2)) * kBlk + 256 * (l & 3) + 64 * (c ^ (l & 3)) + 16 * lg;
            int vo = vro[0] + 32 * w - (w >= 4 && (lg & 1) ? 256 : 0);
            asm volatile("" : "+v"(ko), "+v"(vo));  // (or it keeps their terms)
            lds_u8* const fr = L + kSwWide * kSwSlot + 16 * l;
            auto convert = [&](int n, const lds_u8* S) __attribute__((always_inline)) {
                lds_u8* F = fr + (n & 1) * kSwFrag;
                const uint4_t x = *(const lds_uint4*)(S + ko);
                const int2_t y0 = __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_int2*)(S + vo));
                const int2_t y1 = __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_int2*)(S + vo + 16));
                *(lds_half8*)(F + (8 * u + 2 * c) * 1024) = widen_i8x8_exact(x.x, x.y);
                *(lds_half8*)(F + (8 * u + 2 * c + 1) * 1024) = widen_i8x8_exact(x.z, x.w);
                *(lds_half8*)(F + (16 + 2 * w) * 1024) = widen_i8x8_exact((unsigned)y0.x, (unsigned)y0.y);
                *(lds_half8*)(F + (16 + 2 * w + 1) * 1024) = widen_i8x8_exact((unsigned)y1.x, (unsigned)y1.y);
            };
            const int first = min(cnt, kRing - 1);
            lookup(0);
            for (int n = 0; n < first; ++n) issue(n);
            if (cnt >= kRing - 1)
                wait_vm<(kRing - 2) * kCopies>();
            else
                wait_vm<0>();
            __syncthreads();
            const lds_u8 *S0 = L, *S1 = L + kSwSlot;  // slots of tiles n, n + 1
            auto next_slot = [&](const lds_u8* S) __attribute__((always_inline)) {
                return S == L + (kRing - 1) * kSwSlot ? (const lds_u8*)L : S + kSwSlot;
            };
            convert(0, S0);
#pragma unroll 1
            for (int n = 0; n < cnt; ++n) {
                // tile n + 1 has landed (issued: up to n + kRing - 2; near the end all that are in flight)
                if (n + kRing - 1 <= cnt)
                    wait_vm<(kRing - 3) * kCopies>();
                else
                    wait_vm<0>();
                __syncthreads();  // tile n's fragments are there
                // The two waves of a SIMD (w, w + 4) copy and convert before and behind their products: the one's conversions run
                // beside the other's MFMAs.
                auto prepare = [&]() __attribute__((always_inline)) {
                    if (n + kRing - 1 < cnt) issue(n + kRing - 1);  // into tile n - 1's slot, which every wave is done with
                    if (n + 1 < cnt) convert(n + 1, S1);
                };
                if (w < 4) prepare();
                if (rows) {
                    const int kb = (t0 + n) * kTile;
                    const lds_u8* F = fr + (n & 1) * kSwFrag;
                    scores(kb, S0, F, nullptr);
                    values(kb, S0, F);
                }
                if (w >= 4) prepare();
                S0 = S1;
                S1 = next_slot(S1);
            }
        } else if constexpr (RW > 1) {
            unsigned slot_in = 0;  // ring position (bytes) of the next tile to copy
            auto issue = [&](int n) __attribute__((always_inline)) {
                locate(n);
                copy_k(n, group + slot_in);
                copy_v(n, group + slot_in);
                slot_in = slot_in + kSwSlot == kRing * kSwSlot ? 0 : slot_in + kSwSlot;
                lookup(n + 1);
            };
            const int first = min(mine, kRing - 1), all = (cnt + KW - 1) / KW;
            if (mine > 0) lookup(0);
            for (int n = 0; n < first; ++n) issue(n);
            const lds_u8* S = L + k * kRing * kSwSlot;
            int left = kRing;  // tiles to the ring's end
#pragma unroll 1
            for (int n = 0; n < all; ++n) {
                // tile n has landed (issued: up to n + kRing - 2; near the end all that are in flight)
                if (n + kRing - 1 <= mine)
                    wait_vm<(kRing - 2) * kCopies>();
                else
                    wait_vm<0>();
                __syncthreads();
                if (n + kRing - 1 < mine) issue(n + kRing - 1);  // into tile n - 1's slot, which every wave is done with
                if (rows && n < mine) {
                    const int kb = (t0 + KW * n + k) * kTile;
                    scores(kb, S, nullptr, nullptr);
                    values(kb, S, nullptr);
                }
                S += kSwSlot;
                if (--left == 0) {
                    left = kRing;
                    S -= kRing * kSwSlot;
                }
            }
        } else if (mine > 0) {
            // Two slots of V and scales per wave; K goes to registers, where its operands lie as the rows do. All of tile n + 1
            // is requested before tile n is computed.
            const unsigned slots = (unsigned)(uintptr_t)L + k * 2 * kSwOwn;
            uint4_t kc[8], kn[8];
            auto request = [&](int n) __attribute__((always_inline)) {
                locate(n);
                if constexpr (!kFast) {
                    base0 = row_base(tile_of(n), li);
                    base1 = row_base(tile_of(n), 16 + li);
                }
                const int ko = (kFast ? li * a.k_ss : 0) + 16 * lg;
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    __builtin_memcpy(&kn[i], __builtin_assume_aligned((i < 4 ? base0 : base1) + ko + 64 * (i & 3), 4), 16);
                copy_v(n, slots + (n & 1) * kSwOwn - kImgV);
                copy_scales(n, slots + (n & 1) * kSwOwn + (kSwOwn - 256));
                lookup(n + 1);
            };
            lookup(0);
            request(0);
#pragma unroll 1
            for (int n = 0; n < mine; ++n) {
                wait_vm<0>();
#pragma unroll
                for (int i = 0; i < 8; ++i) kc[i] = kn[i];
                if (n + 1 < mine) request(n + 1);
                const int kb = (t0 + KW * n + k) * kTile;
                const lds_u8* S = L + (k * 2 + (n & 1)) * kSwOwn - kImgV;  // (as if a K image came first)
                scores(kb, S, nullptr, kc);
                values(kb, S, nullptr);
                wait_lds();  // the slot has been read
            }
        }
    };
    if (pt.in_lds)
        tile_loop(std::true_type{});
    else
        tile_loop(std::false_type{});

    float m_run[RB];
#pragma unroll
    for (int j = 0; j < RB; ++j) {
        l_run[j] = xor_sum(xor_sum(l_run[j], 16), 32);
        m_run[j] = thr_run[j] == kNegInf ? kNegInf : -nm_run[j];
    }
    // ---- the key groups' states: the upper half's into the lower half's, until one is left ----
    if constexpr (KW > 1) {
#pragma unroll
        for (int half = KW / 2; half >= 1; half >>= 1) {
            if (half >= cnt) continue;  // (only groups below cnt have seen a tile)
            // a state: O [row block][dim block][lane] 16 bytes, then [row block][m, l][lane] 4
            __syncthreads();  // the slots, or the last step's states, have been read
            lds_u8* at = L + ((k % half) * RW + r) * (64 * RB * 264);
            if (rows && k >= half && k < 2 * half) {
#pragma unroll
                for (int j = 0; j < RB; ++j) {
#pragma unroll
                    for (int m = 0; m < 16; ++m) *(lds_float4*)(at + ((j * 16 + m) * 64 + l) * 16) = oacc[m][j];
                    *(lds_float*)(at + RB * 16384 + (2 * j * 64 + l) * 4) = m_run[j];
                    *(lds_float*)(at + RB * 16384 + ((2 * j + 1) * 64 + l) * 4) = l_run[j];
                }
            }
            __syncthreads();
            if (rows && k < half) {
#pragma unroll
                for (int j = 0; j < RB; ++j) {
                    const float m2 = *(const lds_float*)(at + RB * 16384 + (2 * j * 64 + l) * 4);
                    const float l2 = *(const lds_float*)(at + RB * 16384 + ((2 * j + 1) * 64 + l) * 4);
                    const float top = fmaxf(m_run[j], m2);
                    const float f1 = m_run[j] == kNegInf ? 0.f : __builtin_amdgcn_exp2f(m_run[j] - top);
                    const float f2 = m2 == kNegInf ? 0.f : __builtin_amdgcn_exp2f(m2 - top);
                    m_run[j] = top;
                    l_run[j] = l_run[j] * f1 + l2 * f2;
#pragma unroll
                    for (int m = 0; m < 16; ++m) oacc[m][j] = oacc[m][j] * f1 + *(const lds_float4*)(at + ((j * 16 + m) * 64 + l) * 16) * f2;
                }
            }
        }
        if (k != 0) return;
    }

    // ---- the rows' unnormalised O, running max and sum, in the decode's units (O and l carry 2^kPLog2, which m takes off) ----
    int le = threadIdx.x;
    asm volatile("" : "+v"(le));  // (nor its end's around its tile loop)
    le &= 63;
#pragma unroll
    for (int j = 0; j < RB; ++j) {
        const int x = 16 * (RB * r + j) + (le & 15);
        if (x < wk.nrow) {
            int tok, hd;
            row_at(x, tok, hd);
            const int64_t at = ((int64_t)(wk.q0 + tok) * a.Hq + (g * G + hd)) * a.nseg + wk.seg;
            float* prow = a.part_o + at * kDim + 4 * (le >> 4);
#pragma unroll
            for (int m = 0; m < 16; ++m) *reinterpret_cast<float4_t*>(prow + 16 * m) = oacc[m][j];
            if (le < 16) {
                a.part_m[at] = m_run[j];
                a.part_l[at] = l_run[j];
            }
        }
    }
}

}  // namespace pd
