// The split-K decode's workgroup (see pd_decode.hip for the method): a run of key tiles of one sequence against up to
// 48 query rows of one kv head, into one segment of the partial buffers. Shared by the decode kernels (pd_decode.hip)
// and the shared-prefix decode (pd_shared.hip).
#pragma once

#include "pd_tile.hpp"

namespace pd {

constexpr int kWaveLds = 2 * kSlot;                // LDS bytes per wave
constexpr int kWaves = 4;                          // independent tile streams per workgroup
constexpr int kThreads = 64 * kWaves;
constexpr int kBtCache = 1024;                     // block-table entries of a split kept in LDS
// With Q staged in LDS as well (block sizes that are multiples of 16) the block-table slice
// is smaller:
constexpr int kBtEarly = 384;                      // per-block row offsets (48 tiles per wave)
constexpr int kBtRaw = 384;                        // raw block-table entries (96 per wave)
constexpr int kBtWave = kBtEarly / 4;              // 16-key blocks staged per wave

// The 17 DMAs of one tile into the slot at LDS address `slot` (8 K blocks, 8 V blocks, tail).
template <bool kFast, class P>
__device__ __forceinline__ void issue_tile(const P& a, const TileSrc& src, const DmaLane& d,
                                           unsigned slot, int lane) {
    if constexpr (kFast) {
        static_for<0, 8>([&](auto ic) {
            constexpr int i = decltype(ic)::value;
            dma16_so<kImgK + i * kBlk>(src.base[i >> 2] + (int64_t)(4 * (i & 3)) * a.k_ss, d.kvo, slot);
        });
        static_for<0, 8>([&](auto ic) {
            constexpr int i = decltype(ic)::value;
            dma16_so<kImgV + i * kBlk>(src.base[i >> 2] + (int64_t)(i & 3) * a.k_ss, d.vvo, slot);
        });
        const int64_t delta = src.base[1] - src.base[0];
        dma16_vo<kImgT>(src.base[0] + (delta & -(int64_t)d.tsel) + d.toff, slot);
    } else {
        // chunk-major images: lanes 0-31 copy chunk 2 i of rows 0..31, lanes 32-63 chunk 2 i + 1
        const int8_t* row = src.base[0];  // tile row lane & 31
        const int8_t* p = row + 16 * (lane >> 5);
        dma16_v<0>(p, slot + kImgK + 0 * 1024);
        dma16_v<32>(p, slot + kImgK + 1 * 1024);
        dma16_v<64>(p, slot + kImgK + 2 * 1024);
        dma16_v<96>(p, slot + kImgK + 3 * 1024);
        dma16_v<128>(p, slot + kImgK + 4 * 1024);
        dma16_v<160>(p, slot + kImgK + 5 * 1024);
        dma16_v<192>(p, slot + kImgK + 6 * 1024);
        dma16_v<224>(p, slot + kImgK + 7 * 1024);
        dma16_v<256>(p, slot + kImgV + 0 * 1024);
        dma16_v<288>(p, slot + kImgV + 1 * 1024);
        dma16_v<320>(p, slot + kImgV + 2 * 1024);
        dma16_v<352>(p, slot + kImgV + 3 * 1024);
        dma16_v<384>(p, slot + kImgV + 4 * 1024);
        dma16_v<416>(p, slot + kImgV + 5 * 1024);
        dma16_v<448>(p, slot + kImgV + 6 * 1024);
        dma16_v<480>(p, slot + kImgV + 7 * 1024);
        dma16_v<504>(row, slot + kImgT);
    }
}

// The operands of one tile, read from its LDS slot.
struct TileOps {
    uint4_t k[4][2];  // K operand: row 16 u + li, source chunk 4 c + lg
    int2_t v[17];     // transposed V reads, one per 16-dim block
    float ks[8];      // k_scale of this lane's keys 16 u + 4 lg + j
    float vs[8];      // v_scale of the same keys
};

// One workgroup = kWaves independent waves. Wave w of split s streams tiles tb + w, tb + w + 4,
// ... of the split and computes all R query rows of the kv head for each (NRB row blocks of
// 16), so every K/V byte is loaded and widened once. Each wave double-buffers its tiles in LDS:
// tile n + 1 is copied while tile n is computed, and tile n + 2 is issued as soon as tile n is
// done, so while the wave waits it has two tiles in flight.
template <int NRB, bool kEarly>
struct PartialLds {
    static constexpr int kStats = kWaves * kWaveLds;      // m, l: [wave][NRB][16]
    static constexpr int kBt = kStats + 2 * kWaves * NRB * 16 * 4;
    static constexpr int kRaw = kBt + (kEarly ? kBtEarly : kBtCache) * 8;
    static constexpr int kQ = kRaw + (kEarly ? kBtRaw * 4 : 0);
    // (three row blocks: Q is staged in the V images of slot 1 of waves 0..2 instead, 16 rows
    // each; those slots receive their V copies only after Q is in registers)
    static constexpr bool kQInSlots = NRB >= 3;
    static constexpr int kBytes = kQ + (kEarly && !kQInSlots ? 16 * NRB * 2 * kDim : 0);
    static_assert(2 * 17 * 1024 <= kWaveLds && kWaveLds % 16 == 0,
                  "two row blocks of accumulator blocks fit the slots of their wave");
    static_assert(kBytes <= 160 * 1024, "gfx950 has 160 KiB of LDS per CU");
};

// What a workgroup computes: rows [row0, row0 + R) of one GQA group of one sequence over the key tiles
// of one split, and the segment of the partial buffers it writes.
struct Work {
    int g, b, row0;            // kv head, sequence, first row of the group
    int q0, q_len, seq_len;    // first query token, query tokens, keys (the new tokens' among them)
    int seg;                   // segment of the partial buffers
    int tb, te;                // tiles [tb, te) of the split
    bool interleave;           // the waves instead take every W-th tile from t_first + gw of the ntiles
    int t_first, ntiles, W;
    int ctx0, lo, ql;          // (kRange) position of the first query token, first visible key, query tokens computed
};

// kRange: the rows and keys are as the work says (ctx0, lo, ql) instead of the sequence's last q_len tokens in the window.
template <int NRB, bool kFast, bool kRange = false>
__device__ __forceinline__ void partial_body(const PartialParams& a, const Work& wk, unsigned char* lds) {
    // kEarly (block sizes that are multiples of 16): Q and the block-table slice are copied into
    // LDS like the tiles, and each wave's
    // first tile is issued before anything is waited for (addressed with scalar block-table
    // loads), so the copies start one memory round trip after the kernel does; the second
    // tile's K copies follow at once, its other copies after the set-up (a copy issue stalls
    // while the memory queues are full).
    constexpr bool kEarly = kFast;
    using Lds = PartialLds<NRB, kEarly>;
    constexpr int kLdsStats = Lds::kStats, kLdsBt = Lds::kBt, kLdsRaw = Lds::kRaw, kLdsQ = Lds::kQ;
    constexpr bool kQInSlots = Lds::kQInSlots;

    const int g = wk.g, b = wk.b, row0 = wk.row0, q0 = wk.q0, q_len = wk.q_len, seq_len = wk.seq_len;
    const int tb = wk.tb, te = wk.te, t_first = wk.t_first, ntiles = wk.ntiles, W = wk.W;
    const bool interleave = wk.interleave;
    const int tid = threadIdx.x, l = tid & 63, lg = l >> 4, li = l & 15;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);  // wave index, uniform by construction
    const int ql = kRange ? wk.ql : min(q_len, a.qmax);
    const int G = a.G;
    const int R = min(16 * NRB, ql * G - row0);  // rows of this workgroup: group rows row0 + [0, R)
    const int ctx0 = kRange ? wk.ctx0 : seq_len - q_len;  // absolute position of query token 0
    const int lo = kRange ? wk.lo : a.window > 0 ? max(0, ctx0 - a.window + 1) : 0;
    const int hi = seq_len;
    const int gw = kWaves * wk.seg + w;  // interleaved: this wave among the W of the (sequence, kv head)

    auto prow = [&](int r) -> int64_t {  // partial row index of query row r
        const int i = (row0 + r) / G, hh = (row0 + r) - i * G;
        return ((int64_t)(q0 + i) * a.Hq + (g * G + hh)) * a.nseg + wk.seg;
    };

    const int nt = interleave ? (gw < ntiles ? (ntiles - 1 - gw) / W + 1 : 0)
                              : max(0, (te - tb - w + kWaves - 1) / kWaves);  // tiles of this wave
    auto tile_of = [&](int n) { return interleave ? t_first + gw + W * n : tb + w + kWaves * n; };

    lds_u8* L = (lds_u8*)lds;
    const unsigned lds_base = (unsigned)(uintptr_t)L;
    const unsigned wslots = lds_base + (unsigned)(w * kWaveLds);  // this wave's two slots
    const int8_t* gbase = a.kc + (int64_t)g * a.k_sh;

    DmaLane dl;
    {
        const int qq = l >> 4, c16 = l & 15, p = l & 31;
        dl.kvo = (unsigned)(qq * a.k_ss) + 16u * (unsigned)(c16 ^ (4 * qq));
        dl.vvo = (unsigned)(4 * qq * a.k_ss) + 256u + 16u * (unsigned)(c16 ^ (8 * (qq & 1)));
        const int rr = p < 16 ? p : ((p - 16) ^ 8);  // row inside its key block of tail position p
        dl.toff = kFast ? (unsigned)(rr * a.k_ss) + 504u : 0u;
        dl.tsel = p >> 4;
    }

    // The block table is read-only for the kernel's lifetime: read it through the constant
    // address space so uniform lookups become scalar loads.
    const_int_ptr bt_row = (const_int_ptr)(uintptr_t)(a.block_table + (int64_t)b * a.bt_stride);
    PageTable pt;
    pt.glob = bt_row;
    pt.lds = (const lds_int*)(L + kLdsBt);
    pt.rows16 = (const lds_ull2*)(L + kLdsBt + (kEarly ? w * kBtWave * 8 : 0));
    pt.pfirst = max(tb * kTile, lo) / a.block_size;

    // ---- Q^T operand (B of S^T = K Q^T) of every row block; lane (lg, li) holds row 16 rb + li,
    //      dims 64 (st / 2) + 16 lg + 8 (st % 2) + [0, 8) in qop[rb][st] ----
    half8_t qop[NRB][8];
    bool rvalid[NRB];
    int rpos[NRB];
#pragma unroll
    for (int rb = 0; rb < NRB; ++rb) {
        const int r = 16 * rb + li;
        rvalid[rb] = r < R;
        const int qi = (row0 + r) / G, qh = (row0 + r) - qi * G;
        rpos[rb] = ctx0 + qi;
        if constexpr (kEarly) continue;
        const _Float16* qrow =
            a.q + (int64_t)(q0 + (rvalid[rb] ? qi : 0)) * a.q_st + (int64_t)(g * G + (rvalid[rb] ? qh : 0)) * kDim;
#pragma unroll
        for (int st = 0; st < 8; ++st) {
            half8_t v;
            const int dim = 64 * (st >> 1) + 16 * lg + 8 * (st & 1);
            __builtin_memcpy(&v, __builtin_assume_aligned(qrow + dim, 4), 16);
            qop[rb][st] = rvalid[rb] ? v : (half8_t)(_Float16)0.0f;
        }
    }
    asm volatile("" ::: "memory");  // every Q load is issued before the block table is read

    // Running state per row block: max (log2 units), this lane's partial sum of p, and O^T in
    // 17 blocks of 16 "dims" (block m < 16: dims 16 m - 4 .. 16 m + 11; block 16: dims 244..255,
    // then 4 rows from the v_scale bytes in lane group 3, never stored).
    float m_run[NRB], l_run[NRB];
    float4_t oacc[NRB][17];
#pragma unroll
    for (int rb = 0; rb < NRB; ++rb) {
        m_run[rb] = kNegInf;
        l_run[rb] = 0.f;
#pragma unroll
        for (int m = 0; m < 17; ++m) oacc[rb][m] = (float4_t)0.f;
    }

    // ---- block-table slice of the split into LDS ----
    if constexpr (kEarly) {
        // the wave's own blocks (two per tile) are staged in its part of the table
        const int nblk = 2 * nt;
        pt.in_lds = nblk <= kBtWave;
        // block j of this wave: the first key of its 16-key block clamped into the tile's visible
        // keys (the tile_src rule), and that key's page
        auto wave_block = [&](int j, int& key0, int& lb) {
            const int kb = tile_of(j >> 1) * kTile;
            const int kfirst = max(kb, lo), klast = min(kb + kTile - 1, hi - 1);
            key0 = min(max(kb + 16 * (j & 1), kfirst), klast) & ~15;
            lb = a.bs_shift >= 0 ? key0 >> a.bs_shift : key0 / a.block_size;
        };
        // (0) the block-table entries of this wave's first two tiles (scalar loads), requested
        //     before any copy so that they do not queue behind the kernel's first copies
        //     (all four entries in one round trip; the tile_src rule, keys clamped into the tile's
        //     visible range, which also keeps the entries of a missing tile in bounds)
        int key0[4], lb[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int kb = tile_of(i >> 1) * kTile;
            const int kfirst = max(kb, lo), klast = min(kb + kTile - 1, hi - 1);
            key0[i] = min(max(kb + 16 * (i & 1), kfirst), klast) & ~15;
            lb[i] = a.bs_shift >= 0 ? key0[i] >> a.bs_shift : key0[i] / a.block_size;
        }
        int ent[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) ent[i] = pt.glob[lb[i]];
        TileSrc src0, src1;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int8_t* base = gbase + (int64_t)ent[i] * a.k_sb + (int64_t)(key0[i] - lb[i] * a.block_size) * a.k_ss;
            if (i < 2)
                src0.base[i] = base;
            else
                src1.base[i - 2] = base;
        }
        // (1) Q rows (two 512-byte rows per copy; rows past R repeat row R - 1), spread over the
        //     waves, and the raw block-table entries of each wave's blocks
        const int nq = (R + 1) / 2;
        for (int i = w; i < nq; i += kWaves) {
            const int r = row0 + min(2 * i + (l >> 5), R - 1);
            const int qi = r / G, qh = r - qi * G;
            const _Float16* qrow = a.q + (int64_t)(q0 + qi) * a.q_st + (int64_t)(g * G + qh) * kDim;
            const int qdst = kQInSlots ? (2 * i / 16) * kWaveLds + kSlot + kImgV + (2 * i % 16) * (2 * kDim)
                                       : kLdsQ + 1024 * i;
            dma16_v<0>(reinterpret_cast<const int8_t*>(qrow) + 16 * (l & 31), lds_base + (unsigned)qdst);
        }
        if (pt.in_lds) {
            const int* bt_glob = a.block_table + (int64_t)b * a.bt_stride;
            for (int j0 = 0; j0 < nblk; j0 += 64) {
                if (j0 + l < nblk) {  // lanes past the wave's blocks write nothing
                    int key0, lb;
                    wave_block(j0 + l, key0, lb);
                    dma4_v(bt_glob + lb, lds_base + (unsigned)(kLdsRaw + 4 * (w * kBtWave + j0)));
                }
            }
        }
        // (2) this wave's first tile
        if (nt > 0) issue_tile<kFast>(a, src0, dl, wslots, l);
        // the K blocks of the second tile follow at once, its other copies after the set-up
        if (nt > 1) {
            static_for<0, 8>([&](auto ic) {
                constexpr int i = decltype(ic)::value;
                dma16_so<kSlot + kImgK + i * kBlk>(src1.base[i >> 2] + (int64_t)(4 * (i & 3)) * a.k_ss, dl.kvo, wslots);
            });
        }
        // (3) wait for (1) only
        if (nt > 1)
            wait_vm<25>();
        else if (nt > 0)
            wait_vm<17>();
        else
            wait_vm<0>();
        __syncthreads();
        if (pt.in_lds) {  // the wave's own entries have landed (the wait above): row offsets
            const lds_int* raw = (const lds_int*)(L + kLdsRaw) + w * kBtWave;
            lds_u64* dst = (lds_u64*)(L + kLdsBt) + w * kBtWave;
            for (int j = l; j < nblk; j += 64) {
                int key0, lb;
                wave_block(j, key0, lb);
                dst[j] = (uint64_t)((int64_t)raw[j] * a.k_sb + (int64_t)(key0 - lb * a.block_size) * a.k_ss);
            }
        }
#pragma unroll
        for (int rb = 0; rb < NRB; ++rb) {
            const lds_u8* qrow = kQInSlots ? L + rb * kWaveLds + kSlot + kImgV + li * (2 * kDim)
                                           : L + kLdsQ + (16 * rb + li) * (2 * kDim);
#pragma unroll
            for (int st = 0; st < 8; ++st) {
                const int dim = 64 * (st >> 1) + 16 * lg + 8 * (st & 1);
                const half8_t v = *(const lds_half8*)(qrow + 2 * dim);
                qop[rb][st] = rvalid[rb] ? v : (half8_t)(_Float16)0.0f;
            }
        }
        __syncthreads();  // the block offsets are visible
        if (nt > 1) {
            static_for<0, 8>([&](auto ic) {
                constexpr int i = decltype(ic)::value;
                dma16_so<kSlot + kImgV + i * kBlk>(src1.base[i >> 2] + (int64_t)(i & 3) * a.k_ss, dl.vvo, wslots);
            });
            const int64_t delta = src1.base[1] - src1.base[0];
            dma16_vo<kSlot + kImgT>(src1.base[0] + (delta & -(int64_t)dl.tsel) + dl.toff, wslots);
        }
    } else {
        const int pk_first = max(tb * kTile, lo), pk_last = min(te * kTile, hi) - 1;
        const int* bt_glob = a.block_table + (int64_t)b * a.bt_stride;
        if constexpr (kFast) {
            // byte offset (from this kv head's base) of the first row of every 16-key block of
            // the split, two per tile; blocks outside [lo, hi) point at a visible block of the tile
            const int nblk = 2 * (te - tb);
            pt.in_lds = nblk <= kBtCache;
            if (pt.in_lds) {
                lds_u64* dst = (lds_u64*)(L + kLdsBt);
                for (int i = tid; i < nblk; i += kThreads) {
                    const int kb = (tb + (i >> 1)) * kTile;
                    const int kfirst = max(kb, lo), klast = min(kb + kTile - 1, hi - 1);
                    const int key0 = min(max(kb + 16 * (i & 1), kfirst), klast) & ~15;
                    const int lb = key0 / a.block_size;
                    dst[i] = (uint64_t)((int64_t)bt_glob[lb] * a.k_sb + (int64_t)(key0 - lb * a.block_size) * a.k_ss);
                }
            }
        } else {
            const int npages = pk_last / a.block_size - pt.pfirst + 1;
            pt.in_lds = npages <= kBtCache;
            if (pt.in_lds) {
                lds_int* dst = (lds_int*)(L + kLdsBt);
                for (int i = tid; i < npages; i += kThreads) dst[i] = bt_glob[pt.pfirst + i];
            }
        }
        __syncthreads();
    }

    // ---- per-lane LDS read offsets inside a slot ----
    // K operand (u, c): row 16 u + li, source chunk 4 c + lg
    int kro[4];
#pragma unroll
    for (int c = 0; c < 4; ++c)
        kro[c] = kFast ? kImgK + (li >> 2) * kBlk + 256 * (li & 3) + 64 * (c ^ (li & 3)) + 16 * lg
                       : kImgK + (4 * c + lg) * 512 + 16 * li;
    constexpr int kKroU = kFast ? 4 * kBlk : 256;  // + for key block u = 1
    // transposed V reads: lane pair (2 i, 2 i + 1) of a 16-lane group names tile row tkey
    const int tslot = li >> 1;
    const int tkey = tslot < 4 ? 4 * lg + tslot : 16 + 4 * lg + (tslot - 4);
    const int th = 8 * (li & 1);
    // chunk m of row tkey: fast: block (tkey & 3) + 4 (tkey >> 4), slot lg, position m ^ 8 (lg & 1)
    const int vblk = kImgV + ((tkey & 3) + 4 * (tkey >> 4)) * kBlk + 256 * lg + th;
    const int vro_lo = kFast ? vblk + ((lg & 1) ? 128 : 0) : kImgV + 16 * tkey + th;   // chunks 0..7
    const int vro_hi = kFast ? vblk - ((lg & 1) ? 128 : 0) : kImgV + 16 * tkey + th;   // chunks 8..15
    constexpr int kVroStep = kFast ? 16 : 512;
    const int tpos = kFast ? (tkey < 16 ? tkey : 16 + ((tkey - 16) ^ 8)) : tkey;
    const int vro_t = kImgT + 16 * tpos + th;
    // scales of this lane's keys 16 u + 4 lg + j: k_scale = first word of V chunk 0, v_scale
    // the last word of the tail
    int kso[2], vso[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        const int t0 = 16 * u + 4 * lg;
        kso[u] = kFast ? kImgV + (4 * u) * kBlk + 256 * lg + ((lg & 1) ? 128 : 0) : kImgV + 16 * t0;
        const int tp0 = kFast ? (u == 0 ? t0 : 16 + ((t0 - 16) ^ 8)) : t0;
        vso[u] = kImgT + 16 * tp0 + 12;
    }
    constexpr int kKsoStep = kFast ? kBlk : 16;  // + per j

    int tile_cur = tb;  // the tile being computed

    // ---- S^T = K Q^T for every row block (K exact in fp16, the widening bias removed before the
    //      products), times k_scale, relative to the running max: sv = s - m (log2 units; s itself
    //      while a row has no max yet); masked scores are -inf. Returns whether some row has to
    //      raise its max: its tile max exceeds the running max by more than kLazy, or it has none ----
    auto tile_scores = [&](const TileOps& o, float (&sv)[NRB][8], bool& interior) __attribute__((always_inline)) {
        float4_t sacc[NRB][2];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const uint4_t* kr = o.k[c];
#pragma unroll
            for (int hh = 0; hh < 2; ++hh) {
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    // K exact in fp16 (no widening bias): the accumulator holds only partial
                    // scores, whose rounding is ~1152 / |k| times smaller than with the bias
                    // removed at the end
                    const half8_t kf = hh == 0 ? widen_i8x8_exact(kr[u].x, kr[u].y) : widen_i8x8_exact(kr[u].z, kr[u].w);
#pragma unroll
                    for (int rb = 0; rb < NRB; ++rb)
                        sacc[rb][u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                            kf, qop[rb][2 * c + hh], (c | hh) ? sacc[rb][u] : (float4_t)0.f, 0, 0, 0);
                }
            }
        }
        float ks[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) ks[e] = o.ks[e] * a.scale_log2;
        const int kb = tile_cur * kTile;
        // Interior tile: every key is visible to every row (padding rows have Q = 0 and are
        // never written out), so no per-element mask is needed.
        interior = kb >= lo && kb + kTile <= hi;
        if (a.causal) interior = interior && kb + kTile - 1 <= ctx0;
        if (a.window > 0) interior = interior && (ctx0 + ql - 1) - kb < a.window;
        bool need = false;
#pragma unroll
        for (int rb = 0; rb < NRB; ++rb) {
            const bool fresh = m_run[rb] == kNegInf;
            const float nm = fresh ? 0.f : -m_run[rb];
            // the scores are formed in place in both cases (no copies where the paths meet); a tile
            // at the edge of the visible range then masks its invisible keys to -inf
#pragma unroll
            for (int e = 0; e < 8; ++e) sv[rb][e] = __builtin_fmaf(sacc[rb][e >> 2][e & 3], ks[e], nm);
            if (!interior) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int t = kb + 16 * (e >> 2) + 4 * lg + (e & 3);
                    const int rp = rpos[rb];
                    const bool vis = rvalid[rb] & (t >= lo) & (t < hi) & (!a.causal | (t <= rp)) &
                                     ((a.window <= 0) | ((rp - t) < a.window));
                    sv[rb][e] = vis ? sv[rb][e] : kNegInf;
                }
            }
            float mx = kNegInf;
#pragma unroll
            for (int e = 0; e < 8; ++e) mx = fmaxf(mx, sv[rb][e]);
            need |= fresh ? mx > kNegInf : mx > kLazy;
        }
        return need;
    };

    // rare path: raise the running max of the rows that need it, shift their relative scores and
    // rescale their state
    // With three row blocks the rescale goes through LDS (4 KiB of scratch in V blocks 4..7 of
    // the current tile's slot: its operands are all in registers by now, and only the K image and
    // V blocks 0..3 can already be refilling): the accumulators are then only ever
    // touched by MFMAs and by asm with AGPR operands, so the compiler keeps them in the AGPR
    // file (multiplying them in place made it spill ~250 registers, partly in the fast loop).
    // With fewer row blocks the registers suffice and the multiply in place is faster.
    auto raise_max = [&](float (&sv)[NRB][8], lds_u8* scr_slot) __attribute__((always_inline)) {
        const unsigned scr = (unsigned)(uintptr_t)(scr_slot + 16 * l);
#pragma unroll
        for (int rb = 0; rb < NRB; ++rb) {
            float mloc = kNegInf;
#pragma unroll
            for (int e = 0; e < 8; ++e) mloc = fmaxf(mloc, sv[rb][e]);
            const float mrow = xor_max(xor_max(mloc, 16), 32);  // tile max, relative to m_run
            const bool fresh = m_run[rb] == kNegInf;
            const bool raise = fresh ? mrow > kNegInf : mrow > kLazy;
            const float shift = raise ? mrow : 0.f;
            const float alpha = fresh ? 0.f : __builtin_amdgcn_exp2f(-shift);
            if (raise) m_run[rb] = fresh ? mrow : m_run[rb] + mrow;
#pragma unroll
            for (int e = 0; e < 8; ++e) sv[rb][e] -= shift;
            l_run[rb] *= alpha;
            // O is still zero while every row of the block is fresh, and a row that keeps its
            // max would be multiplied by 1: rescale only when a row with state raises
            if (__builtin_amdgcn_ballot_w64(raise && !fresh) != 0) {
                if constexpr (NRB >= 3) {
#pragma unroll
                    for (int m = 0; m < 16; m += 4)
                        agpr_scale4_via_lds(oacc[rb][m], oacc[rb][m + 1], oacc[rb][m + 2], oacc[rb][m + 3], alpha, scr);
                    agpr_scale_via_lds(oacc[rb][16], alpha, scr);
                } else {
#pragma unroll
                    for (int m = 0; m < 17; ++m) oacc[rb][m] *= alpha;
                }
            }
        }
    };

    // ---- p = 2^sv; P' = p * v_scale * 16 as two fp16 parts (hi + lo, ~22 significant bits: a
    //      single fp16 would put 2^-12 relative error on every term, too much next to outlier V
    //      rows); then O^T += V^T hi^T + V^T lo^T for every row block, V widened exactly (no
    //      bias: the fp32 accumulators hold only the products' own sums) ----
    auto tile_values = [&](const TileOps& o, const float (&sv)[NRB][8], bool interior) __attribute__((always_inline)) {
        float vsc[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) vsc[e] = o.vs[e] * kPScale;
        if (!interior) {  // outside [lo, hi) a scale may be garbage or NaN: use 0
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int t = tile_cur * kTile + 16 * (e >> 2) + 4 * lg + (e & 3);
                vsc[e] = (t >= lo) & (t < hi) ? vsc[e] : 0.f;
            }
        }
        half8_t phi[NRB], plo[NRB];
#pragma unroll
        for (int rb = 0; rb < NRB; ++rb) {
            float psum = 0.f;
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
                const float p0 = __builtin_amdgcn_exp2f(sv[rb][e]);  // masked: 2^-inf = 0
                const float p1 = __builtin_amdgcn_exp2f(sv[rb][e + 1]);
                psum += p0;
                psum += p1;
                half2_t h, lo;
                split_fp16x2(p0, vsc[e], p1, vsc[e + 1], h, lo);
                phi[rb][e] = h.x;
                phi[rb][e + 1] = h.y;
                plo[rb][e] = lo.x;
                plo[rb][e + 1] = lo.y;
            }
            l_run[rb] += psum;
        }
#pragma unroll
        for (int m = 0; m < 17; ++m) {
            const half8_t vf = widen_i8x8_exact((unsigned)o.v[m].x, (unsigned)o.v[m].y);
#pragma unroll
            for (int rb = 0; rb < NRB; ++rb)
                oacc[rb][m] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, phi[rb], oacc[rb][m], 0, 0, 0);
#pragma unroll
            for (int rb = 0; rb < NRB; ++rb)
                oacc[rb][m] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, plo[rb], oacc[rb][m], 0, 0, 0);
        }
    };

    // ---- every operand of a tile from its slot into registers, so the slot can be refilled
    //      before the tile is computed: v_scale of this lane's keys, the K operand, k_scale, and
    //      the 17 transposed V reads ----
    auto read_ops = [&](lds_u8* T, TileOps& o) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int j = 0; j < 4; ++j) o.vs[4 * u + j] = *(const lds_float*)(T + vso[u] + 16 * j);
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int u = 0; u < 2; ++u) o.k[c][u] = *(const lds_uint4*)(T + kro[c] + u * kKroU);
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int j = 0; j < 4; ++j) o.ks[4 * u + j] = *(const lds_float*)(T + kso[u] + j * kKsoStep);
#pragma unroll
        for (int m = 0; m < 17; ++m) {
            const int ofs = m < 8 ? vro_lo + kVroStep * m : (m < 16 ? vro_hi + kVroStep * m : vro_t);
            o.v[m] = __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_int2*)(T + ofs));
        }
    };

    // ---- the tile stream of this wave ----
    auto tile_loop = [&](auto lds_flag) __attribute__((always_inline)) {
        constexpr bool kLds = decltype(lds_flag)::value;
        auto issue = [&](int n) __attribute__((always_inline)) {
            wait_lds();  // every LDS access to the slot being refilled has completed
            issue_tile<kFast>(a, tile_src<kFast, kLds>(a, pt, gbase, tile_of(n), n, lo, hi, l), dl,
                              wslots + (unsigned)((n & 1) * kSlot), l);
        };
        // The same copies in two parts (16-key row blocks): the 8 K blocks, then the 8 V blocks
        // and the tail, from the addresses the first part looked up.
        TileSrc nsrc;
        auto issue_k = [&](int n) __attribute__((always_inline)) {
            wait_lds();  // every LDS access to the slot being refilled has completed
            nsrc = tile_src<kFast, kLds>(a, pt, gbase, tile_of(n), n, lo, hi, l);
            const unsigned slot = wslots + (unsigned)((n & 1) * kSlot);
            static_for<0, 8>([&](auto ic) {
                constexpr int i = decltype(ic)::value;
                dma16_so<kImgK + i * kBlk>(nsrc.base[i >> 2] + (int64_t)(4 * (i & 3)) * a.k_ss, dl.kvo, slot);
            });
        };
        // While the stream ramps up (the refills of its first kRampTiles tiles) the first four V
        // blocks go between the scores and the values, the rest after the values.
        constexpr int kRampTiles = 2;
        auto ramp = [&](int n) { return n - 2 < kRampTiles; };  // refill n is issued by iteration n - 2
        auto issue_v0 = [&](int n) __attribute__((always_inline)) {
            const unsigned slot = wslots + (unsigned)((n & 1) * kSlot);
            static_for<0, 4>([&](auto ic) {
                constexpr int i = decltype(ic)::value;
                dma16_so<kImgV + i * kBlk>(nsrc.base[i >> 2] + (int64_t)(i & 3) * a.k_ss, dl.vvo, slot);
            });
        };
        auto issue_v = [&](int n) __attribute__((always_inline)) {
            const unsigned slot = wslots + (unsigned)((n & 1) * kSlot);
            if (!ramp(n)) {
                static_for<0, 4>([&](auto ic) {
                    constexpr int i = decltype(ic)::value;
                    dma16_so<kImgV + i * kBlk>(nsrc.base[i >> 2] + (int64_t)(i & 3) * a.k_ss, dl.vvo, slot);
                });
            }
            static_for<4, 8>([&](auto ic) {
                constexpr int i = decltype(ic)::value;
                dma16_so<kImgV + i * kBlk>(nsrc.base[i >> 2] + (int64_t)(i & 3) * a.k_ss, dl.vvo, slot);
            });
            const int64_t delta = nsrc.base[1] - nsrc.base[0];
            dma16_vo<kImgT>(nsrc.base[0] + (delta & -(int64_t)dl.tsel) + dl.toff, slot);
        };
        // The first two tiles (issued during the set-up when kEarly): all loads the compiler can
        // see (Q, block table) have been waited for by now, so no compiler-inserted wait will
        // include these copies.
        if constexpr (!kEarly) {
            if (nt > 0) issue(0);
            if (nt > 1) issue(1);
        }
        float sv[NRB][8];
        TileOps ops;
        bool interior = true;
        int n = 0;
        // The fast inner loop never rescales: O stays in the MFMA accumulators, untouched by
        // the vector ALU. When some row's max must be raised the loop is left, the rows are
        // rescaled, the tile is finished and the loop resumes with the next tile.
        while (n < nt) {
            bool rare = false;
            for (; n < nt; ++n) {
                if (n + 1 < nt)
                    wait_vm<17>();  // tile n has landed; tile n + 1 may still be in flight
                else
                    wait_vm<0>();
                lds_u8* T = L + w * kWaveLds + (n & 1) * kSlot;
                tile_cur = tile_of(n);
                read_ops(T, ops);
                if (kFast && n + 2 < nt) issue_k(n + 2);
                const bool need = tile_scores(ops, sv, interior);
                if (kFast && n + 2 < nt && ramp(n + 2)) issue_v0(n + 2);
                if (__builtin_amdgcn_ballot_w64(need) != 0) {
                    rare = true;
                    break;
                }
                tile_values(ops, sv, interior);
                if (n + 2 < nt) {
                    if constexpr (kFast)
                        issue_v(n + 2);
                    else
                        issue(n + 2);
                }
            }
            if (!rare) break;
            raise_max(sv, L + w * kWaveLds + (n & 1) * kSlot + kImgV + 4 * kBlk);
            tile_values(ops, sv, interior);
            if (n + 2 < nt) {
                if constexpr (kFast)
                    issue_v(n + 2);
                else
                    issue(n + 2);
            }
            ++n;
        }
    };
    if (pt.in_lds)
        tile_loop(std::true_type{});
    else
        tile_loop(std::false_type{});

    // ---- merge the waves through LDS and write one partial per row ----
    {
        // Each wave stores its accumulators as they are (a 1 KiB block per accumulator and row
        // block, straight from the AGPRs: no vector ALU work) into its own slots as soon as its
        // tiles are done, with its per-row max and sum. Row blocks go through the slots two at a
        // time (kRawRounds rounds). Dims of an accumulator block: block m < 16 holds dims
        // 16 m - 4 + 4 lg .. + 3 in lane group lg (row li), block 16 holds 244..255 in lane
        // groups 0-2. Row factors: M = max_w m_w, e_w = 2^(m_w - M), O = sum_w e_w O_w / 16,
        // L = sum_w e_w l_w.
        //
        // Two or three row blocks: thread (row, 32 dims) derives the factors of its row, sums the
        // four waves' blocks with them and writes its part of the row (a block holds the float4 of
        // (lg, row rr) at 16 lg + rr).
        //
        // One row block (at most 16 rows, single-token decodes): each wave takes whole rows, so
        // the lanes of rows that do not exist issue nothing. For one row the 64 lanes read dims
        // 4 L .. 4 L + 3 (block (L + 1) / 4, group (L + 1) % 4) and store the row's 1 KiB with one
        // instruction. A block then holds the float4 of (lg, rr) at 16 lg + ((rr + lg + 4 (m & 3))
        // & 15), so that the row reads (position (rr + L + 1) & 15) and the stores (16 rows of
        // one lane group) both spread over all banks. (With two row blocks this layout measured
        // 0.26 us slower per launch at 24 rows.)
        constexpr bool kRowStores = NRB == 1;
        constexpr int kRawRounds = (NRB + 1) / 2;
        float* wm = reinterpret_cast<float*>(lds + kLdsStats);  // [wave][NRB][16] running max
        float* wl = wm + kWaves * NRB * 16;                     // [wave][NRB][16] row sum of p
#pragma unroll
        for (int rb = 0; rb < NRB; ++rb) {
            const float l_row = xor_sum(xor_sum(l_run[rb], 16), 32);
            if (lg == 0) {
                wm[(w * NRB + rb) * 16 + li] = m_run[rb];
                wl[(w * NRB + rb) * 16 + li] = l_row;
            }
        }
        unsigned raw[4];  // this wave's slots, by block index m & 3
#pragma unroll
        for (int k = 0; k < 4; ++k)
            raw[k] = lds_base + (unsigned)(w * kWaveLds + 16 * (kRowStores ? 16 * lg + ((li + lg + 4 * k) & 15) : l));
        auto store_round = [&](int rd) __attribute__((always_inline)) {
#pragma unroll
            for (int rb = 2 * rd; rb < 2 * rd + 2 && rb < NRB; ++rb)
#pragma unroll
                for (int m = 0; m < 17; ++m)
                    asm volatile("ds_write_b128 %0, %1 offset:%2" ::"v"(raw[m & 3]), "a"(oacc[rb][m]),
                                 "i"(((rb - 2 * rd) * 17 + m) * 1024)
                                 : "memory");
        };
        store_round(0);
        wait_lds();
        __syncthreads();  // every wave's stats and first accumulator blocks are in LDS
        auto factors = [&](int row, float* f) __attribute__((always_inline)) {
            float M = kNegInf;
#pragma unroll
            for (int v = 0; v < kWaves; ++v) M = fmaxf(M, wm[v * NRB * 16 + row]);
            float Lr = 0.f;
#pragma unroll
            for (int v = 0; v < kWaves; ++v) {
                const float mw = wm[v * NRB * 16 + row];
                const float e = mw == kNegInf ? 0.f : exp2f(mw - M);
                f[v] = e * (1.0f / kPScale);
                Lr += e * wl[v * NRB * 16 + row];
            }
            return float2_t{M, Lr};
        };
        if constexpr (kRowStores) {
            // wave w takes rows w + 4 j; lane j computes the factors of row j of its wave, which
            // are then read from it as scalars
            const int rown = w + 4 * (l & 3);
            float f[kWaves];
            const float2_t ml = factors(rown, f);
            if (l < 4 && rown < R) {
                const int64_t pr = prow(rown);
                a.part_m[pr] = ml.x;
                a.part_l[pr] = ml.y;
            }
            const int m_l = l < 63 ? (l + 1) >> 2 : 16;
            const int g_l = l < 63 ? (l + 1) & 3 : 2;
            const lds_u8* rd_base = L + (m_l * 1024 + 256 * g_l);
            const int c_l = g_l + 4 * (m_l & 3);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int row = w + 4 * j;  // uniform
                if (row >= R) break;
                const lds_u8* p = rd_base + 16 * ((row + c_l) & 15);
                float fs[kWaves];
#pragma unroll
                for (int v = 0; v < kWaves; ++v)
                    fs[v] = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, f[v]), j));
                float4_t acc = *(const lds_float4*)p * fs[0];
#pragma unroll
                for (int v = 1; v < kWaves; ++v) acc += *(const lds_float4*)(p + v * kWaveLds) * fs[v];
                *reinterpret_cast<float4_t*>(a.part_o + prow(row) * kDim + 4 * l) = acc;
            }
        } else {
#pragma unroll
            for (int rd = 0; rd < kRawRounds; ++rd) {
                if (rd > 0) {
                    store_round(rd);
                    wait_lds();
                    __syncthreads();
                }
                // thread: row 32 rd + (lane & 31), wave w's two 32-dim parts
                const int row = 32 * rd + (l & 31), part = 2 * w + (l >> 5);
                if (row < R) {
                    float f[kWaves];
                    const float2_t ml = factors(row, f);
                    const int64_t pr = prow(row);
                    if (part == 0) {
                        a.part_m[pr] = ml.x;
                        a.part_l[pr] = ml.y;
                    }
                    const int rbl = (row >> 4) - 2 * rd;  // row block within the round
                    float* dst = a.part_o + pr * kDim;
                    const float4_t* rawp = reinterpret_cast<const float4_t*>(lds);
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const int d = 32 * part + 4 * j;
                        const int m = d < 252 ? (d + 4) >> 4 : 16;
                        const int glg = d < 252 ? ((d + 4) >> 2) & 3 : 2;
                        const int blk = (rbl * 17 + m) * 64 + 16 * glg + (row & 15);
                        float4_t acc = rawp[blk] * f[0];
#pragma unroll
                        for (int v = 1; v < kWaves; ++v) acc += rawp[v * (kWaveLds / 16) + blk] * f[v];
                        *reinterpret_cast<float4_t*>(dst + d) = acc;
                    }
                }
                if (rd + 1 < kRawRounds) __syncthreads();  // the blocks are rewritten for the next round
            }
        }
    }
}

}  // namespace pd
