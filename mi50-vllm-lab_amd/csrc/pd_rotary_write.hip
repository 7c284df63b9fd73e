// Rotary positions and the cache write of one layer's new tokens in one launch: the query heads are
// rotated (in place or into another tensor), the key heads are rotated and quantised with the value heads into
// the 520-byte cache rows. Between the projection and the attention a token's query is then read and written once and
// its key read once; the rotated key never leaves the registers.
//
// Pair i of a head, i < rotary_dim / 2, is (x, y) = dims (i, i + rotary_dim / 2), or (2 i, 2 i + 1) when
// interleaved; with c, s = cos_sin[position][i], cos_sin[position][rotary_dim / 2 + i] it becomes
// (x c - y s, y c + x s), in fp32 with each product and each sum rounded (no fma), so that the result does not
// depend on which form the compiler would contract; the dims from rotary_dim on stay as they are. The key is quantised
// from these fp32 values (pd_quant.hpp), without a rounding to its input type in between.
//
// A head is 32 octets of 8 values: octet o < rotary_dim / 8 holds pairs 4 o .. 4 o + 3 (two runs of four dims,
// rotary_dim / 2 apart or adjacent), the others eight dims that are not rotated. A lane takes one octet, so
// no value crosses lanes before the row's absmax, both layouts read the same table entries with two 16-byte loads, and a
// head in place touches only its rotated octets.
//
// What bounds it: small calls a trip to memory for positions and slots and one for the rows (2.8 us at 1 token, 3.8 at 129); large ones
// memory, 32,768 fp16 tokens of 12 / 2 heads 113 us for 537 MB, 4.7 TB/s; bf16 109, fp32 into fp32 190 for 1,008 MB, 5.3 TB/s (24 / 4 heads
// 203, 201 and 364).
#include "pd_quant.hpp"
#include "pth_dec.h"

namespace pd {

// Pairs (a[e], b[e]) (half layout) or (a[0], a[1]), (a[2], a[3]), (b[0], ...) (interleaved) by the angles c, s.
__device__ __forceinline__ void rotate_octet(float4_t& a, float4_t& b, float4_t c, float4_t s, bool interleaved) {
#pragma clang fp contract(off)
    if (interleaved) {
        const float4_t x = {a.x, a.z, b.x, b.z}, y = {a.y, a.w, b.y, b.w};
        const float4_t u = x * c - y * s, v = y * c + x * s;
        a = float4_t{u.x, v.x, u.y, v.y};
        b = float4_t{u.z, v.z, u.w, v.w};
    } else {
        const float4_t x = a, y = b;
        a = x * c - y * s;
        b = y * c + x * s;
    }
}

// First dims of the two runs of octet o.
struct OctetDims {
    int a, b;
};
__device__ __forceinline__ OctetDims octet_dims(int o, int rotary_dim, bool interleaved) {
    const int n = rotary_dim >> 3;
    if (o < n && !interleaved) return {4 * o, 4 * o + (rotary_dim >> 1)};
    return {8 * o, 8 * o + 4};
}

// Heads of one token that a group of lanes takes, their loads in flight together and the angles read once. One head instead:
// 4,096 bf16 tokens 54.6 us with their rows read back, four 50.2; 1,024 18.7 and 17.6; from 1 token to 512 the same (1: 2.8 us, 129: 3.8).
constexpr int kHeads = 4;

// kLanes: lanes of a head (each an octet). Workgroups [0, kv_groups) take key/value rows, 32 lanes each, the others query heads.
template <class In, class Out, int kLanes>
__global__ void __launch_bounds__(256) pd_rotary_write_kernel(const RotaryWriteParams a) {
    const int rd = a.rotary_dim, half = rd >> 1, nrot = rd >> 3;
    const bool il = a.interleaved != 0;
    if ((int)blockIdx.x < a.kv_groups) {
        const int row = (int)blockIdx.x * 8 + (threadIdx.x >> 5), o = threadIdx.x & 31;
        if (row >= a.T * a.Hkv) return;
        const int t = row / a.Hkv, h = row - t * a.Hkv;
        const int64_t pos = a.positions[t], slot = a.slots[t];
        if (pos < 0 || pos >= a.max_positions || slot < 0 || slot >= a.num_slots) return;
        const OctetDims d = octet_dims(o, rd, il);
        const In* kin = static_cast<const In*>(a.key) + t * a.k_st + h * a.k_sh;
        const In* vin = static_cast<const In*>(a.value) + t * a.v_st + h * a.v_sh + 8 * o;
        float4_t k0 = load4(kin + d.a), k1 = load4(kin + d.b);
        const float4_t v0 = load4(vin), v1 = load4(vin + 4);
        if (o < nrot) {
            const float* cs = a.cos_sin + pos * a.cs_st + 4 * o;
            rotate_octet(k0, k1, *reinterpret_cast<const float4_t*>(cs), *reinterpret_cast<const float4_t*>(cs + half), il);
        }
        float km = row16_max(fmaxf(absmax4(k0), absmax4(k1))), vm = row16_max(fmaxf(absmax4(v0), absmax4(v1)));
        km = fmaxf(km, __shfl_xor(km, 16, 64));
        vm = fmaxf(vm, __shfl_xor(vm, 16, 64));
        const float ks = km / 127.f, vs = vm / 127.f;
        const int64_t blk = slot / a.block_size, off = slot - blk * a.block_size;
        int8_t* r = a.kc + blk * a.c_sb + off * a.c_ss + h * a.c_sh;
        *reinterpret_cast<unsigned*>(r + d.a) = quant4(k0, ks);
        *reinterpret_cast<unsigned*>(r + d.b) = quant4(k1, ks);
        *reinterpret_cast<unsigned*>(r + 260 + 8 * o) = quant4(v0, vs);
        *reinterpret_cast<unsigned*>(r + 264 + 8 * o) = quant4(v1, vs);
        if (o == 0) {
            *reinterpret_cast<float*>(r + 256) = ks;
            *reinterpret_cast<float*>(r + 516) = vs;
        }
        return;
    }
    const int groups = (a.Hq + kHeads - 1) / kHeads;  // of a token
    const int64_t unit = (int64_t)((int)blockIdx.x - a.kv_groups) * (256 / kLanes) + threadIdx.x / kLanes;
    if (unit >= (int64_t)a.T * groups) return;
    const int t = (int)(unit / groups), h0 = (int)(unit - (int64_t)t * groups) * kHeads, o = threadIdx.x % kLanes;
    const int64_t pos = a.positions[t];
    if (pos < 0 || pos >= a.max_positions) return;
    const bool turns = o < nrot;
    if (!turns && a.in_place) return;
    const OctetDims d = octet_dims(o, rd, il);
    const In* qin = static_cast<const In*>(a.query) + t * a.q_st + h0 * a.q_sh;
    Out* qout = static_cast<Out*>(a.query_out) + t * a.o_st + h0 * a.o_sh;
    float4_t c = (float4_t)1.f, s = (float4_t)0.f;
    if (turns) {
        const float* cs = a.cos_sin + pos * a.cs_st + 4 * o;
        c = *reinterpret_cast<const float4_t*>(cs);
        s = *reinterpret_cast<const float4_t*>(cs + half);
    }
    float4_t x[kHeads], y[kHeads];
#pragma unroll
    for (int i = 0; i < kHeads; ++i) {
        const int64_t at = min(i, a.Hq - 1 - h0) * a.q_sh;  // (a head past the last: the last again, not stored)
        x[i] = load4(qin + at + d.a);
        y[i] = load4(qin + at + d.b);
    }
#pragma unroll
    for (int i = 0; i < kHeads; ++i) {
        if (h0 + i >= a.Hq) break;
        if (turns) rotate_octet(x[i], y[i], c, s, il);
        store_out4(qout + i * a.o_sh + d.a, x[i]);
        store_out4(qout + i * a.o_sh + d.b, y[i]);
    }
}

// ---------------------------------------------------------------------------------------
// host side

// A launch has fewer than 2^32 threads, 2^24 workgroups: longer batches go a run of tokens at a time.
template <class In, class Out, int kLanes>
static void launch_groups(RotaryWriteParams p, hipStream_t stream) {
    const int64_t tokens = p.T, groups = (p.Hq + kHeads - 1) / kHeads;
    const int64_t most = (((int64_t)1 << 24) - 2) * 256 / (32 * (int64_t)p.Hkv + kLanes * groups);
    const RotaryWriteParams all = p;
    for (int64_t t = 0; t < tokens; t += most) {
        p.T = (int)(tokens - t < most ? tokens - t : most);
        p.query = static_cast<const In*>(all.query) + t * p.q_st;
        p.query_out = static_cast<Out*>(all.query_out) + t * p.o_st;
        p.key = static_cast<const In*>(all.key) + t * p.k_st;
        p.value = static_cast<const In*>(all.value) + t * p.v_st;
        p.positions = all.positions + t;
        p.slots = all.slots + t;
        const int64_t kv = ((int64_t)p.T * p.Hkv + 7) / 8, q = (p.T * groups + 256 / kLanes - 1) / (256 / kLanes);
        p.kv_groups = (int)kv;
        hipLaunchKernelGGL((pd_rotary_write_kernel<In, Out, kLanes>), dim3((unsigned)(kv + q)), dim3(256), 0, stream, p);
    }
}

template <class In, class Out>
static void launch_lanes(const RotaryWriteParams& p, hipStream_t stream) {
    // lanes of a query head: one for each octet it touches
    const int octets = p.in_place ? p.rotary_dim / 8 : 32;
    if (octets <= 8)
        launch_groups<In, Out, 8>(p, stream);
    else if (octets <= 16)
        launch_groups<In, Out, 16>(p, stream);
    else
        launch_groups<In, Out, 32>(p, stream);
}

hipError_t launch_rotary_write(const RotaryWriteParams& p, int dtype, int out_dtype, hipStream_t stream) {
    if (dtype == PD_DTYPE_FP16)
        launch_lanes<_Float16, _Float16>(p, stream);
    else if (dtype == PD_DTYPE_BF16 && out_dtype == PD_DTYPE_BF16)
        launch_lanes<__bf16, __bf16>(p, stream);
    else if (dtype == PD_DTYPE_BF16)
        launch_groups<__bf16, _Float16, 32>(p, stream);
    else if (out_dtype == PD_DTYPE_FP32)
        launch_lanes<float, float>(p, stream);
    else
        launch_groups<float, _Float16, 32>(p, stream);
    return hipGetLastError();
}

}  // namespace pd
