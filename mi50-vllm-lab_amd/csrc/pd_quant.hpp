// What the cache writers share (pd_cache_write.hip, pd_rotary_write.hip): the loads of four values, a row's
// largest magnitude and the int8 rounding. scale = absmax / 127 (0 for an all-zero row), q = clamp(rint(x / scale),
// -127, 127) with x / scale correctly rounded: both writers store the same bytes for the same fp32 values.
#pragma once

#include <type_traits>

#include "pd_tile.hpp"

namespace pd {

template <class In>
__device__ __forceinline__ float4_t load4(const In* p) {
    if constexpr (sizeof(In) == 4) {
        return *reinterpret_cast<const float4_t*>(p);
    } else {
        typedef In in4_t __attribute__((ext_vector_type(4)));
        const in4_t v = *reinterpret_cast<const in4_t*>(p);
        return float4_t{(float)v.x, (float)v.y, (float)v.z, (float)v.w};
    }
}

__device__ __forceinline__ unsigned quant4(float4_t x, float scale) {
    if (scale == 0.f) return 0u;
    auto q = [&](float v) -> unsigned {
        const float r = fminf(fmaxf(__builtin_rintf(v / scale), -127.f), 127.f);
        return (unsigned)((int)r & 0xff);
    };
    return q(x.x) | (q(x.y) << 8) | (q(x.z) << 16) | (q(x.w) << 24);
}

// quant4 through y = x * inv, inv = 1 / scale rounded once per row: y is within 2^-15 of the
// correctly rounded x / scale (|x / scale| <= 127, so both carry relative errors below 2^-23),
// hence rint(y) is the same integer unless y lies within 2^-14 of a half-integer. Those values,
// and rows whose inverse is not finite, take the division itself, so the bytes are exactly
// quant4's.
__device__ __forceinline__ unsigned quant4_inv(float4_t x, float scale, float inv) {
    if (scale == 0.f) return 0u;
    const float y[4] = {x.x * inv, x.y * inv, x.z * inv, x.w * inv};
    bool near = !__builtin_isfinite(inv);
#pragma unroll
    for (int e = 0; e < 4; ++e) near = near || fabsf(y[e] - __builtin_floorf(y[e]) - 0.5f) < 0x1p-14f;
    if (near) return quant4(x, scale);
    unsigned r = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e)
        r |= ((unsigned)((int)fminf(fmaxf(__builtin_rintf(y[e]), -127.f), 127.f) & 0xff)) << (8 * e);
    return r;
}

// Max over the 16 lanes of a DPP row, in every lane of the row (rotations by 8, 4, 2, 1).
__device__ __forceinline__ float row16_max(float v) {
    auto ror = [](float x, auto ctrl) {
        return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x),
                                                                     decltype(ctrl)::value, 0xf, 0xf, false));
    };
    v = fmaxf(v, ror(v, std::integral_constant<int, 0x128>{}));  // row_ror:8
    v = fmaxf(v, ror(v, std::integral_constant<int, 0x124>{}));  // row_ror:4
    v = fmaxf(v, ror(v, std::integral_constant<int, 0x122>{}));  // row_ror:2
    return fmaxf(v, ror(v, std::integral_constant<int, 0x121>{}));  // row_ror:1
}

__device__ __forceinline__ float absmax4(float4_t x) {
    return fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w)));
}

}  // namespace pd
