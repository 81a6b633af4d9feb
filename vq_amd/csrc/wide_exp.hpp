// Exponentials and sums in 64 bits.
#pragma once
#include "logprobs.hpp"

namespace vq {

constexpr double kLog2e64 = 1.4426950408889634074;

// 2^(y * c), off by less than 1.2e-12 of it, for y * c between -1001 and 1000: the power of the nearest whole number, which the sum with
// 1.5 * 2^52 leaves in its lowest bits, times a polynomial in the rest (the one of degree 8 that meets 2^f at the nine Chebyshev nodes of
// [-1/2, 1/2]).  Nothing but additions, fused operations and one on whole numbers: conversions and roundings take four times as long.
__device__ __forceinline__ double exp2_of(double y, double c) {
    constexpr double MAGIC = 6755399441055744.0;
    const double t = __builtin_fma(y, c, MAGIC), f = __builtin_fma(y, c, MAGIC - t);
    double p = 1.32552248786688170e-6;
    p = __builtin_fma(p, f, 1.53100794022492974e-5);
    p = __builtin_fma(p, f, 1.54034558524538394e-4);
    p = __builtin_fma(p, f, 1.33334505680006457e-3);
    p = __builtin_fma(p, f, 9.61812915940255819e-3);
    p = __builtin_fma(p, f, 5.55041094120593299e-2);
    p = __builtin_fma(p, f, 2.40226506958129882e-1);
    p = __builtin_fma(p, f, 6.93147180545933455e-1);
    p = __builtin_fma(p, f, 1.0);
    typedef uint32_t Halves __attribute__((ext_vector_type(2)));  // (one instruction; in whole numbers of 64 bits it takes five)
    Halves bits = __builtin_bit_cast(Halves, p);
    bits.y += __builtin_bit_cast(Halves, t).x << 20;
    return __builtin_bit_cast(double, bits);
}
// 2^d, from d = 1000 on 2^1000 (more than binary32 holds: from 1024 on the whole part would run over into the sign), 0 below -1000; no NaN.
__device__ __forceinline__ double exp2_wide(double d) {
    const double e = exp2_of(fmin(fmax(d, -1000.0), 1000.0), 1.0);
    return d < -1000.0 ? 0.0 : e;
}

template <int CTRL, int ROWS, bool ALL> __device__ __forceinline__ double dpp_double(double v) {  // (0 where nothing comes)
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    uint32_t lo, hi;
    if constexpr (ALL)
        lo = dpp_all<CTRL>((uint32_t)b), hi = dpp_all<CTRL>((uint32_t)(b >> 32));
    else
        lo = dpp_keep<CTRL, ROWS>(0u, (uint32_t)b), hi = dpp_keep<CTRL, ROWS>(0u, (uint32_t)(b >> 32));
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
// Sum over a wave, for every lane, in an order that is the same in every run.
__device__ __forceinline__ double wave_sum(double v) {
    v += dpp_double<0xB1, 0xf, true>(v);
    v += dpp_double<0x4E, 0xf, true>(v);
    v += dpp_double<0x141, 0xf, true>(v);
    v += dpp_double<0x140, 0xf, true>(v);
    v += dpp_double<0x142, 0xa, false>(v);  // a row's last lane to the next row
    v += dpp_double<0x143, 0xc, false>(v);  // the lower half's to the upper half
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    return __builtin_bit_cast(double, (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(b >> 32), 63) << 32 |
                                          (uint32_t)__builtin_amdgcn_readlane((int)b, 63));
}
// Sum of the lanes up to this one.
__device__ __forceinline__ double wave_scan(double v, int lane) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const double o = __shfl_up(v, d);
        if (lane >= d) v += o;
    }
    return v;
}

}  // namespace vq
