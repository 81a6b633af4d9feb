// Exponentials and sums in 64 bits.
#pragma once
#include <hip/hip_runtime.h>

namespace vq {

constexpr double kLog2e64 = 1.4426950408889634074;

// 2^d, off by less than 3e-13 of it: the power of the nearest whole number times the series of 2^f = e^(f ln 2), |f| <= 1/2, up to its tenth
// power (the eleventh's term is 2.2e-13).  d is a number, below 1000; beneath -2000 the result is 0.
__device__ __forceinline__ double exp2_wide(double d) {
    const double whole = __builtin_rint(d), f = d - whole;
    double p = 7.0549116208011233e-9;  // ln(2)^n / n!, n = 10 ... 0
    p = __builtin_fma(p, f, 1.0178086009239700e-7);
    p = __builtin_fma(p, f, 1.3215486790144310e-6);
    p = __builtin_fma(p, f, 1.5252733804059840e-5);
    p = __builtin_fma(p, f, 1.5403530393381610e-4);
    p = __builtin_fma(p, f, 1.3333558146428443e-3);
    p = __builtin_fma(p, f, 9.6181291076284772e-3);
    p = __builtin_fma(p, f, 5.5504108664821580e-2);
    p = __builtin_fma(p, f, 2.4022650695910071e-1);
    p = __builtin_fma(p, f, 6.9314718055994531e-1);
    p = __builtin_fma(p, f, 1.0);
    return __builtin_ldexp(p, (int)whole);
}

// Sum over a wave, for every lane, in an order that is the same in every run.
__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) v += __shfl_xor(v, d);
    return v;
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
