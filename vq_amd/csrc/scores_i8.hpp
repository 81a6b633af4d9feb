// Rows to 8-bit integers with a scale each, and scores of 8-bit rows against 8-bit codes on the matrix cores.
//
// This translation unit must be compiled with -ffp-contract=off.
#pragma once
#include "logprobs.hpp"

namespace vq {

typedef int32_t i32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

// x / scale to the nearest integer, ties to even, from the exact quotient: the rounded product with the reciprocal is
// at most one off, and the distance r = x - q * scale to it is exact in f32 (a multiple of the last bit of
// `scale`, or of x where that is finer and q <= 1, of less than 2^24 of them).
__device__ __forceinline__ int nearest_i8(float x, float scale, float inv) {
    float q = __builtin_rintf(x * inv);
    const float r = __builtin_fmaf(-q, scale, x), half = 0.5f * scale;
    const bool odd = ((int)q & 1) != 0;
    if (r > half || (r == half && odd)) q += 1.0f;
    if (r < -half || (r == -half && odd)) q -= 1.0f;
    return (int)fminf(fmaxf(q, -127.0f), 127.0f);
}

struct RowsI8Args {
    const void *x;
    int64_t n, ld;
    int dim;
    int8_t *q;
    int64_t ld_q;
    float *scale;
};

// A wave per row.
template <typename T>
__global__ void __launch_bounds__(256) k_rows_i8(RowsI8Args a) {
    const int lane = threadIdx.x & 63;
    for (int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); row < a.n; row += (int64_t)gridDim.x * 4) {
        const typename T::Raw *x = (const typename T::Raw *)a.x + row * a.ld;
        uint32_t m = 0;  // magnitudes as integers: an infinity is above every number and a NaN above it
        for (int t = lane; t < a.dim; t += 64) m = max(m, __float_as_uint(T::up(x[t])) & 0x7fffffffu);
        for (int o = 32; o; o >>= 1) m = max(m, (uint32_t)__shfl_xor((int)m, o));
        const bool bad = m >= 0x7f800000u;
        const float scale = bad ? __builtin_nanf("") : __uint_as_float(m) / 127.0f;
        // small scales: both sides of the quotient times 2^60, exactly, so that the reciprocal is finite
        const float up = scale < 0x1p-100f ? 0x1p60f : 1.0f, sc = scale * up, inv = 1.0f / sc;
        for (int t = lane; t < a.dim; t += 64)
            a.q[row * a.ld_q + t] = (int8_t)(scale > 0.0f ? nearest_i8(T::up(x[t]) * up, sc, inv) : 0);
        if (lane == 0) a.scale[row] = scale;
    }
}

struct ScoresArgs {
    const int8_t *x;
    const float *xs;
    int64_t n, ld_x;
    const int8_t *w;
    const float *ws;
    int k;
    int64_t ld_w;
    int dim;
    const float *bias;
    void *out;
    int64_t ld_out;
};

// 16 bytes of a row from component t on, zeros beyond the row; any alignment.
__device__ __forceinline__ i32x4 piece16(const int8_t *row, int t, int dim) {
    if (t + 16 <= dim && (((uintptr_t)(row + t)) & 15) == 0) return *reinterpret_cast<const i32x4 *>(row + t);
    union {
        i32x4 v;
        int8_t b[16];
    } u;
    u.v = i32x4{0, 0, 0, 0};
    for (int i = 0; i < 16; ++i)
        if (t + i < dim) u.b[i] = row[t + i];
    return u.v;
}

// 64 rows x 64 codes per workgroup, operands staged through LDS in steps of 64 components, for any stride and
// alignment.  A wave makes 16 codes x 64 rows: the codes are the first operand, so that a lane ends with four consecutive codes of a row.
template <typename OutT>
__global__ void __launch_bounds__(256) k_scores_any(ScoresArgs a) {
    __shared__ i32x4 lx[64][5], lw[64][5];  // (rows of 80 bytes: no more than two lanes of a read meet in a bank)
    const int64_t row0 = (int64_t)blockIdx.y * 64;
    const int code0 = blockIdx.x * 64, tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    i32x4 acc[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) acc[u] = i32x4{0, 0, 0, 0};
    const int r = tid >> 2, c = tid & 3;
    const int64_t xr = min(row0 + r, a.n - 1);
    const int wr = min(code0 + r, a.k - 1);
    for (int t = 0; t < a.dim; t += 64) {
        const i32x4 px = piece16(a.x + xr * a.ld_x, t + c * 16, a.dim), pw = piece16(a.w + wr * a.ld_w, t + c * 16, a.dim);
        __syncthreads();
        lx[r][c] = px;
        lw[r][c] = pw;
        __syncthreads();
        const i32x4 fw = lw[wave * 16 + (lane & 15)][lane >> 4];
#pragma unroll
        for (int u = 0; u < 4; ++u)
            acc[u] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fw, lx[u * 16 + (lane & 15)][lane >> 4], acc[u], 0, 0, 0);
    }
    typedef typename OutT::Raw Raw;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        const int64_t row = row0 + u * 16 + (lane & 15);
        const int code = code0 + wave * 16 + (lane >> 4) * 4;
        if (row >= a.n) continue;
        const float xs = a.xs[row];
        for (int i = 0; i < 4; ++i)
            if (code + i < a.k) {
                const float y = (float)acc[u][i] * xs * a.ws[code + i];
                ((Raw *)a.out)[row * a.ld_out + code + i] = OutT::down(a.bias ? y + a.bias[code + i] : y);
            }
    }
}

}  // namespace vq
