// Log probabilities of codes, entropy and alternatives from rows of scores, and the gradient.
//
// This translation unit must be compiled with -ffp-contract=off.
#pragma once
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace vq {

constexpr float kNegInf = -__builtin_inff();
constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.693147180559945309417f;

struct F32 {
    typedef float Raw;
    static __device__ __forceinline__ float up(Raw v) { return v; }
    static __device__ __forceinline__ Raw down(float v) { return v; }
};
struct F16 {
    typedef uint16_t Raw;
    static __device__ __forceinline__ float up(Raw v) { return __half2float(__ushort_as_half(v)); }
    static __device__ __forceinline__ Raw down(float v) { return __half_as_ushort(__float2half_rn(v)); }
};
struct BF16 {
    typedef uint16_t Raw;
    static __device__ __forceinline__ float up(Raw v) { return __uint_as_float((uint32_t)v << 16); }
    static __device__ __forceinline__ Raw down(float v) { return __builtin_bit_cast(uint16_t, (__bf16)v); }
};

struct LogprobArgs {
    const void *s;
    int64_t n, ld;
    int k;
    float beta;
    const void *codes;
    int64_t code_stride;
    int code_bytes, top;
    float *logprob, *max, *logsum, *entropy, *top_logprob;
    int32_t *top_code;
};

__device__ __forceinline__ int64_t code_at(const void *codes, int bytes, int64_t at) {
    return bytes == 1 ? (int64_t)((const uint8_t *)codes)[at]
                      : bytes == 2 ? (int64_t)((const uint16_t *)codes)[at] : (int64_t)((const int32_t *)codes)[at];
}

// Order of the alternatives as an unsigned number: the larger score, of equal ones the lower code.  (-0 counts as 0.)
__device__ __forceinline__ uint64_t rank_key(float v, uint32_t code) {
    const uint32_t u = __float_as_uint(v + 0.0f);
    return (uint64_t)(u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u)) << 32 | (uint32_t)~code;
}
__device__ __forceinline__ float key_score(uint64_t key) {
    const uint32_t u = (uint32_t)(key >> 32);
    return __uint_as_float(u & 0x80000000u ? u ^ 0x80000000u : ~u);
}
__device__ __forceinline__ int32_t key_code(uint64_t key) { return (int32_t)~(uint32_t)key; }

// What a row's thread writes: x_c is the score of its code.
template <typename T>
__device__ __forceinline__ void write_row(const LogprobArgs &a, int64_t row, float m, float S, float W) {
    const bool none = m == kNegInf;
    const float L = logf(S);
    if (a.max) a.max[row] = m;
    if (a.logsum) a.logsum[row] = L;
    if (a.entropy) a.entropy[row] = none ? 0.0f : L - W / S;
    if (a.logprob) {
        const int64_t c = code_at(a.codes, a.code_bytes, row * a.code_stride);
        float lp = 0.0f;
        if (c >= a.k)
            lp = __builtin_nanf("");
        else if (c >= 0)
            lp = none ? kNegInf : a.beta * (T::up(((const typename T::Raw *)a.s)[row * a.ld + c]) - m) - L;
        a.logprob[row] = lp;
    }
}
__device__ __forceinline__ void write_alternative(const LogprobArgs &a, int64_t row, int t, uint64_t key, float m, float L) {
    const float v = key_score(key);
    const bool bad = L != L, none = key == 0 || v == kNegInf;
    a.top_logprob[row * a.top + t] = bad ? __builtin_nanf("") : none ? kNegInf : a.beta * (v - m) - L;
    a.top_code[row * a.top + t] = bad || none ? -1 : key_code(key);
}

// A workgroup per row: the largest score, the sums relative to it, then one round per alternative.
template <typename T>
__global__ void __launch_bounds__(256) k_logprobs_rows(LogprobArgs a) {
    __shared__ float part[3][4];
    __shared__ uint64_t best[4];
    const int tid = threadIdx.x, wave = tid >> 6;
    for (int64_t row = blockIdx.x; row < a.n; row += gridDim.x) {
    const typename T::Raw *s = (const typename T::Raw *)a.s + row * a.ld;
    float m = kNegInf;
    for (int j = tid; j < a.k; j += 256) m = __builtin_elementwise_maximum(m, T::up(s[j]));
    for (int o = 32; o; o >>= 1) m = __builtin_elementwise_maximum(m, __shfl_xor(m, o));
    if ((tid & 63) == 0) part[0][wave] = m;
    __syncthreads();
    m = __builtin_elementwise_maximum(__builtin_elementwise_maximum(part[0][0], part[0][1]),
                                      __builtin_elementwise_maximum(part[0][2], part[0][3]));
    const float ms = m == kNegInf ? 0.0f : m;
    float S = 0.0f, W = 0.0f;
    for (int j = tid; j < a.k; j += 256) {
        const float d = a.beta * (T::up(s[j]) - ms), e = expf(d);
        S += e;
        W += e == 0.0f ? 0.0f : e * d;
    }
    for (int o = 32; o; o >>= 1) S += __shfl_xor(S, o), W += __shfl_xor(W, o);
    if ((tid & 63) == 0) part[1][wave] = S, part[2][wave] = W;
    __syncthreads();
    S = part[1][0] + part[1][1] + part[1][2] + part[1][3];
    W = part[2][0] + part[2][1] + part[2][2] + part[2][3];
    if (tid == 0) write_row<T>(a, row, m, S, W);
    uint64_t last = ~0ull;
    for (int t = 0; t < a.top; ++t) {
        uint64_t key = 0;
        for (int j = tid; j < a.k; j += 256) {
            const uint64_t c = rank_key(T::up(s[j]), (uint32_t)j);
            key = c < last && c > key ? c : key;
        }
        for (int o = 32; o; o >>= 1) {
            const uint64_t c = __shfl_xor(key, o);
            key = c > key ? c : key;
        }
        if ((tid & 63) == 0) best[wave] = key;
        __syncthreads();
        for (int w = 0; w < 4; ++w) key = best[w] > key ? best[w] : key;
        __syncthreads();
        last = key;
        if (tid == 0) write_alternative(a, row, t, key, m, logf(S));
    }
    }
}

struct GradArgs {
    const void *s;
    int64_t n, ld;
    int k;
    float beta;
    const void *codes;
    int64_t code_stride;
    int code_bytes;
    const float *max, *logsum, *entropy, *g_logprob, *g_entropy;
    void *grad;
    int64_t ld_grad;
};

// The gradient of one score: lp = log p, one: whether this is the row's code.
__device__ __forceinline__ float grad_one(float lp, bool one, float beta, float gl, float gh, float H) {
    const float p = expf(lp), t = p == 0.0f ? 0.0f : p * (gl + gh * (lp + H));
    return beta * ((one ? gl : 0.0f) - t);
}

template <typename T>
__global__ void __launch_bounds__(256) k_logprobs_grad(GradArgs a) {
    for (int64_t row = blockIdx.x; row < a.n; row += gridDim.x) {
    const typename T::Raw *s = (const typename T::Raw *)a.s + row * a.ld;
    typename T::Raw *g = (typename T::Raw *)a.grad + row * a.ld_grad;
    const float m = a.max[row], L = a.logsum[row];
    const bool none = m == kNegInf;
    const float ms = none ? 0.0f : m, gh = a.g_entropy ? a.g_entropy[row] : 0.0f, H = a.g_entropy ? a.entropy[row] : 0.0f;
    float gl = 0.0f;
    int64_t c = -1;
    if (a.g_logprob) {
        c = code_at(a.codes, a.code_bytes, row * a.code_stride);
        gl = c >= a.k ? __builtin_nanf("") : c < 0 ? 0.0f : a.g_logprob[row];
    }
    for (int j = threadIdx.x; j < a.k; j += 256)
        g[j] = T::down(none ? 0.0f : L != L || gl != gl ? __builtin_nanf("")
                                                          : grad_one(a.beta * (T::up(s[j]) - ms) - L, j == c, a.beta, gl, gh, H));
    }
}

}  // namespace vq
