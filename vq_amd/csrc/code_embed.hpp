// Tables of vectors that codes name: sums of their rows, and the gradient of the table.
//
// This translation unit must be compiled with -ffp-contract=off.
#pragma once
#include "code_rules.hpp"
#include "logprobs.hpp"

namespace vq {

// V values of a row from `s` on, as floats; `left` of them are the row's, the others 0.
template <typename T, int V> struct Values {
    typedef typename T::Raw Raw;
    struct __attribute__((packed, aligned(sizeof(Raw)))) Piece {
        Raw v[V];
    };
    static __device__ __forceinline__ Piece fetch(const Raw *s, int left) {
        Piece p;
        if (left >= V) {
            p = *reinterpret_cast<const Piece *>(s);
        } else {
#pragma unroll
            for (int v = 0; v < V; ++v) p.v[v] = v < left ? s[v] : (Raw)0;
        }
        return p;
    }
    static __device__ __forceinline__ void store(Raw *to, const float (&x)[V], int left) {
        Piece p;
#pragma unroll
        for (int v = 0; v < V; ++v) p.v[v] = T::down(x[v]);
        if (left >= V) {
            *reinterpret_cast<Piece *>(to) = p;
        } else {
#pragma unroll
            for (int v = 0; v < V; ++v)
                if (v < left) to[v] = p.v[v];
        }
    }
};

struct EmbedArgs {
    const void *table;
    int64_t ld;
    int k, dim, m;
    const void *codes;
    int code_bytes;
    int64_t n, code_stride;
    float scale;
    void *out;
    int64_t ld_out;
};

// out[i] = scale * sum over the stages s, in their order, of table[s * k + code]: 1 << shift lanes of a row, 16 bytes of the table each,
// rows side by side in a workgroup, a row's further pieces by blockIdx.y.
template <typename T, typename O>
__global__ void __launch_bounds__(256) k_code_embed(EmbedArgs a, int shift) {
    typedef typename T::Raw Raw;
    constexpr int V = 16 / (int)sizeof(Raw), AHEAD = 4;
    typedef Values<T, V> In;
    const int64_t row = (int64_t)blockIdx.x * (256 >> shift) + (threadIdx.x >> shift);
    const int at = ((blockIdx.y << shift) + (threadIdx.x & ((1 << shift) - 1))) * V, left = a.dim - at;
    if (row >= a.n || left <= 0) return;
    const Raw *table = (const Raw *)a.table + at;
    float sum[V];
#pragma unroll
    for (int v = 0; v < V; ++v) sum[v] = 0.0f;
    bool bad = false;
    for (int s = 0; s < a.m; s += AHEAD) {
        typename In::Piece p[AHEAD];
        bool has[AHEAD];
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {
            const int64_t code = s + j < a.m ? code_at(a.codes, a.code_bytes, row * a.code_stride + s + j) : -1;
            bad |= code >= a.k;
            has[j] = code >= 0 && code < a.k;
            if (has[j]) p[j] = In::fetch(table + ((int64_t)(s + j) * a.k + code) * a.ld, left);
        }
#pragma unroll
        for (int j = 0; j < AHEAD; ++j)
            if (has[j]) {
#pragma unroll
                for (int v = 0; v < V; ++v) sum[v] += T::up(p[j].v[v]);
            }
    }
#pragma unroll
    for (int v = 0; v < V; ++v) sum[v] = bad ? __builtin_nanf("") : a.scale * sum[v];
    Values<O, V>::store((typename O::Raw *)a.out + row * a.ld_out + at, sum, left);
}

// ---- the positions by code ---------------------------------------------------------------------------
struct ListArgs {
    const void *codes;
    int code_bytes;
    int64_t code_stride;
    int n, k, width;  // codes of a bucket
    int32_t *start, *rows, *row_codes;
};

// A workgroup lists the positions of its bucket of codes, blockIdx.x, in stage blockIdx.y: every workgroup reads all codes of the stage, counts those
// below its bucket, whose number is where its list begins, and those in it, by wave and code; each wave has a run of the positions, so that
// the order within a code is that of the positions.
template <int WAVES>
__global__ void __launch_bounds__(64 * WAVES) k_code_lists(ListArgs a) {
    __shared__ int hist[WAVES][kBucketMost];
    __shared__ int below_of[WAVES], total_of[WAVES];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), stage = blockIdx.y;
    const int lo = blockIdx.x * a.width, width = min(a.width, a.k - lo);
    const int share = (a.n + 64 * WAVES - 1) / (64 * WAVES) * 64, from = min(a.n, wave * share), to = min(a.n, from + share);
    for (int i = tid; i < WAVES * kBucketMost; i += 64 * WAVES) hist[i / kBucketMost][i % kBucketMost] = 0;
    __syncthreads();
    constexpr int AHEAD = 8;
    const auto code_of = [&](int i) { return i < to ? (uint32_t)code_at(a.codes, a.code_bytes, (int64_t)i * a.code_stride + stage) : 0xffffffffu; };
    int below = 0;
    for (int i = from + lane; i - lane < to; i += 64 * AHEAD) {
        uint32_t c[AHEAD];
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) c[j] = code_of(i + 64 * j);
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {
            below += c[j] < (uint32_t)lo;
            if (c[j] - (uint32_t)lo < (uint32_t)width) atomicAdd(&hist[wave][c[j] - lo], 1);
        }
    }
    below = (int)over_group<64>((uint32_t)below, 0u, [](uint32_t x, uint32_t y) { return x + y; });
    if (lane == 0) below_of[wave] = below;
    __syncthreads();
    int base = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) base += below_of[w];
    // where each code's list begins, and in it each wave's share; a lane per code
    int mine = 0;
    if (tid < width) {
#pragma unroll
        for (int w = 0; w < WAVES; ++w) mine += hist[w][tid];
    }
    int before = mine;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(before, d);
        if (lane >= d) before += o;
    }
    if (lane == 63) total_of[wave] = before;
    __syncthreads();
    int at = base + before - mine;
    for (int w = 0; w < wave; ++w) at += total_of[w];
    int32_t *start = a.start + (int64_t)stage * (a.k + 1);
    if (tid < width) {
        start[lo + tid] = at;
        if (lo + tid == a.k - 1) start[a.k] = at + mine;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            const int here = hist[w][tid];
            hist[w][tid] = at;
            at += here;
        }
    }
    __syncthreads();
    int32_t *rows = a.rows + (int64_t)stage * a.n, *row_codes = a.row_codes + (int64_t)stage * a.n;
    for (int i = from + lane; i - lane < to; i += 64 * AHEAD) {
        uint32_t c[AHEAD];
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) c[j] = code_of(i + 64 * j) - (uint32_t)lo;
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {
            unsigned long long left = __ballot(c[j] < (uint32_t)width);
            while (left) {  // uniform: the codes among these 64 positions, one after another
                const uint32_t code = (uint32_t)__builtin_amdgcn_readlane((int)c[j], __ffsll(left) - 1);
                const unsigned long long same = __ballot(c[j] == code);
                const int first = hist[wave][code];
                wave_sync();
                if (c[j] == code) {
                    const int place = first + __popcll(same & ((1ull << lane) - 1));
                    rows[place] = i + 64 * j;
                    row_codes[place] = lo + (int)code;
                }
                if (lane == 0) hist[wave][code] = first + __popcll(same);
                wave_sync();
                left &= ~same;
            }
        }
    }
}

// ---- the sums ------------------------------------------------------------------------------------------
struct SumArgs {
    const void *g;
    int64_t ld;
    int n, dim, k;
    float scale;
    int accumulate;
    void *grad;
    int64_t ld_grad;
    const int32_t *start, *rows, *row_codes;
    float *partial;  // [stage][chunk][2][padded dim]
    int chunks, padded, keys, groups;  // codes of 16 lanes one after another; workgroups of codes
};

constexpr int kOwnMembers = 32;  // a code of more positions is summed by the whole workgroup

// V columns of the members number a, a + step, ... below b of a list, summed in that order.
template <typename T, int V>
__device__ __forceinline__ void sum_members(const SumArgs &s, const int32_t *rows, int a, int b, int step, int at, int left, float (&sum)[V]) {
    typedef typename T::Raw Raw;
    typedef Values<T, V> In;
    constexpr int AHEAD = 8;
#pragma unroll
    for (int v = 0; v < V; ++v) sum[v] = 0.0f;
    const Raw *g = (const Raw *)s.g + at;
    for (int p = a; p < b; p += AHEAD * step) {
        typename In::Piece x[AHEAD];
#pragma unroll
        for (int j = 0; j < AHEAD; ++j)
            if (p + j * step < b) x[j] = In::fetch(g + (int64_t)rows[p + j * step] * s.ld, left);
#pragma unroll
        for (int j = 0; j < AHEAD; ++j)
            if (p + j * step < b) {
#pragma unroll
                for (int v = 0; v < V; ++v) sum[v] += T::up(x[j].v[v]);
            }
    }
}

// Rows of the gradient: 16 lanes sum V columns each of a code's members.  The first a.groups workgroups take codes, those behind them the
// chunks of the list that belong to codes of more than kLongCode members.  blockIdx.y: pieces of 16 * V columns, blockIdx.z: stages.
template <typename T, typename O>
__global__ void __launch_bounds__(256) k_embed_sums(SumArgs a) {
    typedef typename T::Raw Raw;
    typedef typename O::Raw Out;
    constexpr int V = 16 / (int)sizeof(Raw), COLUMNS = 16 * V;
    __shared__ float red[16][COLUMNS];
    __shared__ int longer[16 * 8], count;
    const int tid = threadIdx.x, sub = tid >> 4, column = blockIdx.y * COLUMNS, at = column + (tid & 15) * V, left = a.dim - at, stage = blockIdx.z;
    const int32_t *start = a.start + (int64_t)stage * (a.k + 1), *rows = a.rows + (int64_t)stage * a.n;
    Out *grad = (Out *)a.grad + (int64_t)stage * a.k * a.ld_grad;
    float sum[V];
    // all 16 groups of lanes sum members [from, to); the sums of COLUMNS columns are in the first lanes then
    const auto together = [&](int from, int to) {
        if (left > 0) {
            sum_members<T, V>(a, rows, from + sub, to, 16, at, left, sum);
#pragma unroll
            for (int v = 0; v < V; ++v) red[sub][(tid & 15) * V + v] = sum[v];
        }
        __syncthreads();
        float total = 0.0f;
        if (tid < COLUMNS && column + tid < a.dim) {
#pragma unroll
            for (int j = 0; j < 16; ++j) total += red[j][tid];
        }
        __syncthreads();
        return total;
    };
    if ((int)blockIdx.x >= a.groups) {
        const int chunk = blockIdx.x - a.groups, all = start[a.k], first = chunk * kLongCode, last = min(all, first + kLongCode) - 1;
        if (first > last) return;
        const int32_t *row_codes = a.row_codes + (int64_t)stage * a.n;
        const int c0 = row_codes[first], c1 = row_codes[last];
        for (int slot = 0; slot < 2; ++slot) {
            const int c = slot ? c1 : c0;
            if (slot && c1 == c0) break;
            const int s0 = start[c], s1 = start[c + 1];
            if (s1 - s0 <= kLongCode) continue;
            const float total = together(max(s0, first), min(s1, last + 1));
            if (tid < COLUMNS && column + tid < a.dim) a.partial[(((int64_t)stage * a.chunks + chunk) * 2 + slot) * a.padded + column + tid] = total;
        }
        return;
    }
    if (tid == 0) count = 0;
    __syncthreads();
    for (int q = 0; q < a.keys; ++q) {
        const int64_t code = (int64_t)blockIdx.x * 16 * a.keys + q * 16 + sub;
        if (code >= a.k) continue;
        const int s0 = start[code], s1 = start[code + 1];
        if (s1 - s0 > kOwnMembers) {
            if ((tid & 15) == 0 && s1 - s0 <= kLongCode) longer[atomicAdd(&count, 1)] = (int)code;
            continue;
        }
        if (left <= 0 || (a.accumulate && s0 == s1)) continue;
        sum_members<T, V>(a, rows, s0, s1, 1, at, left, sum);
        Out *to = grad + code * a.ld_grad + at;
        if (a.accumulate) {
            const typename Values<O, V>::Piece old = Values<O, V>::fetch(to, left);
#pragma unroll
            for (int v = 0; v < V; ++v) sum[v] = __builtin_fmaf(a.scale, sum[v], O::up(old.v[v]));
        } else {
#pragma unroll
            for (int v = 0; v < V; ++v) sum[v] *= a.scale;
        }
        Values<O, V>::store(to, sum, left);
    }
    __syncthreads();
    const int n_longer = count;
    for (int i = 0; i < n_longer; ++i) {
        const int code = longer[i];
        const float total = together(start[code], start[code + 1]);
        if (tid < COLUMNS && column + tid < a.dim) {
            Out *to = grad + (int64_t)code * a.ld_grad + column + tid;
            *to = O::down(a.accumulate ? __builtin_fmaf(a.scale, total, O::up(*to)) : a.scale * total);
        }
    }
}

// The sums of the chunks of a code of more than kLongCode members, by the workgroup of the chunk in which the code's list begins:
// 64 columns (blockIdx.y), 16 groups of 16 lanes that share the chunks.
template <typename O>
__global__ void __launch_bounds__(256) k_embed_join(SumArgs a) {
    typedef typename O::Raw Out;
    __shared__ float red[16][64];
    const int tid = threadIdx.x, sub = tid >> 4, column = blockIdx.y * 64, at = column + (tid & 15) * 4, stage = blockIdx.z, chunk = blockIdx.x;
    const int32_t *start = a.start + (int64_t)stage * (a.k + 1), *row_codes = a.row_codes + (int64_t)stage * a.n;
    const int all = start[a.k], first = chunk * kLongCode, last = min(all, first + kLongCode) - 1;
    if (first > last) return;
    const int code = row_codes[last], s0 = start[code], s1 = start[code + 1];
    if (s1 - s0 <= kLongCode || s0 < first) return;
    const int end = (s1 - 1) / kLongCode;  // the last chunk with members of this code
    const float *partial = a.partial + (int64_t)stage * a.chunks * 2 * a.padded;
    float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (at < a.dim) {
        for (int c = chunk + sub; c <= end; c += 16) {
            const int slot = c == chunk && row_codes[first] != code ? 1 : 0;
            const float4 x = *reinterpret_cast<const float4 *>(partial + ((int64_t)c * 2 + slot) * a.padded + at);
            sum[0] += x.x, sum[1] += x.y, sum[2] += x.z, sum[3] += x.w;
        }
    }
#pragma unroll
    for (int v = 0; v < 4; ++v) red[sub][(tid & 15) * 4 + v] = sum[v];
    __syncthreads();
    if (tid >= 64 || column + tid >= a.dim) return;
    float total = 0.0f;
#pragma unroll
    for (int j = 0; j < 16; ++j) total += red[j][tid];
    Out *to = (Out *)a.grad + ((int64_t)stage * a.k + code) * a.ld_grad + column + tid;
    *to = O::down(a.accumulate ? __builtin_fmaf(a.scale, total, O::up(*to)) : a.scale * total);
}

}  // namespace vq
