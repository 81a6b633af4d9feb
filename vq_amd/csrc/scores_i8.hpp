// Rows to 8-bit integers with a scale each, and scores of 8-bit rows against 8-bit codes on the matrix cores.
//
// This translation unit must be compiled with -ffp-contract=off.
#pragma once
#include <algorithm>

#include "logprobs.hpp"

namespace vq {

typedef int32_t i32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

// x / scale to the nearest integer, ties to even, from the exact quotient: the rounded product with the reciprocal is
// at most one off, and the distance r = x - q * scale to it is exact in f32 (a multiple of the last bit of
// `scale`, or of x where that is finer and q <= 1, of less than 2^24 of them), so r says which way to go.
__device__ __forceinline__ int nearest_i8(float x, float scale, float inv, float half) {
    const float q = __builtin_rintf(x * inv), r = __builtin_fmaf(-q, scale, x), far = fabsf(r);
    const int i = (int)q, there = i + (r < 0.0f ? -1 : 1);
    return max(-127, min(127, far > half || (far == half && (i & 1)) ? there : i));
}

// The scale of a row from its largest magnitude, given as the bits of a number (an infinity is above every
// number and a NaN above it).
struct RowScale {
    float scale, up, sc, inv, half;
    __device__ __forceinline__ explicit RowScale(uint32_t most) {
        scale = most >= 0x7f800000u ? __builtin_nanf("") : __uint_as_float(most) / 127.0f;
        up = scale < 0x1p-100f ? 0x1p60f : 1.0f;  // small scales: both sides of the quotient times 2^60, exactly, so that the reciprocal is finite
        sc = scale * up;
        inv = 1.0f / sc;
        half = 0.5f * sc;
    }
    __device__ __forceinline__ int of(float x) const { return nearest_i8(x * up, sc, inv, half); }
    __device__ __forceinline__ bool usable() const { return scale > 0.0f; }
};

struct RowsI8Args {
    const void *x;
    int64_t n, ld;
    int dim;
    int8_t *q;
    int64_t ld_q;
    float *scale;
};

__device__ __forceinline__ uint32_t magnitude(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// G lanes per row, which lies in their registers between the search for its largest magnitude and the quotients.  The vectors at
// its end overlap (Share) where its length is no multiple of theirs: what they share, both write alike.
template <typename T, int G, int NV>
__global__ void __launch_bounds__(256) k_rows_i8(RowsI8Args a) {
    typedef Share<T, G, NV> S;
    constexpr int VEC = S::VEC;
    const int lane = threadIdx.x & (G - 1);
    const int64_t mine = (int64_t)blockIdx.x * (256 / G) + threadIdx.x / G, row = min(mine, a.n - 1);
    S r;
    r.fetch_once((const typename T::Raw *)a.x + row * a.ld, 0, a.dim, lane);
    uint32_t m = 0;
#pragma unroll
    for (int u = 0; u < NV; ++u) {
        if (u > 0 && u * G * VEC >= a.dim) break;  // uniform
        S::values(r.raw[u], r.x + u * VEC);
#pragma unroll
        for (int v = 0; v < VEC; ++v) m = max(m, magnitude(r.x[u * VEC + v]));
    }
    const auto most = [](uint32_t p, uint32_t q) { return p > q ? p : q; };
    m = over_group<(G > 64 ? 64 : G)>(m, 0u, most);
    if constexpr (G == 256) {
        __shared__ uint32_t part[4];
        if ((lane & 63) == 0) part[lane >> 6] = m;
        __syncthreads();
        m = most(most(part[0], part[1]), most(part[2], part[3]));
    }
    const RowScale s(m);
    if (mine >= a.n) return;
    if (lane == 0) a.scale[row] = s.scale;
    int8_t *q = a.q + row * a.ld_q;
#pragma unroll
    for (int u = 0; u < NV; ++u) {
        if (u > 0 && u * G * VEC >= a.dim) break;
        struct __attribute__((packed, aligned(1))) Bytes {
            uint32_t w[VEC / 4];
        } o;
#pragma unroll
        for (int w = 0; w < VEC / 4; ++w) {
            o.w[w] = 0;
#pragma unroll
            for (int v = 0; v < 4; ++v) o.w[w] |= ((uint32_t)s.of(r.x[u * VEC + w * 4 + v]) & 0xffu) << (8 * v);
            if (!s.usable()) o.w[w] = 0;
        }
        *reinterpret_cast<Bytes *>(q + S::base(u, lane, 0, a.dim)) = o;
    }
}

// Rows longer than registers hold, or shorter than a vector: a workgroup per row, which is read twice.
template <typename T>
__global__ void __launch_bounds__(256) k_rows_i8_any(RowsI8Args a) {
    __shared__ uint32_t part[4];
    for (int64_t row = blockIdx.x; row < a.n; row += gridDim.x) {
        const typename T::Raw *x = (const typename T::Raw *)a.x + row * a.ld;
        uint32_t m = 0;
        for (int t = threadIdx.x; t < a.dim; t += 256) m = max(m, magnitude(T::up(x[t])));
        const auto most = [](uint32_t p, uint32_t q) { return p > q ? p : q; };
        m = over_group<64>(m, 0u, most);
        if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = m;
        __syncthreads();
        const RowScale s(most(most(part[0], part[1]), most(part[2], part[3])));
        for (int t = threadIdx.x; t < a.dim; t += 256) a.q[row * a.ld_q + t] = (int8_t)(s.usable() ? s.of(T::up(x[t])) : 0);
        if (threadIdx.x == 0) a.scale[row] = s.scale;
        __syncthreads();
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
struct __attribute__((packed, aligned(1))) Bytes16 {
    i32x4 v;
};
__device__ __forceinline__ i32x4 piece16(const int8_t *row, int t, int dim) {
    if (t + 16 <= dim) return reinterpret_cast<const Bytes16 *>(row + t)->v;
    i32x4 v = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 16; ++i)
        if (t + i < dim) v[i >> 2] |= (int32_t)((uint32_t)(uint8_t)row[t + i] << (8 * (i & 3)));
    return v;
}

// Rows to rows of whole 16 bytes, zeros behind their components: a piece per lane.
__global__ void __launch_bounds__(256) k_pack_i8(const int8_t *__restrict__ x, int64_t n, int64_t ld, int dim, int8_t *__restrict__ to) {
    const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x, per_row = (dim + 15) / 16, row = at / per_row;
    if (row < n) reinterpret_cast<i32x4 *>(to)[at] = piece16(x + row * ld, (int)(at - row * per_row) * 16, dim);
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

// ---- tiles ----------------------------------------------------------------------------------------------
typedef int32_t i32x16 __attribute__((ext_vector_type(16)));

// A tile's place: workgroup i runs on XCD i % 8, and every XCD gets a run of consecutive tiles, column by column through panels
// of four tiles of rows, so that what its compute units read at a time comes from its own L2.
struct TilePlace {
    int64_t r;
    int c;
};
__device__ __forceinline__ TilePlace tile_place(uint32_t id, uint32_t row_tiles, uint32_t code_tiles) {
    const uint32_t all = row_tiles * code_tiles, q = all / 8, rest = all % 8, xcd = id % 8;
    const uint32_t at = xcd * q + min(xcd, rest) + id / 8, panel = at / (4 * code_tiles), in = at - panel * 4 * code_tiles;
    const uint32_t high = min(4u, row_tiles - panel * 4);
    return {(int64_t)(panel * 4 + in % high), (int)(in / high)};
}

// 16 bytes per lane from base + offset to LDS, in the order of the lanes; zeros from `bytes` on, which the hardware checks.
// `base`, `bytes` and `to` are the same in every lane.
__device__ __forceinline__ void copy_to_lds(const int8_t *base, int bytes, char *to, int offset) {
#if defined(__HIP_DEVICE_COMPILE__)  // (the host pass does not know the type of a buffer)
    __amdgpu_buffer_rsrc_t from = __builtin_amdgcn_make_buffer_rsrc((void *)base, 0, bytes, 0x00020000);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(from, (__attribute__((address_space(3))) void *)to, 16, offset, 0, 0, 0);
#endif
}

// Everyone's copies into LDS but for each wave's last LEFT are there, and what everyone read from it.
template <int LEFT> __device__ __forceinline__ void step_barrier() {
    static_assert(LEFT < 64, "the counter has six bits");
    asm volatile("" ::: "memory");  // (the compiler moves no access across)
    __builtin_amdgcn_s_waitcnt(0x0070 | (LEFT & 15) | (LEFT >> 4) << 14);
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// Where in its 128 bytes a row has a piece of 16 (and which piece lies at a place): 16 rows' same pieces, two rows to a line of the 64 banks,
// meet every bank once.  (By the row's lowest three bits, two and two in the same banks, half of the time in LDS was lost: 104M of
// 212M cycles over the compute units at 16,384 x 8192 against 8192 codes, now 3M of 111M.)
__device__ __forceinline__ int piece_place(int row, int piece) { return (piece ^ (row >> 1 & 7)) * 16; }

// TR rows x TC codes by WR x WC waves, each TR / WR rows x TC / WC codes in blocks of 32 x 32.  The operands come in steps of 128
// components straight into LDS, the next step's on their way while a step is worked on; one barrier per step.  A row of a step
// is 128 bytes there, its eight 16-byte pieces in an order that depends on the row, so that the reads of a fragment (32 rows at the
// same place) meet all banks; since the copies fill LDS in the order of the lanes, each lane fetches the piece that belongs at its place.
// Buffer addresses are checked by the hardware: rows behind the last read as zeros.  Every row's bytes behind component `dim`
// are somebody's data: they are cleared in the rows of x before the last step is worked on, and count for nothing in w then.
// The codes are the first operand: a lane ends with runs of four codes of a row, scales them, and the tile leaves through LDS in whole lines.
// Aligned rows only (address and stride multiples of 16).
template <typename OutT, int TR, int TC, int WR, int WC, int KS, int STAGES>
__global__ void __launch_bounds__(64 * WR * WC) k_scores_tile(ScoresArgs a, uint32_t row_tiles, uint32_t code_tiles, int lds_bytes) {
    constexpr int NW = WR * WC, R = TR / WR / 32, C = TC / WC / 32, XI = TR / 8 / NW, WI = TC / 8 / NW, HALF = (TR + TC) * 128, STAGE = KS * HALF, STEP = KS * 128;
    static_assert(XI * 8 * NW == TR && WI * 8 * NW == TC && R * 32 * WR == TR && C * 32 * WC == TC, "whole blocks");
    typedef typename OutT::Raw Raw;
    extern __shared__ __attribute__((aligned(1024))) char tile_lds[];
    constexpr int LINE = C * 32 * (int)sizeof(Raw), PITCH = LINE + 16, PIECES = LINE / 16;  // of a block of rows on its way out
    float *lws = reinterpret_cast<float *>(tile_lds + lds_bytes), *lbias = lws + TC;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), wr = wave / WC, wc = wave % WC;
    const TilePlace place = tile_place(blockIdx.x, row_tiles, code_tiles);
    const int64_t row0 = place.r * TR;
    const int code0 = place.c * TC, rows = (int)min((int64_t)TR, a.n - row0), codes = min(TC, a.k - code0);
    const int steps = (a.dim + STEP - 1) / STEP, dim16 = (a.dim + 15) & ~15;
    const int8_t *px = a.x + row0 * a.ld_x, *pw = a.w + (int64_t)code0 * a.ld_w;
    const int ldx = (int)a.ld_x, ldw = (int)a.ld_w, left_x = (rows - 1) * ldx + dim16, left_w = (codes - 1) * ldw + dim16;
    int vx[XI], vw[WI];
#pragma unroll
    for (int i = 0; i < XI; ++i) {
        const int row = (wave * XI + i) * 8 + (lane >> 3);
        vx[i] = row * ldx + piece_place(row, lane & 7);
    }
#pragma unroll
    for (int i = 0; i < WI; ++i) {
        const int row = (wave * WI + i) * 8 + (lane >> 3);
        vw[i] = row * ldw + piece_place(row, lane & 7);
    }
    const auto bring = [&](int step, int buf) {
#pragma unroll
        for (int kb = 0; kb < KS; ++kb) {
            const int at = step * STEP + kb * 128;
            char *to = tile_lds + buf * STAGE + kb * HALF;
            const bool any = KS == 1 || at < dim16;  // else nothing is read, and LDS gets zeros
#pragma unroll
            for (int i = 0; i < XI; ++i) copy_to_lds(px + at, any ? left_x - at : 0, to + (wave * XI + i) * 1024, vx[i]);
#pragma unroll
            for (int i = 0; i < WI; ++i) copy_to_lds(pw + at, any ? left_w - at : 0, to + TR * 128 + (wave * WI + i) * 1024, vw[i]);
        }
    };
    for (int j = tid; j < TC; j += 64 * NW) {
        lws[j] = j < codes ? a.ws[code0 + j] : 0.0f;
        lbias[j] = a.bias && j < codes ? a.bias[code0 + j] : -0.0f;  // (adding -0 changes nothing, not even a zero's sign)
    }
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i)
        if (i < steps) bring(i, i);
    i32x16 acc[R][C];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[r][c][i] = 0;
    const int l32 = lane & 31, h = lane >> 5;
    int off[4];
#pragma unroll
    for (int s = 0; s < 4; ++s) off[s] = l32 * 128 + piece_place(l32, 2 * s + h);
    int buf = 0;  // step % STAGES
    for (int step = 0; step < steps; ++step) {
        if (step + STAGES - 1 <= steps)
            step_barrier<(STAGES - 2) * KS * (XI + WI)>();
        else
            step_barrier<0>();
        if (step + STAGES - 1 < steps) bring(step + STAGES - 1, buf == 0 ? STAGES - 1 : buf - 1);  // where the step before lay
        char *at = tile_lds + buf * STAGE;
        buf = buf + 1 == STAGES ? 0 : buf + 1;
        if (step + 1 == steps && a.dim % STEP) {  // uniform
            for (int i = tid; i < KS * TR * 8; i += 64 * NW) {
                const int kb = i / (TR * 8), row = i / 8 % TR, p = step * STEP + kb * 128 + (i & 7) * 16;  // the piece of components p to p + 15
                if (p + 16 > a.dim) {
                    i32x4 *v = reinterpret_cast<i32x4 *>(at + kb * HALF + row * 128 + piece_place(row, i & 7));
                    i32x4 x = *v;
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const int keep = min(max(a.dim - p - 4 * q, 0), 4);
                        x[q] = keep == 4 ? x[q] : x[q] & ((1 << (8 * keep)) - 1);
                    }
                    *v = x;
                }
            }
            __syncthreads();
        }
        const char *ax = at + wr * (R * 32 * 128), *aw = at + TR * 128 + wc * (C * 32 * 128);
        i32x4 fx[2][R], fw[2][C];  // of a quarter of the step, and of the next
        const auto read = [&](int s) {
#pragma unroll
            for (int c = 0; c < C; ++c) fw[s & 1][c] = *reinterpret_cast<const i32x4 *>(aw + (s >> 2) * HALF + c * 4096 + off[s & 3]);
#pragma unroll
            for (int r = 0; r < R; ++r) fx[s & 1][r] = *reinterpret_cast<const i32x4 *>(ax + (s >> 2) * HALF + r * 4096 + off[s & 3]);
        };
        read(0);
#pragma unroll
        for (int s = 0; s < 4 * KS; ++s) {
            if (s + 1 < 4 * KS) read(s + 1);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int c = 0; c < C; ++c)
                    acc[r][c] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fw[s & 1][c], fx[s & 1][r], acc[r][c], 0, 0, 0);
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    step_barrier<0>();  // LDS is free
    char *mine = tile_lds + wave * (32 * PITCH);
    // Whole lines of 128 bytes pass the caches (16,384 x 512 x 16,384 to f32 367 -> 285 us, 100,000 x 384 x 1024 142 -> 103); parts of
    // lines would each cost memory a line (1M x 128 x 256 to bf16 with 64 bytes per wave and row 172 -> 190, 3000 x 300 x 3000, whose
    // rows end inside lines, 15.7 -> 19.8).
    const bool past = ((uintptr_t)a.out & 127) == 0 && a.ld_out % (128 / (int)sizeof(Raw)) == 0;
    const int wcode = code0 + wc * (C * 32);
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int64_t brow = row0 + wr * (R * 32) + r * 32;
        const float xs = a.xs[min(brow + l32, a.n - 1)];
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int j = wc * (C * 32) + c * 32 + q * 8 + h * 4;
                const f32x4 s4 = *reinterpret_cast<const f32x4 *>(lws + j), b4 = *reinterpret_cast<const f32x4 *>(lbias + j);
                struct __attribute__((aligned(4 * sizeof(Raw)))) {
                    Raw v[4];
                } o;
#pragma unroll
                for (int i = 0; i < 4; ++i) o.v[i] = OutT::down((float)acc[r][c][q * 4 + i] * xs * s4[i] + b4[i]);
                __builtin_memcpy(mine + l32 * PITCH + (c * 32 + q * 8 + h * 4) * sizeof(Raw), &o, sizeof(o));
            }
        wave_sync();
#pragma unroll
        for (int i = lane; i < 32 * PIECES; i += 64) {
            const int row = i / PIECES, piece = i % PIECES, code = wcode + piece * (16 / (int)sizeof(Raw));
            struct __attribute__((packed, aligned(sizeof(Raw)))) Piece {
                uint32_t w[4];
            };
            const i32x4 v = *reinterpret_cast<const i32x4 *>(mine + row * PITCH + piece * 16);
            if (brow + row < a.n && code < a.k) {
                Raw *to = (Raw *)a.out + (brow + row) * a.ld_out + code;
                if (code + 16 / (int)sizeof(Raw) > a.k)
                    for (int e = 0; e < 16 / (int)sizeof(Raw); ++e) {
                        if (code + e < a.k) to[e] = reinterpret_cast<const Raw *>(mine + row * PITCH + piece * 16)[e];
                    }
                else if (LINE >= 128 && past)
                    __builtin_nontemporal_store(v, reinterpret_cast<i32x4 *>(to));
                else
                    *reinterpret_cast<Piece *>(to) = __builtin_bit_cast(Piece, v);
            }
        }
        wave_sync();
    }
}
// LDS of a workgroup below its codes' scales and biases (8 bytes each): the steps in flight, or a block of rows per wave on its way
// out.  Short rows have fewer steps than are provided for; more workgroups share a compute unit then.
inline int tile_lds_bytes(int tr, int tc, int waves, int waves_c, int ks, int stages, int dim, int bytes) {
    const int steps = std::min(stages, (dim + ks * 128 - 1) / (ks * 128));
    return std::max(steps * ks * (tr + tc) * 128, waves * 32 * (tc / waves_c * bytes + 16));
}

// ---- few tiles: the components shared out among the waves -------------------------------------------------
// A workgroup makes RB * 16 rows x CB * 16 codes, each of its KW waves from every KW-th run of 128 components, straight from memory into the
// operands' registers, the next run on its way; the waves' sums meet in LDS.  16 rows of 64 consecutive bytes per read.  Rows and
// codes behind the last are read as the last; components behind `dim` count as zero in x.  Aligned rows only.
template <typename OutT, int RB, int CB, int KW>
__global__ void __launch_bounds__(64 * KW) k_scores_few(ScoresArgs a) {
    constexpr int TR = RB * 16, TC = CB * 16, PITCH = TC + 4;
    typedef typename OutT::Raw Raw;
    __shared__ __attribute__((aligned(16))) int32_t sums[KW][TR][PITCH];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), l16 = lane & 15, h = lane >> 4;
    const int64_t row0 = (int64_t)blockIdx.y * TR;
    const int code0 = blockIdx.x * TC;
    const int8_t *px[RB], *pw[CB];
#pragma unroll
    for (int r = 0; r < RB; ++r) px[r] = a.x + min(row0 + r * 16 + l16, a.n - 1) * a.ld_x;
#pragma unroll
    for (int c = 0; c < CB; ++c) pw[c] = a.w + (int64_t)min(code0 + c * 16 + l16, a.k - 1) * a.ld_w;
    i32x4 acc[RB][CB];
#pragma unroll
    for (int r = 0; r < RB; ++r)
#pragma unroll
        for (int c = 0; c < CB; ++c) acc[r][c] = i32x4{0, 0, 0, 0};
    struct Run {
        i32x4 x[RB][2], w[CB][2];
    };
    const auto bring = [&](Run &f, int t0) {
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const int t = t0 + s * 64 + h * 16, at = t < a.dim ? t : 0;  // (what is behind the row counts for nothing)
#pragma unroll
            for (int c = 0; c < CB; ++c) f.w[c][s] = *reinterpret_cast<const i32x4 *>(pw[c] + at);
#pragma unroll
            for (int r = 0; r < RB; ++r) f.x[r][s] = *reinterpret_cast<const i32x4 *>(px[r] + at);
        }
    };
    const auto use = [&](Run &f, int t0) {
        if (t0 + 128 > a.dim) {  // uniform
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int keep = min(max(a.dim - (t0 + s * 64 + h * 16 + 4 * q), 0), 4);
                    const int mask = keep == 4 ? -1 : (1 << (8 * keep)) - 1;
#pragma unroll
                    for (int r = 0; r < RB; ++r) f.x[r][s][q] &= mask;
                }
        }
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int r = 0; r < RB; ++r)
#pragma unroll
                for (int c = 0; c < CB; ++c) acc[r][c] = __builtin_amdgcn_mfma_i32_16x16x64_i8(f.w[c][s], f.x[r][s], acc[r][c], 0, 0, 0);
    };
    Run f[2];
    int t = wave * 128;
    if (t < a.dim) bring(f[0], t);
    for (; t < a.dim; t += KW * 256) {
        if (t + KW * 128 < a.dim) bring(f[1], t + KW * 128);
        use(f[0], t);
        if (t + KW * 256 < a.dim) bring(f[0], t + KW * 256);
        if (t + KW * 128 < a.dim) use(f[1], t + KW * 128);
    }
#pragma unroll
    for (int r = 0; r < RB; ++r)
#pragma unroll
        for (int c = 0; c < CB; ++c) *reinterpret_cast<i32x4 *>(&sums[wave][r * 16 + l16][c * 16 + h * 4]) = acc[r][c];
    __syncthreads();
#pragma unroll
    for (int i = tid; i < TR * TC; i += 64 * KW) {
        const int row = i / TC, j = i % TC;
        int32_t sum = 0;
#pragma unroll
        for (int w = 0; w < KW; ++w) sum += sums[w][row][j];
        if (row0 + row < a.n && code0 + j < a.k) {
            const float y = (float)sum * a.xs[row0 + row] * a.ws[code0 + j];
            ((Raw *)a.out)[(row0 + row) * a.ld_out + code0 + j] = OutT::down(a.bias ? y + a.bias[code0 + j] : y);
        }
    }
}

}  // namespace vq
