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

// ---- the codes of a lane ----------------------------------------------------------------------------
// A row, or a part of it, lies in the registers of LANES lanes for the whole of its pass, so that it is read once: vector u
// of a lane holds the codes from lo + (u * LANES + lane) * VEC on, 16 bytes of them.  A vector that would pass the end
// hi is read from hi - VEC on instead, without a branch, and what lies before its own place in it becomes -inf.
typedef uint32_t AnyWords __attribute__((ext_vector_type(4), aligned(2)));  // 16 bytes at any element
template <typename T, int LANES, int NV> struct Share {
    typedef typename T::Raw Raw;
    static constexpr int VEC = 16 / (int)sizeof(Raw), E = NV * VEC;
    struct __attribute__((packed, aligned(sizeof(Raw)))) Piece {
        uint32_t w[4];
    };
    Piece raw[NV];
    float x[E];

    static __device__ __forceinline__ int base(int u, int lane, int lo, int hi) { return min(lo + (u * LANES + lane) * VEC, hi - VEC); }

    // The reads of a row that nobody is expected to read after this: they pass the caches (rows to 8 bits and their scores, 1M x 128 x 256
    // 306 -> 274 us, gradients of 8192 x 65,536 401 -> 389; short rows' log probabilities 215 -> 219, they go by load).
    __device__ __forceinline__ void fetch_once(const Raw *s, int lo, int hi, int lane) {
#pragma unroll
        for (int u = 0; u < NV; ++u)
            if (u == 0 || lo + u * LANES * VEC < hi)
                raw[u] = __builtin_bit_cast(Piece, __builtin_nontemporal_load(reinterpret_cast<const AnyWords *>(s + base(u, lane, lo, hi))));
    }
    static __device__ __forceinline__ void values(const Piece &piece, float *to) {
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            if constexpr (sizeof(Raw) == 4)
                to[v] = __uint_as_float(piece.w[v]);
            else
                to[v] = T::up((Raw)(v & 1 ? piece.w[v >> 1] >> 16 : piece.w[v >> 1] & 0xffffu));
        }
    }
    __device__ __forceinline__ void load(const Raw *s, int lo, int hi, int lane) {
        if (lo + LANES * E <= hi) {  // uniform: whole vectors all of them
#pragma unroll
            for (int u = 0; u < NV; ++u) raw[u] = *reinterpret_cast<const Piece *>(s + lo + (u * LANES + lane) * VEC);
#pragma unroll
            for (int u = 0; u < NV; ++u) values(raw[u], x + u * VEC);
            return;
        }
#pragma unroll
        for (int u = 0; u < NV; ++u) raw[u] = *reinterpret_cast<const Piece *>(s + base(u, lane, lo, hi));
#pragma unroll
        for (int u = 0; u < NV; ++u) {
            values(raw[u], x + u * VEC);
            if (lo + (u + 1) * LANES * VEC > hi) {  // uniform: the vectors that are read from elsewhere, or have nothing of the row
                const int skip = lo + (u * LANES + lane) * VEC - base(u, lane, lo, hi);
#pragma unroll
                for (int v = 0; v < VEC; ++v) x[u * VEC + v] = v < skip ? kNegInf : x[u * VEC + v];
            }
        }
    }
    __device__ __forceinline__ int code(int e, int lane, int lo, int hi) const { return base(e / VEC, lane, lo, hi) + e % VEC; }
};

// The larger one: of a number and a NaN the number (a NaN in a row shows in its sums), and the NaN.
__device__ __forceinline__ float larger(float a, float b) { return __builtin_fmaxf(a, b); }
__device__ __forceinline__ float larger_or_nan(float a, float b) { return __builtin_elementwise_maximum(a, b); }

// Over the lanes of aligned groups of G, for every lane of the group, in an order that is the same in every run.  f's first
// operand stays where a step brings nothing.
template <int CTRL, int ROWS = 0xf> __device__ __forceinline__ uint32_t dpp_keep(uint32_t old, uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp((int)old, (int)v, CTRL, ROWS, 0xf, false);
}
template <int CTRL> __device__ __forceinline__ uint32_t dpp_all(uint32_t v) {  // every lane of a row brings something
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true);
}
template <int G, typename F> __device__ __forceinline__ uint32_t over_group(uint32_t v, uint32_t none, F f) {
    if constexpr (G >= 2) v = f(v, dpp_all<0xB1>(v));
    if constexpr (G >= 4) v = f(v, dpp_all<0x4E>(v));
    if constexpr (G >= 8) v = f(v, dpp_all<0x141>(v));
    if constexpr (G >= 16) v = f(v, dpp_all<0x140>(v));
    static_assert(G <= 16 || G == 64, "rows of 16 lanes, or the wave");
    if constexpr (G == 64) {
        v = f(v, dpp_keep<0x142, 0xa>(none, v));  // a row's last lane to the next row
        v = f(v, dpp_keep<0x143, 0xc>(none, v));  // the lower half's to the upper half
        v = (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
    }
    return v;
}
template <int G> __device__ __forceinline__ float group_max(float v) {
    return __uint_as_float(over_group<G>(__float_as_uint(v), __float_as_uint(kNegInf), [](uint32_t a, uint32_t b) {
        return __float_as_uint(larger(__uint_as_float(a), __uint_as_float(b)));
    }));
}
template <int G> __device__ __forceinline__ float group_sum(float v) {
    return __uint_as_float(over_group<G>(__float_as_uint(v), 0u, [](uint32_t a, uint32_t b) {
        return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
    }));
}
template <int G> __device__ __forceinline__ int group_min(int v) {
    return (int)over_group<G>((uint32_t)v, 0x7fffffffu, [](uint32_t a, uint32_t b) { return (uint32_t)min((int)a, (int)b); });
}
// Sums of the scores of a lane relative to the largest score m of their row or part: S = sum 2^d, W = sum 2^d d with
// d = (x - m) * c, c = beta * log2 e, held above -200 (2^-200 is zero in f32, and zero times it a zero) but for a NaN, which makes the
// sums NaN: m is the largest number of the row.  One fused operation per exponent, x * c - M with M = m * c rounded; what M is off by, r = m * c - M, is exact and the same for all of
// them, and taken out of the joined sums (away).  Below |M| = 10^6 r is at most 1/32; from there on exponents are formed from x - m.
struct Sums {
    float m, S = 0.0f, W = 0.0f, r = 0.0f;
    template <int E> __device__ __forceinline__ Sums(const float (&x)[E], float most, float c) : m(most) {
        const float from = is_bad(m) || m == kNegInf ? 0.0f : m, M = from * c;  // (such rows' sums are not looked at)
        if (__ballot(fabsf(M) >= 1e6f) == 0) {
            r = __builtin_fmaf(from, c, -M);
#pragma unroll
            for (int e = 0; e < E; ++e) add(__builtin_fmaf(x[e], c, -M));
        } else {  // each row of the wave in its own way, so that its bits do not depend on what the others hold
            const bool far = fabsf(M) >= 1e6f;
            const float off = far ? from : 0.0f, by = far ? 0.0f : M;
            r = far ? 0.0f : __builtin_fmaf(from, c, -M);
#pragma unroll
            for (int e = 0; e < E; ++e) add(__builtin_fmaf(x[e] - off, c, -by));
        }
    }
    __device__ __forceinline__ Sums(float most, float sum, float weighted) : m(most), S(sum), W(weighted) {}
    __device__ __forceinline__ void add(float exponent) {
        const float d = larger_or_nan(exponent, -200.0f), p = __builtin_amdgcn_exp2f(d);
        S += p;
        W = __builtin_fmaf(p, d, W);
    }
    __device__ __forceinline__ void away() {
        const float f = __builtin_amdgcn_exp2f(-r);
        W = f * __builtin_fmaf(-r, S, W);
        S *= f;
    }
    static __device__ __forceinline__ bool is_bad(float m) { return !(m < __builtin_inff()); }
};

struct RowSums {
    float m, L, H;
};
__device__ __forceinline__ RowSums row_sums(const Sums &s) {
    if (s.S != s.S) return {s.S, s.S, s.S};
    if (Sums::is_bad(s.m)) return {s.m, __builtin_nanf(""), __builtin_nanf("")};
    if (s.m == kNegInf) return {s.m, kNegInf, 0.0f};
    // S is 1 or above, the largest score's own term, and -W zero or above; rounding may leave either a bit short, so L and H are held at 0:
    // no log probability is above zero and no entropy below
    const float L = fmaxf(__builtin_amdgcn_logf(s.S) * kLn2, 0.0f);  // (log2)
    return {s.m, L, fmaxf(__builtin_fmaf(-s.W * __builtin_amdgcn_rcpf(s.S), kLn2, L), 0.0f)};
}
// The log probability of the row's code, whose score was read with the row.
struct CodeScore {
    int64_t code = -1;
    float score = 0.0f;
    template <typename T> __device__ __forceinline__ void read(const LogprobArgs &a, int64_t row, T) {
        if (!a.logprob) return;
        code = code_at(a.codes, a.code_bytes, row * a.code_stride);
        if (code >= 0 && code < a.k) score = T::up(((const typename T::Raw *)a.s)[row * a.ld + code]);
    }
};
// beta * (s - m) - L for a score s of a row, by half the difference: scores of +-3e38 are further apart than f32 reaches, and a beta
// below 1 brings them back.
__device__ __forceinline__ float log_probability(float beta, float s, const RowSums &r) {
    return 2.0f * beta * __builtin_fmaf(0.5f, s, -0.5f * r.m) - r.L;
}
__device__ __forceinline__ void write_row(const LogprobArgs &a, int64_t row, const RowSums &r, const CodeScore &c) {
    if (a.max) a.max[row] = r.m;
    if (a.logsum) a.logsum[row] = r.L;
    if (a.entropy) a.entropy[row] = r.H;
    if (a.logprob)
        a.logprob[row] = c.code < 0 ? 0.0f : c.code >= a.k ? __builtin_nanf("") : r.m == kNegInf ? kNegInf : log_probability(a.beta, c.score, r);
}
// An alternative as it is written: its log probability and its code.
struct Alternative {
    float lp = 0.0f;
    int32_t code = -1;
    __device__ __forceinline__ void set(const LogprobArgs &a, float v, int c, const RowSums &r) {
        const bool bad = r.L != r.L, none = v == kNegInf || c < 0;
        lp = bad ? __builtin_nanf("") : none ? kNegInf : log_probability(a.beta, v, r);
        code = bad || none ? -1 : c;
    }
    __device__ __forceinline__ void write(const LogprobArgs &a, int64_t row, int t) const {
        a.top_logprob[row * a.top + t] = lp;
        a.top_code[row * a.top + t] = code;
    }
};
__device__ __forceinline__ void write_alternative(const LogprobArgs &a, int64_t row, int t, uint64_t key, const RowSums &r) {
    Alternative o;
    o.set(a, key_score(key), key ? key_code(key) : -1, r);
    o.write(a, row, t);
}

// One round per alternative over the scores of G lanes, which it empties: the largest score left, the first code that has
// it, which then leaves.  Lane t % G keeps alternative t, and the lanes write G of them at a time.  code_of(e): the code of a lane's score e.
template <int G, int E, typename F>
__device__ __forceinline__ void best_by_rounds(const LogprobArgs &a, int64_t row, bool writes, float (&x)[E], const RowSums &r, int lane, F code_of) {
    float best = x[0];
#pragma unroll
    for (int e = 1; e < E; ++e) best = larger(best, x[e]);
    best = group_max<G>(best);
    Alternative o;
    for (int t = 0; t < a.top; ++t) {
        int e0 = -1;
#pragma unroll
        for (int e = E - 1; e >= 0; --e) e0 = x[e] == best ? e : e0;
        const int at = e0 < 0 ? 0x7fffffff : code_of(e0), first = group_min<G>(at);
        if ((t & (G - 1)) == lane) o.set(a, best, first == 0x7fffffff ? -1 : first, r);
        if (((t & (G - 1)) == G - 1 || t + 1 == a.top) && lane <= (t & (G - 1)) && writes) o.write(a, row, (t & ~(G - 1)) + lane);
        if (t + 1 == a.top) break;
        const int gone = at == first ? e0 : -1;
        best = kNegInf;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            x[e] = e == gone ? kNegInf : x[e];
            best = larger(best, x[e]);
        }
        best = group_max<G>(best);
    }
}

// ---- short rows: G lanes each ------------------------------------------------------------------------
// Up to 16 codes per lane, or 32, 64 / G rows per wave: no LDS, no waits.  Bound by its instructions as much as by memory, so a
// row of 256 has 8 lanes rather than 16, and what every row costs is shared by eight of them (a million rows of 256 scores, two alternatives 215 -> 190 us).
// TINY: rows shorter than a vector, one lane each.
template <typename T, int G, int E, bool TINY>
__global__ void __launch_bounds__(256) k_logprobs_short(LogprobArgs a) {
    typedef Share<T, G, TINY ? 1 : E * (int)sizeof(typename T::Raw) / 16> SE;
    const int lane = threadIdx.x & (G - 1);
    const int64_t mine = (int64_t)blockIdx.x * (256 / G) + threadIdx.x / G, row = min(mine, a.n - 1);
    const typename T::Raw *s = (const typename T::Raw *)a.s + row * a.ld;
    SE r;
    if constexpr (TINY) {
#pragma unroll
        for (int e = 0; e < SE::E; ++e) r.x[e] = e < a.k ? T::up(s[e]) : kNegInf;
    } else
        r.load(s, 0, a.k, lane);
    CodeScore cs;
    cs.read(a, row, T());
    float m = r.x[0];
#pragma unroll
    for (int e = 1; e < SE::E; ++e) m = larger(m, r.x[e]);
    m = group_max<G>(m);
    Sums sum(r.x, m, a.beta * kLog2e);
    sum.S = group_sum<G>(sum.S);
    sum.W = group_sum<G>(sum.W);
    sum.away();
    const RowSums sums = row_sums(sum);
    const bool writes = mine < a.n;
    if (writes && lane == 0) write_row(a, row, sums, cs);
    if (a.top) best_by_rounds<G>(a, row, writes, r.x, sums, lane, [&](int e) { return TINY ? e : r.code(e, lane, 0, a.k); });
}

__device__ __forceinline__ void wave_sync() {  // a wave's reads and writes of LDS stay in order
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// A value that q of the lanes' values reach, of which `most` is the largest: the q-th largest of them, in a round per value up to eight,
// beyond that the bits of its rank from the highest down to bit LOW, a compare and a count of lanes each.
template <int LOW> __device__ __forceinline__ float lane_floor(float value, float most, int q, int lane) {
    if (q > 8) {  // uniform
        const uint32_t mine = (uint32_t)(rank_key(larger(value, kNegInf), 0) >> 32);
        uint32_t at = 0;
#pragma unroll
        for (int bit = 31; bit >= LOW; --bit) {
            const uint32_t next = at | 1u << bit;
            if (__popcll(__ballot(mine >= next)) >= q) at = next;
        }
        return larger(key_score((uint64_t)at << 32), kNegInf);  // (below the rank of -inf lie NaNs)
    }
    while (--q > 0) {
        const unsigned long long who = __ballot(value == most);
        if (lane == __ffsll(who) - 1) value = kNegInf;
        most = group_max<64>(value);
    }
    return most;
}

// How many of the keys in LDS are above one; zeros up to a whole eight of them lie behind the last.
__device__ __forceinline__ int keys_above(const uint64_t *key, int count, uint64_t mine) {
    int above = 0;
    for (int j = 0; j < count; j += 8) {
        uint64_t o[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) o[u] = key[j + u];
#pragma unroll
        for (int u = 0; u < 8; ++u) above += o[u] > mine;
    }
    return above;
}

// ---- rows of a wave -------------------------------------------------------------------------------------
// E codes per lane, a row per wave.  The alternatives come from a list of the scores that reach a floor, the top-th largest of the
// lanes' largest ones; the list is sorted by counting.  A list that does not fit, as of a row of equal scores, is not taken: then by rounds.
constexpr int kWaveList = 128;

template <typename T, int E>
__global__ void __launch_bounds__(256, E <= 16 ? 8 : E == 32 ? 6 : 4) k_logprobs_wave(LogprobArgs a) {
    typedef Share<T, 64, E * (int)sizeof(typename T::Raw) / 16> SE;
    __shared__ uint64_t lists[4][kWaveList + 8 + 32];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), top = a.top;
    const int64_t row = (int64_t)blockIdx.x * 4 + wave;
    if (row >= a.n) return;  // (no barriers below)
    SE r;
    r.load((const typename T::Raw *)a.s + row * a.ld, 0, a.k, lane);
    CodeScore cs;
    cs.read(a, row, T());
    float most = r.x[0];
#pragma unroll
    for (int e = 1; e < E; ++e) most = larger(most, r.x[e]);
    const float m = group_max<64>(most);
    Sums sum(r.x, m, a.beta * kLog2e);
    sum.S = group_sum<64>(sum.S);
    sum.W = group_sum<64>(sum.W);
    sum.away();
    const RowSums sums = row_sums(sum);
    if (lane == 0) write_row(a, row, sums, cs);
    if (top == 0) return;
    float floor = a.k <= kWaveList ? kNegInf : lane_floor<sizeof(typename T::Raw) == 2 ? 16 : 8>(most, m, top, lane);  // (short rows: all of them)
    floor = fmaxf(floor, -3.402823466e38f);  // -inf is none of them
    uint64_t *list = lists[wave], *best = list + kWaveList + 8;
    int count = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const unsigned long long who = __ballot(r.x[e] >= floor);
        if (!who) continue;
        const int at = count + __popcll(who & ((1ull << lane) - 1));
        if (r.x[e] >= floor && at < kWaveList) list[at] = rank_key(r.x[e], (uint32_t)r.code(e, lane, 0, a.k));
        count += __popcll(who);
    }
    if (count > kWaveList) {  // uniform
        best_by_rounds<64>(a, row, true, r.x, sums, lane, [&](int e) { return r.code(e, lane, 0, a.k); });
        return;
    }
    if (lane < 8) list[count + lane] = 0;
    if (lane < 32) best[lane] = 0;
    wave_sync();
    for (int i = lane; i < count; i += 64) {
        const uint64_t mine = list[i];
        const int rank = keys_above(list, count, mine);
        if (rank < top) best[rank] = mine;
    }
    wave_sync();
    if (lane < top) write_alternative(a, row, lane, best[lane], sums);
}

// ---- longer rows, in parts: a workgroup each ------------------------------------------------------------
constexpr int kMostCandidates = 512;

struct PartArgs {
    LogprobArgs a;
    int parts, part_codes;  // part q has the codes from q * part_codes on
    float *sums;     // [n][parts][3]: largest score, S, W
    uint64_t *keys;  // [n][parts][top], in falling order, 0 behind the last
};

struct PartLds {
    float red[4][4];
    int count;
    uint64_t key[kMostCandidates + 8];
    uint64_t best[32];
};

// The `top` largest of a workgroup's scores, in falling order, into l.best (0 behind the last one above -inf).
// floor: a score that at least `top` of the scores reach, if there are as many.  What reaches it is listed (in whatever order, the
// keys are all different) and sorted by counting; a longer list than there is room for, as of a row of equal scores, is not
// taken: then one round per alternative over the registers, which empties them.
template <typename S64>
__device__ __forceinline__ void part_best(S64 &r, const float (&vmax)[S64::E / S64::VEC], float floor, int lo, int hi, int top, PartLds &l) {
    constexpr int NV = S64::E / S64::VEC;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
#pragma unroll
    for (int u = 0; u < NV; ++u) {
        if (!__ballot(vmax[u] >= floor)) continue;
#pragma unroll
        for (int v = 0; v < S64::VEC; ++v) {
            const float y = r.x[u * S64::VEC + v];
            if (y >= floor) {
                const int at = atomicAdd(&l.count, 1);
                if (at < kMostCandidates) l.key[at] = rank_key(y, (uint32_t)r.code(u * S64::VEC + v, tid, lo, hi));
            }
        }
    }
    if (tid < 32) l.best[tid] = 0;
    __syncthreads();
    const int count = l.count;
    if (count <= kMostCandidates) {
        if (tid < 8) l.key[count + tid] = 0;  // (up to a whole eight)
        __syncthreads();
        for (int i = tid; i < count; i += 256) {
            const uint64_t mine = l.key[i];
            const int above = keys_above(l.key, count, mine);
            if (above < top) l.best[above] = mine;
        }
        __syncthreads();
        return;
    }
    __syncthreads();  // everyone has read the count and the zeros are there
    float best = kNegInf;
#pragma unroll
    for (int e = 0; e < S64::E; ++e) best = fmaxf(best, r.x[e]);
    for (int t = 0; t < top; ++t) {
        best = group_max<64>(best);
        if (lane == 0) l.red[0][wave] = best;
        __syncthreads();
        best = fmaxf(fmaxf(l.red[0][0], l.red[0][1]), fmaxf(l.red[0][2], l.red[0][3]));
        if (best == kNegInf) break;  // the same in every lane
        int e0 = -1;
#pragma unroll
        for (int e = S64::E - 1; e >= 0; --e) e0 = r.x[e] == best ? e : e0;
        const int at = e0 < 0 ? 0x7fffffff : r.code(e0, tid, lo, hi);
        int first = group_min<64>(at);
        if (lane == 0) l.red[1][wave] = __int_as_float(first);
        __syncthreads();
#pragma unroll
        for (int w = 0; w < 4; ++w) first = min(first, __float_as_int(l.red[1][w]));
        if (tid == 0) l.best[t] = rank_key(best, (uint32_t)first);
        best = kNegInf;
#pragma unroll
        for (int e = 0; e < S64::E; ++e) {
            r.x[e] = e == e0 && at == first ? kNegInf : r.x[e];
            best = fmaxf(best, r.x[e]);
        }
    }
    __syncthreads();
}

template <typename T, int NV>
__global__ void __launch_bounds__(256, 16 / (int)sizeof(typename T::Raw) * NV <= 32 ? 8 : 4) k_logprobs_part(PartArgs p) {
    typedef Share<T, 256, NV> S64;
    constexpr int VEC = S64::VEC;
    __shared__ PartLds l;
    const LogprobArgs &a = p.a;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t row = blockIdx.x / (unsigned)p.parts;
    const int part = (int)(blockIdx.x % (unsigned)p.parts), lo = part * p.part_codes, hi = min(a.k, lo + p.part_codes);
    S64 r;
    r.load((const typename T::Raw *)a.s + row * a.ld, lo, hi, tid);
    CodeScore cs;
    if (p.parts == 1 && tid == 0) cs.read(a, row, T());
    float vmax[NV], m;
#pragma unroll
    for (int u = 0; u < NV; ++u) {
        vmax[u] = r.x[u * VEC];
#pragma unroll
        for (int v = 1; v < VEC; ++v) vmax[u] = larger(vmax[u], r.x[u * VEC + v]);
        m = u ? larger(m, vmax[u]) : vmax[u];
    }
    const float mine = m;
    m = group_max<64>(m);
    // The floor of the alternatives: in each of the waves whose lanes all have codes, a share of them, rounded up, of the lanes have a score
    // that reaches the wave's floor, so `top` scores reach the smallest of these.
    const int full = max(1, min(4, (hi - lo) / (64 * VEC)));
    float floor = m;
    if (a.top && wave < full) floor = lane_floor<sizeof(typename T::Raw) == 2 ? 16 : 8>(mine, m, (a.top + full - 1) / full, lane);
    if (lane == 0) l.red[0][wave] = m, l.red[1][wave] = floor;
    if (tid == 0) l.count = 0;
    __syncthreads();
    m = larger(larger(l.red[0][0], l.red[0][1]), larger(l.red[0][2], l.red[0][3]));
    floor = l.red[1][0];
    for (int w = 1; w < full; ++w) floor = fminf(floor, l.red[1][w]);
    floor = fmaxf(floor, -3.402823466e38f);  // -inf is none of them
    Sums sum(r.x, m, a.beta * kLog2e);
    sum.S = group_sum<64>(sum.S);
    sum.W = group_sum<64>(sum.W);
    if (lane == 0) l.red[2][wave] = sum.S, l.red[3][wave] = sum.W;
    if (a.top && !Sums::is_bad(m)) part_best(r, vmax, floor, lo, hi, a.top, l);
    else if (tid < 32) l.best[tid] = 0;
    __syncthreads();
    if (wave) return;
    sum.S = l.red[2][0] + l.red[2][1] + l.red[2][2] + l.red[2][3];
    sum.W = l.red[3][0] + l.red[3][1] + l.red[3][2] + l.red[3][3];
    sum.away();
    if (p.parts == 1) {
        const RowSums sums = row_sums(sum);
        if (lane == 0) write_row(a, row, sums, cs);
        if (lane < a.top) write_alternative(a, row, lane, l.best[lane], sums);
    } else {
        const int64_t at = blockIdx.x;
        if (lane == 0) p.sums[at * 3] = sum.m, p.sums[at * 3 + 1] = sum.S, p.sums[at * 3 + 2] = sum.W;
        if (lane < a.top) p.keys[at * a.top + lane] = l.best[lane];
    }
}

// A wave joins the parts of a row: sums rescaled to the largest score of all, and the alternatives from the parts' lists.
// With j = (top - 1) / parts, rounded down, `top` keys or more reach the q-th largest of the lists' keys number j where
// q * (j + 1) >= top: what reaches that floor, a few at the head of every list, is gathered and sorted by counting.  (One
// round of the whole wave per alternative took 0.2 us each: a row of 32 parts, 20 alternatives 8.0 us, 4.5 so.)  A launch of its
// own: joining in the part that is done last, which takes a counter, stores and loads past the caches, saves nothing for one row
// (10.0 and 9.9 us) and costs 8192 rows of 65,536 203 -> 235.
template <typename T>
__global__ void __launch_bounds__(256) k_logprobs_join(PartArgs p) {
    extern __shared__ uint64_t join_lds[];
    const LogprobArgs &a = p.a;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), top = a.top, parts = p.parts;
    const int64_t row = (int64_t)blockIdx.x * (blockDim.x >> 6) + wave;
    if (row >= a.n) return;  // (no barriers below)
    CodeScore cs;
    cs.read(a, row, T());
    const int total = parts * top;
    const uint64_t *keys = p.keys + row * total;
    uint64_t *lists = join_lds + wave * (2 * total + 8), *found = lists + total;
    for (int i = lane; i < total; i += 512) {
        uint64_t k[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) k[u] = i + 64 * u < total ? keys[i + 64 * u] : 0;
#pragma unroll
        for (int u = 0; u < 8; ++u)
            if (i + 64 * u < total) lists[i + 64 * u] = k[u];
    }
    const float *sums = p.sums + (row * parts + min(lane, parts - 1)) * 3, c = a.beta * kLog2e;
    const float pm = sums[0], pS = lane < parts ? sums[1] : 0.0f, pW = lane < parts ? sums[2] : 0.0f, m = group_max<64>(pm);
    const float d = fmaxf((pm - (Sums::is_bad(m) || m == kNegInf ? 0.0f : m)) * c, -200.0f);
    const float f = lane < parts ? __builtin_amdgcn_exp2f(d) : 0.0f;
    const RowSums r = row_sums({m, group_sum<64>(f * pS), group_sum<64>(f * __builtin_fmaf(pS, d, pW))});
    if (lane == 0) write_row(a, row, r, cs);
    if (top == 0) return;
    wave_sync();
    const uint64_t *list = lists + min(lane, parts - 1) * top;
    const int j = (top - 1) / parts, q = (top + j) / (j + 1);
    const uint64_t probe = lane < parts ? list[j] : 0;
    int above = 0;
    for (int o = 0; o < parts; ++o) {
        const uint64_t other = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(probe >> 32), o) << 32 |
                               (uint32_t)__builtin_amdgcn_readlane((int)probe, o);
        above += other > probe;
    }
    // (keys are different but for those that are 0: where fewer than q are not, the floor is 1)
    const unsigned long long who = __ballot(lane < parts && probe != 0 && above == q - 1);
    const int at = who ? __ffsll(who) - 1 : 0;
    const uint64_t floor = !who ? 1 : (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(probe >> 32), at) << 32 |
                                          (uint32_t)__builtin_amdgcn_readlane((int)probe, at);
    int count = 0;
    uint64_t next = lane < parts ? list[0] : 0;
    for (int i = 1;; ++i) {
        const unsigned long long more = __ballot(next >= floor);
        if (!more) break;
        if (next >= floor) found[count + __popcll(more & ((1ull << lane) - 1))] = next;
        count += __popcll(more);
        next = next >= floor && i < top ? list[i] : 0;
    }
    if (lane < 8) found[count + lane] = 0;
    if (lane < top) lists[lane] = 0;  // (the best of all; the lists have been read)
    wave_sync();
    for (int i = lane; i < count; i += 64) {
        const uint64_t mine = found[i];
        const int rank = keys_above(found, count, mine);
        if (rank < top) lists[rank] = mine;
    }
    wave_sync();
    if (lane < top) write_alternative(a, row, lane, lists[lane], r);
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

// 2^d with d = (x - m) * c - L2 is the probability (c = beta * log2 e, L2 = L * log2 e), d * ln 2 its logarithm; both held above 2^-200,
// which is zero in f32.  A and B hold the factors: beta * (g_lp + g_H * (log p + H)) = A * d + B; where one of them is beyond f32, a
// probability of zero still makes a gradient of zero (a compare and a choice per value: 1M rows of 64 bf16 57.3 -> 58.3 us, longer rows alike).
// A lane has NV vectors of a row, G lanes a row or (G = 256, blockIdx.y) a piece of one; its code's own term is added where one of its
// vectors holds the code.  A vector that would pass the row's end is read from elsewhere (Share) but only its own values are
// written, one by one, so that the gradient may take the scores' place.
template <typename T, int G, int NV>
__global__ void __launch_bounds__(256) k_logprobs_grad(GradArgs a) {
    typedef Share<T, G, NV> S;
    typedef typename T::Raw Raw;
    constexpr int VEC = S::VEC;
    const int lane = threadIdx.x & (G - 1);
    const int64_t mine = (int64_t)blockIdx.x * (256 / G) + threadIdx.x / G, row = min(mine, a.n - 1);
    const int lo = G == 256 ? (int)blockIdx.y * (G * S::E) : 0, hi = a.k;
    S r;
    r.fetch_once((const Raw *)a.s + row * a.ld, lo, hi, lane);
    Raw *to = (Raw *)a.grad + row * a.ld_grad;
    const float m = a.max[row], L = a.logsum[row], gh = a.g_entropy ? a.g_entropy[row] : 0.0f, H = a.g_entropy ? a.entropy[row] : 0.0f;
    int64_t code = -1;
    float gl = 0.0f;
    if (a.g_logprob) {
        code = code_at(a.codes, a.code_bytes, row * a.code_stride);
        if (code >= 0) gl = a.g_logprob[row];
    }
    const bool none = m == kNegInf, bad = L != L || code >= a.k;
    const float from = none ? 0.0f : m, c = a.beta * kLog2e, L2 = none ? 0.0f : L * kLog2e, own = a.beta * gl;
    const float A = none ? 0.0f : a.beta * gh * kLn2, B = none ? 0.0f : bad ? __builtin_nanf("") : a.beta * __builtin_fmaf(gh, H, gl);
    const float gone = bad && !none ? B : 0.0f;  // the gradient where the probability is zero, also times an infinite factor
    if (none) code = -1;  // (before all else: such a row's gradient is zero, whatever its code)
    const bool past = ((uintptr_t)a.grad & 127) == 0 && a.ld_grad % (128 / (int)sizeof(Raw)) == 0;  // whole lines pass the caches (412 -> 401 us)
#pragma unroll
    for (int u = 0; u < NV; ++u) {
        if (u > 0 && lo + u * G * VEC >= hi) break;  // uniform
        const int at = lo + (u * G + lane) * VEC, base = S::base(u, lane, lo, hi);
        float x[VEC];
        S::values(r.raw[u], x);
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            const float d = fmaxf(__builtin_fmaf(x[v] - from, c, -L2), -200.0f);
            const float p = __builtin_amdgcn_exp2f(d);
            x[v] = p == 0.0f ? gone : p * -__builtin_fmaf(d, A, B);
        }
        const int64_t hit = code - base;
        if (hit >= 0 && hit < VEC) {
#pragma unroll
            for (int v = 0; v < VEC; ++v) x[v] = v == hit ? x[v] + own : x[v];
        }
        typename S::Piece o;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            if constexpr (sizeof(Raw) == 4)
                o.w[q] = __float_as_uint(x[q]);
            else
                o.w[q] = (uint32_t)T::down(x[2 * q]) | (uint32_t)T::down(x[2 * q + 1]) << 16;
        }
        if (mine >= a.n || at >= hi) continue;
        if (base == at && past)
            __builtin_nontemporal_store(__builtin_bit_cast(AnyWords, o), reinterpret_cast<AnyWords *>(to + at));
        else if (base == at)
            *reinterpret_cast<typename S::Piece *>(to + at) = o;
        else
#pragma unroll
            for (int v = 0; v < VEC; ++v)
                if (base + v >= at) to[base + v] = T::down(x[v]);
    }
}

// Rows shorter than a vector: a lane each.
template <typename T>
__global__ void __launch_bounds__(256) k_logprobs_grad_tiny(GradArgs a) {
    const int64_t row = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (row >= a.n) return;
    const typename T::Raw *s = (const typename T::Raw *)a.s + row * a.ld;
    const float m = a.max[row], L = a.logsum[row], gh = a.g_entropy ? a.g_entropy[row] : 0.0f, H = a.g_entropy ? a.entropy[row] : 0.0f;
    const int64_t code = a.g_logprob ? code_at(a.codes, a.code_bytes, row * a.code_stride) : -1;
    const float gl = code >= 0 ? a.g_logprob[row] : 0.0f;
    for (int j = 0; j < a.k; ++j) {
        const float lp = fmaxf(a.beta * (T::up(s[j]) - m) - L, -140.0f);
        const float p = __builtin_amdgcn_exp2f(lp * kLog2e);
        const float g = a.beta * ((j == code ? gl : 0.0f) - (p == 0.0f ? 0.0f : p * (gl + gh * (lp + H))));
        ((typename T::Raw *)a.grad)[row * a.ld_grad + j] = T::down(m == kNegInf ? 0.0f : L != L || code >= a.k ? __builtin_nanf("") : g);
    }
}

}  // namespace vq
