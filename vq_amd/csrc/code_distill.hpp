// A loss of rows of scores against a teacher's best alternatives, and its gradient.
//
// This translation unit must be compiled with -ffp-contract=off.
//
// A row of scores s_j and the teacher's alternatives, codes c_t with log probabilities; q_t are the teacher's probabilities, r what they
// leave (0 where the alternatives are to sum to one), p_j those of the scores, R the probability of all codes that are no
// alternative.  Loss = sum_t q_t (log q_t - log p_{c_t}) + r (log r - log R); its gradient by s_j, with Q = sum_t q_t + r:
//   beta (Q p_j - q_j)            of an alternative (q_j: the sum of those with this code)
//   beta (Q R - r) p_j / R        of another code
// So the other codes' gradients are one exponential each, by a factor and an offset that the row's codes have in common; the
// alternatives', at most 64 numbers, are written over what that makes of their codes.  Where R is asked for, the sums of the two kinds are
// kept apart from the start; where the alternatives' is the smaller, log R is log1p of what they hold, and Q R - r is Q + (Q + r)(R - 1):
// neither is a small difference of large numbers.
#pragma once
#include "code_rows.hpp"
#include "code_rules.hpp"
#include "wide_exp.hpp"

namespace vq {

struct DistillArgs {
    const void *s;
    int64_t n, ld;
    int k;
    float beta;
    int top;
    const float *lp;
    const int32_t *code;
    int64_t ld_teacher;
    int rest, split;  // split: the codes that are no alternative have sums of their own
    float *loss, *max, *logsum, *logrest;  // (the backward call reads the last three)
    const float *g;
    void *grad;
    int64_t ld_grad;
    int parts;
    float *sums;  // [row][part][2]: largest score of the codes that are no alternative, their sum
    float *rest_max, *rest_sum;  // the same of a row, from its parts for its gradient
};

// A row's alternatives, one per lane of a wave.
constexpr int kSlots = 4096;
struct Teacher {
    int code = -1;
    bool has = false, first = false;  // an alternative; the first with its code
    bool some, bad;                   // (uniform) the row has any; one of them is no code or no number
    float q = 0.0f, log_q = 0.0f, q_code = 0.0f;  // probability, its logarithm, the sum of the probabilities with this code
    double Q = 0.0;                   // (uniform)

    // where the codes are needed only: which of them there are
    __device__ __forceinline__ void names(const DistillArgs &a, int64_t row, int lane) {
        float l = kNegInf;
        if (lane < a.top) {
            code = a.code[row * a.ld_teacher + lane];
            l = a.lp[row * a.ld_teacher + lane];
        }
        has = code >= 0 && l != kNegInf;
        log_q = l;
    }
    // slots: the wave's own, with anything in them
    __device__ __forceinline__ void read(const DistillArgs &a, int64_t row, int lane, uint8_t *slots) {
        names(a, row, lane);
        const unsigned long long who = __ballot(has);
        some = who != 0;
        bad = __ballot(has && (code >= a.k || !(log_q < __builtin_inff()))) != 0;
        // probabilities in 64 bits: what they leave of one may be small
        float most = 0.0f, l = has ? log_q : kNegInf;
        if (!a.rest) most = group_max<64>(l);
        const double e = has && !bad ? exp2_wide(((double)l - (double)most) * kLog2e64) : 0.0;
        double sum = wave_sum(e);
        if (a.rest) {
            q = (float)e;
            Q = sum;
        } else if (some) {
            q = (float)e * __builtin_amdgcn_rcpf((float)sum);
            log_q = l - most - __builtin_amdgcn_logf((float)sum) * kLn2;
            Q = 1.0;
        }
        first = has;
        q_code = has ? q : 0.0f;
        // The same code twice is rare: where every alternative finds its own mark in the slot of its code's lowest bits there is none.  (Else the
        // sums of the probabilities with this code, in the order of the list.)
        if (has) slots[code & (kSlots - 1)] = (uint8_t)lane;
        wave_sync();
        if (__ballot(has && slots[code & (kSlots - 1)] != lane) == 0) return;
        if (has) q_code = 0.0f;
        for (int t = 0; t < a.top; ++t) {
            if (!(who >> t & 1)) continue;  // uniform
            const int other = __builtin_amdgcn_readlane(code, t);
            const float other_q = __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(q), t));
            if (has && other == code) {
                q_code += other_q;
                if (t < lane) first = false;
            }
        }
    }
};

// What a row's gradients have in common: code j, no alternative, has C * 2^((s_j - from) * c - off), zero where that power is; a NaN
// in a row whose sums are NaN.  The power is a probability or a share of the rest: no rounding of far scores makes it more than one.
struct RowGrad {
    float C, from, off, gone;
    __device__ __forceinline__ float operator()(float s, float c) const {
        const float p = __builtin_amdgcn_exp2f(__builtin_amdgcn_fmed3f(__builtin_fmaf(s - from, c, -off), -200.0f, 0.0f));
        return p == 0.0f ? gone : C * p;
    }
};
// The gradient of a row, from m, L, the log of R and the scores at the alternatives' codes (a lane each): the common part, and value, a lane's
// own.  The other codes' shares of the rest are relative to the rest's largest score mr and their sum Sr where these are at hand (mr above
// -inf), otherwise to m, L and log R, whose rounding they then have: some six steps of 2^-24 of log R, so that from FAR on, where that is more than a
// third, nothing is known of them and their probability counts as the zero that it nearly is.
__device__ __forceinline__ RowGrad row_grad(const DistillArgs &a, int64_t row, const Teacher &t, float m, float L, float log_rest, float score,
                                            float *value, float mr, float Sr) {
    constexpr float FAR = -1048576.0f;
    RowGrad o{0.0f, 0.0f, 0.0f, 0.0f};
    *value = 0.0f;
    const bool none = m == kNegInf;
    if (!t.some || none) return o;  // (uniform)
    const float c = a.beta * kLog2e, bg = a.beta * a.g[row];
    const bool open = a.rest && log_rest != kNegInf;
    const float r = open ? (float)fmax(0.0, 1.0 - t.Q) : 0.0f, total = (float)t.Q + r;
    const bool bad = t.bad || L != L;
    o.from = bad ? 0.0f : m;
    if (bad) {
        o.C = o.gone = *value = __builtin_nanf("");
        return o;
    }
    o.off = L * kLog2e;
    o.C = bg * total;
    if (open) {
        o.C = bg * (log_rest > -0.5f ? __builtin_fmaf(total, expm1f(log_rest), (float)t.Q)
                                     : __builtin_fmaf(total, __builtin_amdgcn_exp2f(log_rest * kLog2e), -r));
        o.off = fmaxf((L + log_rest) * kLog2e, -3e38f);
        if (mr != kNegInf)
            o.from = mr, o.off = __builtin_amdgcn_logf(Sr);
        else if (log_rest < FAR)
            o.C = 0.0f;
    }
    const float p = __builtin_amdgcn_exp2f(fmaxf(__builtin_fmaf(score - m, c, -L * kLog2e), -200.0f));
    *value = bg * __builtin_fmaf(total, p, -t.q_code);
    return o;
}

// The sums of a row: from the largest score mr and the sum Sr of its codes, or (split) of those that are no alternative, and the scores at
// the alternatives' codes.  Log R is -inf where no other code can be, and nowhere else: what lies below f32's lowest number is written as that.  A
// term of the loss whose log probability lies there is formed in 64 bits, since the teacher's probability may bring it back.
struct RowLoss {
    float m, L, log_rest, loss;
};
__device__ __forceinline__ RowLoss row_loss(const DistillArgs &a, const Teacher &t, float mr, float Sr, float score) {
    constexpr float LOWEST = -3.402823466e38f;
    const float c = a.beta * kLog2e, mine = a.split && t.first ? score : kNegInf;
    const float m = larger(group_max<64>(mine), mr);
    const float from = Sums::is_bad(m) || m == kNegInf ? 0.0f : m;
    const float e = __builtin_amdgcn_exp2f(larger_or_nan((mine - from) * c, -200.0f));
    const float A = group_sum<64>(e), S = __builtin_fmaf(Sr, __builtin_amdgcn_exp2f(fmaxf((mr - from) * c, -200.0f)), A);
    const RowSums sums = row_sums(Sums(m, S, 0.0f));
    RowLoss o{sums.m, sums.L, kNegInf, 0.0f};
    const bool bad = sums.L != sums.L, others = a.split && mr != kNegInf;
    const auto beyond = [&](float s, float rest) { return (double)a.beta * ((double)s - (double)m) + (double)rest; };  // a log probability in 64 bits
    if (bad)
        o.log_rest = sums.L;
    else if (others && A <= 0.5f * S)
        o.log_rest = log1pf(-A * __builtin_amdgcn_rcpf(S));
    else if (others)
        o.log_rest = fmaxf(fminf(2.0f * a.beta * __builtin_fmaf(0.5f, mr, -0.5f * m) + (__builtin_amdgcn_logf(Sr) * kLn2 - sums.L), 0.0f), LOWEST);
    const float log_p = sums.m == kNegInf ? kNegInf : log_probability(a.beta, score, sums);
    float term = t.q > 0.0f ? t.q * (t.log_q - log_p) : 0.0f;
    if (t.q > 0.0f && log_p == kNegInf && score > kNegInf) term = (float)((double)t.q * ((double)t.log_q - beyond(score, -sums.L)));
    float loss = group_sum<64>(term);
    if (a.rest && o.log_rest != kNegInf) {
        const float r = (float)fmax(0.0, 1.0 - t.Q);
        if (r > 0.0f) {
            const float log_r = t.Q < 0.5 ? log1pf(-(float)t.Q) : __builtin_amdgcn_logf(r) * kLn2;
            if (o.log_rest > LOWEST)
                loss += r * (log_r - o.log_rest);
            else
                loss += (float)((double)r * ((double)log_r - beyond(mr, __builtin_amdgcn_logf(Sr) * kLn2 - sums.L)));
        }
    }
    o.loss = !t.some ? 0.0f : t.bad || bad ? __builtin_nanf("") : loss;
    return o;
}
__device__ __forceinline__ void write_loss(const DistillArgs &a, int64_t row, const RowLoss &r) {
    if (a.loss) a.loss[row] = r.loss;
    if (a.max) a.max[row] = r.m;
    if (a.logsum) a.logsum[row] = r.L;
    if (a.logrest) a.logrest[row] = r.log_rest;
}

template <int WAVES> __device__ __forceinline__ void row_sync() {
    if constexpr (WAVES == 1)
        wave_sync();
    else
        __syncthreads();
}

// Which codes of a row, or of a part of it, are alternatives: a byte in LDS per vector of a lane, a bit per code.
template <typename T, int LANES, int NV> struct Marks {
    static constexpr int VEC = Held<T, LANES, NV>::VEC;
    uint32_t words[LANES * NV / 4];
    __device__ __forceinline__ void clear(int lane) {
        for (int i = lane; i < LANES * NV / 4; i += LANES) words[i] = 0;
    }
    __device__ __forceinline__ void set(int place) { atomicOr(&words[place / VEC / 4], 1u << (place / VEC % 4 * 8 + place % VEC)); }
    __device__ __forceinline__ uint32_t of(int u, int lane) const { return reinterpret_cast<const uint8_t *>(words)[u * LANES + lane]; }
};

// Writes the gradients of a lane's codes, as if none of them were an alternative.
template <typename T, int LANES, int NV>
__device__ __forceinline__ void write_grad(const DistillArgs &a, const Held<T, LANES, NV> &x, const RowGrad &row, typename T::Raw *to, int lo, int hi, int lane) {
    typedef Held<T, LANES, NV> H;
    const float c = a.beta * kLog2e;
    const bool past = ((uintptr_t)a.grad & 127) == 0 && a.ld_grad % (128 / (int)sizeof(typename T::Raw)) == 0;  // whole lines pass the caches
#pragma unroll
    for (int u = 0; u < NV; ++u) {
        const int at = lo + (u * LANES + lane) * H::VEC;
        if (lo + u * LANES * H::VEC >= hi) break;  // uniform
        float y[H::VEC];
#pragma unroll
        for (int v = 0; v < H::VEC; ++v) y[v] = row(x.at(u, v), c);
        if (at + H::VEC <= hi) {
            typename H::Piece o;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                if constexpr (sizeof(typename T::Raw) == 4)
                    o.w[q] = __float_as_uint(y[q]);
                else
                    o.w[q] = (uint32_t)T::down(y[2 * q]) | (uint32_t)T::down(y[2 * q + 1]) << 16;
            }
            if (past)
                __builtin_nontemporal_store(__builtin_bit_cast(AnyWords, o), reinterpret_cast<AnyWords *>(to + at));
            else
                *reinterpret_cast<typename H::Piece *>(to + at) = o;
        } else {
#pragma unroll
            for (int v = 0; v < H::VEC; ++v)
                if (at + v < hi) to[at + v] = T::down(y[v]);
        }
    }
}

// The largest score and the sum of a wave's codes, or (split) of those that are no alternative: these are dropped.  The scores stay as they are
// stored and are converted twice: 64 of them as floats beside would not fit the registers of a row of sixteen waves.
template <typename T, int LANES, int NV>
__device__ __forceinline__ Sums code_sums(const DistillArgs &a, Held<T, LANES, NV> &x, const Marks<T, LANES, NV> &marks, int lane) {
    typedef Held<T, LANES, NV> H;
    float m = kNegInf;
#pragma unroll
    for (int u = 0; u < NV; ++u) {
        if (a.split) {
            const uint32_t some = marks.of(u, lane);
            if (some) {
#pragma unroll
                for (int v = 0; v < H::VEC; ++v)
                    if (some >> v & 1) x.drop(u, v);
            }
        }
#pragma unroll
        for (int v = 0; v < H::VEC; v += 2) m = larger(larger(x.at(u, v), x.at(u, v + 1)), m);
    }
    // as the sums of a row in floats are made (Sums)
    Sums s(group_max<64>(m), 0.0f, 0.0f);
    const float c = a.beta * kLog2e, from = Sums::is_bad(s.m) || s.m == kNegInf ? 0.0f : s.m, M = from * c;
    const bool far = fabsf(M) >= 1e6f;  // uniform
    s.r = far ? 0.0f : __builtin_fmaf(from, c, -M);
    if (!far) {
#pragma unroll
        for (int u = 0; u < NV; ++u)
#pragma unroll
            for (int v = 0; v < H::VEC; ++v) s.add(__builtin_fmaf(x.at(u, v), c, -M));
    } else {
#pragma unroll
        for (int u = 0; u < NV; ++u)
#pragma unroll
            for (int v = 0; v < H::VEC; ++v) s.add((x.at(u, v) - from) * c);
    }
    s.S = group_sum<64>(s.S);
    s.away();
    return s;
}

// Sums of parts of a row, one per lane below `parts`, to the row's.
__device__ __forceinline__ void join_rest(const DistillArgs &a, float pm, float pS, bool mine, float *mr, float *Sr) {
    const float m = group_max<64>(mine ? pm : kNegInf);
    const float f = mine ? __builtin_amdgcn_exp2f(fmaxf((pm - (Sums::is_bad(m) || m == kNegInf ? 0.0f : m)) * (a.beta * kLog2e), -200.0f)) : 0.0f;
    *mr = m;
    *Sr = group_sum<64>(mine ? f * pS : 0.0f);
}

// Rows that WAVES waves hold: the loss, and the gradient from the same registers where it is asked for, so that the row is read once.  One wave
// keeps the row's teacher.  Bound by memory: 8192 rows of 65,536 bf16 with 20 alternatives, loss and gradient, 432 us = 4.97 TB/s (with reads that
// pass the caches, too, 451; with the scores as floats beside their stored form, which does not fit the registers, 624).
template <typename T, int WAVES, int NV>
__global__ void __launch_bounds__(WAVES == 1 ? 256 : 64 * WAVES) k_distill_row(DistillArgs a) {
    typedef typename T::Raw Raw;
    constexpr int LANES = 64 * WAVES, ROWS = WAVES == 1 ? 4 : 1;
    __shared__ Marks<T, LANES, NV> marks_of[ROWS];
    __shared__ uint8_t slots_of[ROWS][kSlots];
    __shared__ float joined[2][16];
    __shared__ RowGrad common;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, place = WAVES == 1 ? lane : threadIdx.x;
    const int64_t row = (int64_t)blockIdx.x * ROWS + (WAVES == 1 ? wave : 0);
    if (row >= a.n) return;  // (WAVES == 1: no barriers below)
    auto &marks = marks_of[WAVES == 1 ? wave : 0];
    const bool leads = WAVES == 1 || wave == 0;
    const Raw *s = (const Raw *)a.s + row * a.ld;
    Raw *to = (Raw *)a.grad + row * a.ld_grad;
    Held<T, LANES, NV> x;
    x.load(s, 0, a.k, place);
    Teacher t;
    float score = kNegInf, value = 0.0f;
    if (leads) {
        t.read(a, row, lane, slots_of[WAVES == 1 ? wave : 0]);
        if (t.has && t.code < a.k) score = T::up(s[t.code]);
    }
    if (a.split) {  // uniform
        marks.clear(place);
        row_sync<WAVES>();
        if (leads && t.first && t.code < a.k) marks.set(t.code);
        row_sync<WAVES>();
    }
    const Sums sums = code_sums(a, x, marks, place);
    float mr = sums.m, Sr = sums.S;
    if constexpr (WAVES > 1) {
        if (lane == 0) joined[0][wave] = mr, joined[1][wave] = Sr;
        __syncthreads();
    }
    RowGrad grad;
    if (leads) {
        if constexpr (WAVES > 1) join_rest(a, joined[0][lane & 15], joined[1][lane & 15], lane < WAVES, &mr, &Sr);
        const RowLoss o = row_loss(a, t, mr, Sr, score);
        if (lane == 0) write_loss(a, row, o);
        if (a.grad) {
            grad = row_grad(a, row, t, o.m, o.L, o.log_rest, score, &value, mr, Sr);
            if constexpr (WAVES > 1)
                if (lane == 0) common = grad;
        }
    }
    if (!a.grad) return;  // uniform
    if constexpr (WAVES > 1) {
        __syncthreads();
        grad = common;
    }
    write_grad(a, x, grad, to, 0, a.k, place);
    row_sync<WAVES>();  // the alternatives' go over these
    if (leads && t.first && t.code < a.k) to[t.code] = T::down(value);
}

// A part of a long row: the largest score and the sum of its codes, or of those that are no alternative.
template <typename T, int NV>
__global__ void __launch_bounds__(256) k_distill_part(DistillArgs a) {
    typedef typename T::Raw Raw;
    __shared__ Marks<T, 256, NV> marks;
    __shared__ float joined[2][4];
    const int64_t row = blockIdx.x / (unsigned)a.parts;
    const int part = (int)(blockIdx.x % (unsigned)a.parts), size = 256 * Held<T, 256, NV>::E, lo = part * size, hi = min(a.k, lo + size);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    Held<T, 256, NV> x;
    x.load((const Raw *)a.s + row * a.ld, lo, hi, tid);
    if (a.split) {  // uniform
        Teacher t;
        if (wave == 0) t.names(a, row, lane);
        marks.clear(tid);
        __syncthreads();
        if (t.has && t.code >= lo && t.code < hi) marks.set(t.code - lo);
        __syncthreads();
    }
    const Sums sums = code_sums(a, x, marks, tid);
    if (lane == 0) joined[0][wave] = sums.m, joined[1][wave] = sums.S;
    __syncthreads();
    if (wave) return;
    float m, S;
    join_rest(a, joined[0][lane & 3], joined[1][lane & 3], lane < 4, &m, &S);
    if (lane == 0) a.sums[(int64_t)blockIdx.x * 2] = m, a.sums[(int64_t)blockIdx.x * 2 + 1] = S;
}

// A wave joins the parts of a row.
template <typename T>
__global__ void __launch_bounds__(256) k_distill_join(DistillArgs a) {
    __shared__ uint8_t slots_of[4][kSlots];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t row = (int64_t)blockIdx.x * 4 + wave;
    if (row >= a.n) return;
    const float *sums = a.sums + (row * a.parts + min(lane, a.parts - 1)) * 2;
    const float pm = sums[0], pS = sums[1];
    Teacher t;
    t.read(a, row, lane, slots_of[wave]);
    const float score = t.has && t.code < a.k ? T::up(((const typename T::Raw *)a.s)[row * a.ld + t.code]) : kNegInf;
    float mr, Sr;
    join_rest(a, pm, pS, lane < a.parts, &mr, &Sr);
    const RowLoss o = row_loss(a, t, mr, Sr, score);
    if (lane == 0) write_loss(a, row, o);
    if (lane == 0 && a.rest_max) a.rest_max[row] = mr, a.rest_sum[row] = Sr;
}

// The gradient alone, from m, L and log R as the loss's call left them (in that call of rows in parts also from the rest's own sums): a row, or (blockIdx.y) a piece of one, per WAVES waves.  Bound by memory:
// 2048 rows of 65,536 f32 199 us = 5.4 TB/s with reads and whole lines that pass the caches (210 without).
template <typename T, int WAVES, int NV>
__global__ void __launch_bounds__(256) k_distill_grad(DistillArgs a) {
    typedef typename T::Raw Raw;
    constexpr int LANES = 64 * WAVES, ROWS = 4 / WAVES;
    __shared__ uint8_t slots_of[ROWS][kSlots];
    __shared__ RowGrad common;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, place = WAVES == 1 ? lane : threadIdx.x;
    const int64_t row = (int64_t)blockIdx.x * ROWS + (WAVES == 1 ? wave : 0);
    if (row >= a.n) return;  // (WAVES == 1: no barriers below)
    const bool leads = WAVES == 1 || wave == 0;
    const Raw *s = (const Raw *)a.s + row * a.ld;
    Raw *to = (Raw *)a.grad + row * a.ld_grad;
    const int size = LANES * Held<T, LANES, NV>::E, lo = blockIdx.y * size, hi = min(a.k, lo + size);
    Held<T, LANES, NV> x;
    x.template load<true>(s, lo, hi, place);
    RowGrad grad;
    Teacher t;
    float value = 0.0f;
    if (leads) {
        t.read(a, row, lane, slots_of[WAVES == 1 ? wave : 0]);
        const float score = t.has && t.code >= lo && t.code < hi ? T::up(s[t.code]) : kNegInf;
        grad = row_grad(a, row, t, a.max[row], a.logsum[row], a.rest ? a.logrest[row] : kNegInf, score, &value, a.rest_max ? a.rest_max[row] : kNegInf,
                        a.rest_max ? a.rest_sum[row] : 0.0f);
        if constexpr (WAVES > 1)
            if (lane == 0) common = grad;
    }
    if constexpr (WAVES > 1) {
        __syncthreads();  // (the scores at the alternatives' codes have been read, too)
        grad = common;
    }
    write_grad(a, x, grad, to, lo, hi, place);
    row_sync<WAVES>();  // the alternatives' go over these
    if (leads && t.first && t.code >= lo && t.code < hi) to[t.code] = T::down(value);
}

}  // namespace vq
