// Drafted codes against the probabilities of scores, and the code that comes next.
//
// This translation unit must be compiled with -ffp-contract=off.
//
// Probabilities p of a position's target row and q of its draft's (of a draft without scores: 1 for its code).  A drafted code c stays
// where u q_c < p_c.  At the first that does not the next code is drawn from max(p - q, 0), where all stay from p behind the last; drawn with
// v: the first code at which the sum of the weights so far is above v times all of it.  Which code that is hangs on sums that lie
// close together, so exponentials and sums are in 64 bits; a wave's add is as fast in 64 bits as in 32 here.
#pragma once
#include "code_rows.hpp"
#include "code_rules.hpp"
#include "wide_exp.hpp"

namespace vq {

struct VerifyArgs {
    const void *target, *drafts;
    int64_t ld_target, ld_draft;
    double c_target, c_draft;  // beta * log2 e
    int n, draft, k, parts;
    const void *codes;
    int code_bytes;
    int64_t code_stride;
    const float *uniform;
    int64_t ld_uniform;
    int32_t *accepted, *out;
    int64_t ld_out;
    // per part of a row its largest score (-inf for none, NaN where it holds one) and the sum of 2^((s - largest) c); the rows of the
    // targets, then of the drafts.  Without scores of the drafts a drafted code is left out of its row.
    float *most;
    double *sum;
    double *left;  // per sequence and part: the sum of max(p - q, 0)
    int left_parts;  // parts of a workgroup that makes these sums
    int64_t first_draft() const { return (int64_t)n * (draft + 1); }
};

// The drafted codes of a sequence: lane d has code d; returns how many there are before the first that is none.
__device__ __forceinline__ int drafted(const VerifyArgs &a, int64_t seq, int lane, int64_t *code) {
    *code = lane < a.draft ? code_at(a.codes, a.code_bytes, seq * a.code_stride + lane) : -1;
    return __ffsll(__ballot(*code < 0)) - 1;  // (lane 63 has none)
}

constexpr int kVerifyEach = kVerifyPart / 256;  // codes of a lane

template <typename T>
__global__ void __launch_bounds__(256) k_verify_part(VerifyArgs a) {
    typedef typename T::Raw Raw;
    typedef Held<T, 256, kVerifyEach * (int)sizeof(Raw) / 16> H;
    __shared__ float most_of[4];
    __shared__ double sum_of[4];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int64_t row = blockIdx.x / (unsigned)a.parts, targets = (int64_t)a.n * (a.draft + 1);
    const int part = (int)(blockIdx.x % (unsigned)a.parts), lo = part * kVerifyPart, hi = min(a.k, lo + kVerifyPart);
    const bool draft = row >= targets;
    const int64_t seq = draft ? (row - targets) / a.draft : row / (a.draft + 1);
    const int pos = (int)(draft ? (row - targets) % a.draft : row % (a.draft + 1));
    H x;
    int64_t code;
    int length = a.draft;
    if (a.code_bytes == 4 || !a.drafts) length = drafted(a, seq, lane, &code);  // (unsigned codes end no draft)
    if (pos >= length + (draft ? 0 : 1)) return;  // uniform: a row that nothing is drafted for
    x.load(draft ? (const Raw *)a.drafts + (row - targets) * a.ld_draft : (const Raw *)a.target + row * a.ld_target, lo, hi, tid);
    if (!a.drafts && pos < length) {  // the row without its drafted code
        const int64_t c = (int64_t)__shfl((int)code, pos) - lo;
        if (c >= 0 && c < hi - lo) {
            const int place = (int)c / H::VEC;
            if (place % 256 == tid) {
#pragma unroll
                for (int u = 0; u < kVerifyEach / H::VEC; ++u)
#pragma unroll
                    for (int v = 0; v < H::VEC; ++v)
                        if (u == place / 256 && v == (int)c % H::VEC) x.drop(u, v);
            }
        }
    }
    float m = kNegInf;
#pragma unroll
    for (int u = 0; u < kVerifyEach / H::VEC; ++u)
#pragma unroll
        for (int v = 0; v < H::VEC; ++v) m = larger_or_nan(m, x.at(u, v));
    m = __uint_as_float(over_group<64>(__float_as_uint(m), __float_as_uint(kNegInf), [](uint32_t p, uint32_t q) {
        return __float_as_uint(larger_or_nan(__uint_as_float(p), __uint_as_float(q)));
    }));
    if (lane == 0) most_of[wave] = m;
    __syncthreads();
    m = larger_or_nan(larger_or_nan(most_of[0], most_of[1]), larger_or_nan(most_of[2], most_of[3]));
    double sum = 0.0;
    if (m > kNegInf && m < __builtin_inff()) {  // uniform
        const double c = draft ? a.c_draft : a.c_target, from = m, least = -1000.0 / c;  // (the difference first: of scores of 1e38 a rounded product leaves too much)
#pragma unroll
        for (int u = 0; u < kVerifyEach / H::VEC; ++u)
#pragma unroll
            for (int v = 0; v < H::VEC; ++v) sum += exp2_of(fmax((double)x.at(u, v) - from, least), c);
    }
    sum = wave_sum(sum);
    if (lane == 0) sum_of[wave] = sum;
    __syncthreads();
    if (tid == 0) a.most[blockIdx.x] = m, a.sum[blockIdx.x] = sum_of[0] + sum_of[1] + sum_of[2] + sum_of[3];
}

// What the drafts of a sequence come to.
struct Verdict {
    int accepted, length;
    int refused;          // the first drafted code that does not stay, -1 for none
    bool bad;             // the position behind the accepted codes cannot be answered
    double mp, Sp, mq, Sq;  // its rows' largest scores and sums; of a refused draft without scores its code is left out of Sp
};
struct VerdictLds {
    double m[2][kMaxDraft + 1], S[2][kMaxDraft + 1];
    Verdict out;
};

// By a workgroup of four waves: each joins the parts of every fourth row, the first decides.  code: a lane of the first wave's drafted code.
template <typename T> __device__ __forceinline__ Verdict verdict(const VerifyArgs &a, int64_t seq, VerdictLds &l, int64_t *code) {
    typedef typename T::Raw Raw;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int length = drafted(a, seq, lane, code), rows = length + 1 + (a.drafts ? length : 0);
    const bool here = lane <= length, asked = lane < length, known = asked && *code < a.k;
    float s = 0.0f, t = 0.0f, u = 0.0f;  // lane d: the scores of drafted code d, its random number
    if (wave == 0 && asked) {
        u = a.uniform[seq * a.ld_uniform + lane];
        if (known) {
            s = T::up(((const Raw *)a.target)[(seq * (a.draft + 1) + lane) * a.ld_target + *code]);
            if (a.drafts) t = T::up(((const Raw *)a.drafts)[(seq * a.draft + lane) * a.ld_draft + *code]);
        }
    }
    constexpr int AHEAD = 4;
    for (int r0 = wave; r0 < rows; r0 += 4 * AHEAD) {
        float most[AHEAD];
        double sum[AHEAD];
        const auto row_of = [&](int i) {
            const int r = min(r0 + 4 * i, rows - 1);
            return r <= length ? seq * (a.draft + 1) + r : (int64_t)a.n * (a.draft + 1) + seq * a.draft + (r - length - 1);
        };
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            const int64_t at = row_of(i) * a.parts + min(lane, a.parts - 1);
            most[i] = lane < a.parts ? a.most[at] : kNegInf;
            sum[i] = lane < a.parts ? a.sum[at] : 0.0;
        }
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            const int r = r0 + 4 * i;
            if (r >= rows) break;  // uniform
            const bool draft = r > length;
            const double c = draft ? a.c_draft : a.c_target;
            float m = most[i];
            bool bad = __ballot(m != m) != 0;
            m = group_max<64>(m);
            const auto scaled = [&](float pm, double ps) { return pm > kNegInf ? ps * exp2_wide(((double)pm - (double)m) * c) : 0.0; };
            double S;
            if (a.parts <= 64) {
                S = wave_sum(scaled(most[i], sum[i]));
            } else {  // the other parts, 64 at a time
                const int64_t at = row_of(i) * a.parts;
                for (int p = lane + 64; p - lane < a.parts; p += 64) {
                    const float o = p < a.parts ? a.most[at + p] : kNegInf;
                    bad = bad || __ballot(o != o) != 0;
                    m = larger(m, group_max<64>(o));
                }
                double mine = scaled(most[i], sum[i]);
                for (int p = lane + 64; p < a.parts; p += 64) mine += scaled(a.most[at + p], a.sum[at + p]);
                S = wave_sum(mine);
            }
            if (lane == 0) {
                const int d = draft ? r - length - 1 : r;
                l.m[draft][d] = m;
                l.S[draft][d] = bad || m == __builtin_inff() ? __builtin_nan("") : S;
            }
        }
    }
    __syncthreads();
    if (wave == 0) {
        double p = 0.0, q = 1.0;
        bool fine = here;
        const double mp = here ? l.m[0][lane] : 0.0, Sp = here ? l.S[0][lane] : 0.0;
        const bool scored = known && a.drafts;
        const double mq = scored ? l.m[1][lane] : 0.0, Sq = scored ? l.S[1][lane] : 1.0;
        if (known && !a.drafts) {
            // the row's code was left out of its sums
            const bool sound = s < __builtin_inff() && Sp == Sp;
            const double most = sound ? fmax(mp, (double)s) : 0.0;
            const double e = s == kNegInf || !sound ? 0.0 : exp2_wide(((double)s - most) * a.c_target);
            const double others = mp == -__builtin_inf() || !sound ? 0.0 : Sp * exp2_wide((mp - most) * a.c_target);
            p = sound ? e / (e + others) : __builtin_nan("");
            fine = p == p;
        } else if (scored) {
            fine = Sp > 0.0 && Sq > 0.0;
            if (fine) {
                p = exp2_wide(((double)s - mp) * a.c_target) / Sp;
                q = exp2_wide(((double)t - mq) * a.c_draft) / Sq;
            }
        } else if (here)
            fine = !asked && Sp > 0.0;
        const bool stays = asked && fine && (double)u * q < p;
        Verdict o;
        o.length = length;
        o.accepted = __ffsll(__ballot(!stays)) - 1;
        o.refused = o.accepted < length ? __shfl((int)*code, o.accepted) : -1;
        o.bad = !(__ballot(fine) >> o.accepted & 1);
        o.mp = __shfl(mp, o.accepted);
        o.Sp = __shfl(Sp, o.accepted);
        o.mq = __shfl(mq, o.accepted);
        o.Sq = __shfl(Sq, o.accepted);
        if (lane == 0) l.out = o;
    }
    __syncthreads();
    return l.out;
}

// The weights of the codes of the position behind the accepted ones.
struct Weights {
    double c_target, c_draft, mp, mq, by_p, by_q;
    int code;   // this one has none
    bool minus;  // max(p - q, 0), otherwise p
    __device__ __forceinline__ double operator()(float s, float t) const {
        const double p = exp2_wide(((double)s - mp) * c_target) * by_p;
        if (!minus) return p;
        return fmax(p - exp2_wide(((double)t - mq) * c_draft) * by_q, 0.0);
    }
};
__device__ __forceinline__ Weights weights(const VerifyArgs &a, const Verdict &o) {
    const bool minus = o.accepted < o.length && a.drafts;
    return {a.c_target, a.c_draft, o.mp, o.mq, minus ? 1.0 / o.Sp : 1.0, minus ? 1.0 / o.Sq : 0.0, minus ? -1 : o.refused, minus};
}

// 16 codes of a lane one after another, from a part of a row on.
template <typename T> __device__ __forceinline__ void lane_codes(const void *rows, int64_t row, int64_t ld, int at, int k, float (&x)[kVerifyEach]) {
    typedef typename T::Raw Raw;
    typedef Held<T, 1, kVerifyEach * (int)sizeof(Raw) / 16> H;
    H h;
    if (at >= k) {
#pragma unroll
        for (int e = 0; e < kVerifyEach; ++e) x[e] = kNegInf;
        return;
    }
    h.load((const Raw *)rows + row * ld, at, min(k, at + kVerifyEach), 0);
#pragma unroll
    for (int e = 0; e < kVerifyEach; ++e) x[e] = h.at(e / H::VEC, e % H::VEC);
}
template <typename T> __device__ __forceinline__ void lane_weights(const VerifyArgs &a, const Weights &w, int64_t seq, int pos, int at, double (&y)[kVerifyEach]) {
    float s[kVerifyEach], t[kVerifyEach];
    lane_codes<T>(a.target, seq * (a.draft + 1) + pos, a.ld_target, at, a.k, s);
    if (w.minus) lane_codes<T>(a.drafts, seq * a.draft + pos, a.ld_draft, at, a.k, t);
#pragma unroll
    for (int e = 0; e < kVerifyEach; ++e) {
        y[e] = w(s[e], w.minus ? t[e] : 0.0f);
        if (at + e == w.code) y[e] = 0.0;
    }
}

// Sums of max(p - q, 0) where a draft with scores was refused.
template <typename T>
__global__ void __launch_bounds__(256) k_verify_left(VerifyArgs a) {
    __shared__ VerdictLds lds;
    __shared__ double sum_of[4];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), groups = (a.parts + a.left_parts - 1) / a.left_parts;
    const int64_t seq = blockIdx.x / (unsigned)groups;
    const int first = (int)(blockIdx.x % (unsigned)groups) * a.left_parts;
    int64_t code;
    const Verdict o = verdict<T>(a, seq, lds, &code);
    if (o.bad || o.accepted == o.length) return;  // uniform
    const Weights w = weights(a, o);
    for (int part = first; part < min(a.parts, first + a.left_parts); ++part) {
        double y[kVerifyEach], sum = 0.0;
        lane_weights<T>(a, w, seq, o.accepted, part * kVerifyPart + tid * kVerifyEach, y);
#pragma unroll
        for (int e = 0; e < kVerifyEach; ++e) sum += y[e];
        sum = wave_sum(sum);
        __syncthreads();
        if (lane == 0) sum_of[wave] = sum;
        __syncthreads();
        if (tid == 0) a.left[seq * a.parts + part] = sum_of[0] + sum_of[1] + sum_of[2] + sum_of[3];
    }
}

// The outcome of a sequence: how many drafts stay, and the codes: these, the next one, -1 behind it.
template <typename T>
__global__ void __launch_bounds__(256) k_verify_pick(VerifyArgs a) {
    __shared__ double part_of[256], sum_of[4];
    __shared__ int found[4];
    __shared__ VerdictLds lds;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int64_t seq = blockIdx.x;
    int64_t code;
    const Verdict o = verdict<T>(a, seq, lds, &code);
    int next = -1;
    if (!o.bad) {  // uniform
        Weights w = weights(a, o);
        const int64_t row = seq * (a.draft + 1) + o.accepted;
        double total = 0.0, mine = 0.0, before = 0.0;
        for (;;) {  // (a second time where nothing is left of p - q)
            if (tid < a.parts) {
                if (w.minus)
                    mine = a.left[seq * a.parts + tid];
                else {
                    const float m = a.most[row * a.parts + tid];
                    mine = m > kNegInf ? a.sum[row * a.parts + tid] * exp2_wide(((double)m - o.mp) * a.c_target) : 0.0;
                }
            }
            // sums of the parts up to each
            double scan = wave_scan(mine, lane);
            __syncthreads();
            if (lane == 63) sum_of[wave] = scan;
            __syncthreads();
            before = 0.0;
            for (int i = 0; i < wave; ++i) before += sum_of[i];
            scan += before;
            part_of[tid] = scan;
            total = sum_of[0] + sum_of[1] + sum_of[2] + sum_of[3];
            if (total > 0.0 || !w.minus) break;
            w.minus = false;
            w.by_p = 1.0;
        }
        const double goal = (double)a.uniform[seq * a.ld_uniform + a.draft] * total;
        // the first part that reaches the goal, or the last that has any weight
        const auto choose = [&](bool has, double upto) {
            const unsigned long long hit = __ballot(has && upto > goal), any = __ballot(has);
            if (lane == 0) found[wave] = hit ? wave * 64 + __ffsll(hit) - 1 : any ? 1024 + wave * 64 + 63 - __clzll(any) : -1;
            __syncthreads();
            int at = -1;
            for (int i = 3; i >= 0; --i) at = found[i] >= 0 && found[i] < 1024 ? found[i] : at;
            if (at < 0)
                for (int i = 0; i < 4; ++i) at = found[i] >= 0 ? found[i] - 1024 : at;
            __syncthreads();
            return at;
        };
        const int part = choose(mine > 0.0, part_of[tid]);
        if (part >= 0) {  // uniform
            const double base = part ? part_of[part - 1] : 0.0;
            const int at = part * kVerifyPart + tid * kVerifyEach;
            double y[kVerifyEach], sum = 0.0;
            lane_weights<T>(a, w, seq, o.accepted, at, y);
#pragma unroll
            for (int e = 0; e < kVerifyEach; ++e) sum += y[e];
            double scan = wave_scan(sum, lane);
            if (lane == 63) sum_of[wave] = scan;
            __syncthreads();
            double from = base;
            for (int i = 0; i < wave; ++i) from += sum_of[i];
            const int who = choose(sum > 0.0, from + scan);
            if (tid == who) {
                double so_far = from + (scan - sum);
                int last = -1, first = -1;
#pragma unroll
                for (int e = 0; e < kVerifyEach; ++e) {
                    so_far += y[e];
                    if (y[e] > 0.0) {
                        last = e;
                        if (first < 0 && so_far > goal) first = e;
                    }
                }
                found[0] = at + (first >= 0 ? first : last);
            }
            __syncthreads();
            if (who >= 0) next = found[0];
        }
    }
    if (wave) return;
    if (lane == 0) a.accepted[seq] = o.accepted;
    if (lane <= a.draft) a.out[seq * a.ld_out + lane] = lane < o.accepted ? (int32_t)code : lane == o.accepted ? next : -1;
}

}  // namespace vq
