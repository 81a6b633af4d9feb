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
    int n, draft, k, parts;  // parts of kVerifyPart codes
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
    float *own;    // the largest score of the part alone, where `most` is that of the parts that a workgroup summed with it
    double *left;  // per sequence and part: the sum of max(p - q, 0)
    struct Verdict *verdicts;  // per sequence, where those sums are made
};

// The drafted codes of a sequence: lane d has code d; returns how many there are before the first that is none.
__device__ __forceinline__ int drafted(const VerifyArgs &a, int64_t seq, int lane, int64_t *code) {
    *code = lane < a.draft ? code_at(a.codes, a.code_bytes, seq * a.code_stride + lane) : -1;
    return __ffsll(__ballot(*code < 0)) - 1;  // (lane 63 has none)
}

// EACH / 16 parts of a row per workgroup, their sums relative to the largest score of all of them.  Bound by the vector pipe: 15 instructions in 64 bits
// per code (conversion, difference, limit, three for the whole part and the rest, eight of the polynomial, the sum), which go at 580 x 10^9 a second and wave,
// and some six others with those of a wave, at 1000.  128 sequences of 11 rows of 65,536 bf16: 21.6M and 9.4M, 37 + 9 of 61 us.
template <typename T, int EACH>
__global__ void __launch_bounds__(256) k_verify_part(VerifyArgs a) {
    typedef typename T::Raw Raw;
    typedef Held<T, 256, EACH * (int)sizeof(Raw) / 16> H;
    constexpr int WAVES = 4, PARTS = EACH / 16, PIECES = EACH / H::VEC / PARTS;  // vectors of a lane in a part
    __shared__ float most_of[WAVES][PARTS];
    __shared__ double sum_of[WAVES][PARTS];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t groups = (uint32_t)(a.parts + PARTS - 1) / PARTS;
    const uint32_t row = blockIdx.x / groups, targets = (uint32_t)a.n * (uint32_t)(a.draft + 1);  // (a launch has fewer than 2^23)
    const int first = (int)(blockIdx.x - row * groups) * PARTS, lo = first * kVerifyPart, hi = min(a.k, lo + PARTS * kVerifyPart);
    const bool draft = row >= targets;
    const uint32_t of = draft ? row - targets : row, each = draft ? a.draft : a.draft + 1, seq = of / each;
    const int pos = (int)(of - seq * each);
    H x;
    int64_t code;
    int length = a.draft;
    if (a.code_bytes == 4 || !a.drafts) length = drafted(a, seq, lane, &code);  // (unsigned codes end no draft)
    if (pos >= length + (draft ? 0 : 1)) return;  // uniform: a row that nothing is drafted for
    x.load(draft ? (const Raw *)a.drafts + (int64_t)of * a.ld_draft : (const Raw *)a.target + (int64_t)of * a.ld_target, lo, hi, tid);
    if (!a.drafts && pos < length) {  // the row without its drafted code
        const int64_t c = (int64_t)__shfl((int)code, pos) - lo;
        if (c >= 0 && c < hi - lo) {
            const int place = (int)c / H::VEC;
            if (place % (64 * WAVES) == tid) {
#pragma unroll
                for (int u = 0; u < EACH / H::VEC; ++u)
#pragma unroll
                    for (int v = 0; v < H::VEC; ++v)
                        if (u == place / (64 * WAVES) && v == (int)c % H::VEC) x.drop(u, v);
            }
        }
    }
    float m = kNegInf, most[PARTS];
#pragma unroll
    for (int p = 0; p < PARTS; ++p) {
        most[p] = kNegInf;
#pragma unroll
        for (int u = 0; u < PIECES; ++u)
#pragma unroll
            for (int v = 0; v < H::VEC; v += 2) most[p] = larger_or_nan(larger_or_nan(x.at(p * PIECES + u, v), x.at(p * PIECES + u, v + 1)), most[p]);
        most[p] = __uint_as_float(over_group<64>(__float_as_uint(most[p]), __float_as_uint(kNegInf), [](uint32_t p, uint32_t q) {
            return __float_as_uint(larger_or_nan(__uint_as_float(p), __uint_as_float(q)));
        }));
        if (lane == 0) most_of[wave][p] = most[p];
    }
    __syncthreads();
#pragma unroll
    for (int p = 0; p < PARTS; ++p) {
#pragma unroll
        for (int w = 0; w < WAVES; ++w) most[p] = larger_or_nan(most[p], most_of[w][p]);
        m = larger_or_nan(m, most[p]);
    }
    const bool sound = m > kNegInf && m < __builtin_inff();  // uniform
    const double c = draft ? a.c_draft : a.c_target, from = sound ? m : 0.0f, least = -1000.0 / c;  // (the difference first: of scores of 1e38 a rounded product leaves too much)
#pragma unroll
    for (int p = 0; p < PARTS; ++p) {
        double sum = 0.0;
        if (sound) {
#pragma unroll
            for (int u = 0; u < PIECES; ++u)
#pragma unroll
                for (int v = 0; v < H::VEC; ++v) sum += exp2_of(fmax((double)x.at(p * PIECES + u, v) - from, least), c);
        }
        sum = wave_sum(sum);
        if (lane == 0) sum_of[wave][p] = sum;
    }
    __syncthreads();
    if (tid >= PARTS || first + tid >= a.parts) return;
    float own = most[0];
#pragma unroll
    for (int p = 1; p < PARTS; ++p) own = tid == p ? most[p] : own;
    // a part without a weight: its codes are too far below, or none can be
    const bool none = sound && !((double)own - from >= least);
    const int64_t at = (int64_t)row * a.parts + first + tid;
    a.most[at] = none ? kNegInf : m;
    a.own[at] = own;
    double sum = sum_of[0][tid];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) sum += sum_of[w][tid];
    a.sum[at] = none ? 0.0 : sum;
}

constexpr int kVerifyEach = kVerifyPart / 256;  // codes of a lane where weights are summed

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

// The sums of a sequence's rows from those of their parts: the target's of each position up to `length`, then the drafts'.
__device__ __forceinline__ void join_parts(const VerifyArgs &a, int64_t seq, int length, VerdictLds &l) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), rows = length + 1 + (a.drafts ? length : 0);
    constexpr int WAVES = 4, AHEAD = 4;
    for (int r0 = wave; r0 < rows; r0 += WAVES * AHEAD) {
        float most[AHEAD];
        double sum[AHEAD];
        const auto row_of = [&](int i) {
            const int r = min(r0 + WAVES * i, rows - 1);
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
            const int r = r0 + WAVES * i;
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
}

// By a workgroup of four waves: each makes or joins the sums of every fourth row, row_sums(l, length), and the first decides.  code: a lane's
// drafted code.
template <typename T, typename F> __device__ __forceinline__ Verdict verdict(const VerifyArgs &a, int64_t seq, VerdictLds &l, int64_t *code, F row_sums) {
    typedef typename T::Raw Raw;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int length = drafted(a, seq, lane, code);
    const bool here = lane <= length, asked = lane < length, known = asked && *code < a.k;
    float s = 0.0f, t = 0.0f, u = 0.0f;  // lane d: the scores of drafted code d, its random number
    if (wave == 0 && asked) {
        u = a.uniform[seq * a.ld_uniform + lane];
        if (known) {
            s = T::up(((const Raw *)a.target)[(seq * (a.draft + 1) + lane) * a.ld_target + *code]);
            if (a.drafts) t = T::up(((const Raw *)a.drafts)[(seq * a.draft + lane) * a.ld_draft + *code]);
        }
    }
    row_sums(length);
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
    double c_target, c_draft, least_p, least_q, mp, mq, by_p, by_q;
    int code;   // this one has none
    bool minus;  // max(p - q, 0), otherwise p
    __device__ __forceinline__ double operator()(float s, float t) const {
        const double y = (double)s - mp;
        double w = exp2_of(fmax(y, least_p), c_target) * by_p;
        if (minus) w = fmax(w - exp2_of(fmax((double)t - mq, least_q), c_draft) * by_q, 0.0);
        return y < least_p ? 0.0 : w;
    }
};
__device__ __forceinline__ Weights weights(const VerifyArgs &a, const Verdict &o) {
    const bool minus = o.accepted < o.length && a.drafts;
    return {a.c_target, a.c_draft, -1000.0 / a.c_target, minus ? -1000.0 / a.c_draft : 0.0, o.mp, o.mq, minus ? 1.0 / o.Sp : 1.0, minus ? 1.0 / o.Sq : 0.0,
            minus ? -1 : o.refused, minus};
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

template <typename T> __global__ void __launch_bounds__(256) k_verify_verdict(VerifyArgs a) {
    __shared__ VerdictLds lds;
    int64_t code;
    const Verdict o = verdict<T>(a, blockIdx.x, lds, &code, [&](int length) { join_parts(a, blockIdx.x, length, lds); });
    if (threadIdx.x == 0) a.verdicts[blockIdx.x] = o;
}

// Sums of max(p - q, 0) by parts where a draft with scores was refused.  READY: the verdicts are there; else every workgroup comes to its
// sequence's, which takes it 4 us, a launch less, and the first one writes it.
template <typename T, bool READY>
__global__ void __launch_bounds__(256) k_verify_left(VerifyArgs a) {
    __shared__ double sum_of[4];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t seq = blockIdx.x / (uint32_t)a.parts;
    const int part = (int)(blockIdx.x - seq * (uint32_t)a.parts);
    Verdict o;
    if constexpr (READY) {
        o = a.verdicts[seq];
    } else {
        __shared__ VerdictLds lds;
        int64_t code;
        o = verdict<T>(a, seq, lds, &code, [&](int length) { join_parts(a, seq, length, lds); });
        if (part == 0 && tid == 0) a.verdicts[seq] = o;
    }
    if (o.bad || o.accepted == o.length) return;  // uniform
    const Weights w = weights(a, o);
    float s[kVerifyEach], t[kVerifyEach];
    const int at = part * kVerifyPart + tid * kVerifyEach;
    lane_codes<T>(a.target, (int64_t)seq * (a.draft + 1) + o.accepted, a.ld_target, at, a.k, s);
    lane_codes<T>(a.drafts, (int64_t)seq * a.draft + o.accepted, a.ld_draft, at, a.k, t);
    double sum = 0.0;
#pragma unroll
    for (int e = 0; e < kVerifyEach; ++e) sum += w(s[e], t[e]);
    sum = wave_sum(sum);
    if (lane == 0) sum_of[wave] = sum;
    __syncthreads();
    if (tid == 0) a.left[blockIdx.x] = sum_of[0] + sum_of[1] + sum_of[2] + sum_of[3];
}

// Sums over a workgroup of four waves, and the lane that a sum belongs to.
struct Choice {
    double sum[4];
    int found[4];
};
struct Chooser {
    Choice &l;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    __device__ __forceinline__ explicit Chooser(Choice &c) : l(c) {}
    // the sum up to each lane, from `from` on, and of all
    __device__ __forceinline__ double scan(double mine, double from, double *total) {
        const double upto = wave_scan(mine, lane);
        __syncthreads();
        if (lane == 63) l.sum[wave] = upto;
        __syncthreads();
        *total = 0.0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            from += i < wave ? l.sum[i] : 0.0;
            *total += l.sum[i];
        }
        return from + upto;
    }
    // the first lane whose sum is above the goal, or else the last that has any weight; -1: none has
    __device__ __forceinline__ int choose(bool has, double upto, double goal) {
        constexpr int NOT = 1024;
        const unsigned long long hit = __ballot(has && upto > goal), any = __ballot(has);
        if (lane == 0) l.found[wave] = hit ? wave * 64 + __ffsll(hit) - 1 : any ? NOT + wave * 64 + 63 - __clzll(any) : -1;
        __syncthreads();
        int at = -1, last = -1;
#pragma unroll
        for (int i = 3; i >= 0; --i) {
            at = l.found[i] >= 0 && l.found[i] < NOT ? l.found[i] : at;
            last = last < 0 && l.found[i] >= NOT ? l.found[i] - NOT : last;
        }
        __syncthreads();
        return at >= 0 ? at : last;
    }
};
// The same among a lane's codes.
__device__ __forceinline__ int among(const double (&y)[kVerifyEach], double so_far, double goal) {
    int last = -1, first = -1;
#pragma unroll
    for (int e = 0; e < kVerifyEach; ++e) {
        so_far += y[e];
        if (y[e] > 0.0) {
            last = e;
            if (first < 0 && so_far > goal) first = e;
        }
    }
    return first >= 0 ? first : last;
}
__device__ __forceinline__ void write_outcome(const VerifyArgs &a, int64_t seq, const Verdict &o, int64_t code, int next, int lane) {
    if (lane == 0) a.accepted[seq] = o.accepted;
    if (lane <= a.draft) a.out[seq * a.ld_out + lane] = lane < o.accepted ? (int32_t)code : lane == o.accepted ? next : -1;
}

// The outcome of a sequence: how many drafts stay, and the codes: these, the next one, -1 behind it.
// READY: what the drafts come to is there.
template <typename T, bool READY>
__global__ void __launch_bounds__(256) k_verify_pick(VerifyArgs a) {
    __shared__ double part_of[256];
    __shared__ Choice choice;
    __shared__ int next_of;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int64_t seq = blockIdx.x;
    int64_t code;
    Verdict o;
    const float v = a.uniform[seq * a.ld_uniform + a.draft];
    if constexpr (READY) {
        o = a.verdicts[seq];
        code = lane < o.accepted ? code_at(a.codes, a.code_bytes, seq * a.code_stride + lane) : -1;
    } else {
        __shared__ VerdictLds lds;
        o = verdict<T>(a, seq, lds, &code, [&](int length) { join_parts(a, seq, length, lds); });
    }
    Chooser chooser(choice);
    double total;
    if (tid == 0) next_of = -1;
    if (!o.bad) {  // uniform
        Weights w = weights(a, o);
        const int64_t row = seq * (a.draft + 1) + o.accepted;
        double mine, upto;
        for (;;) {  // (a second time where nothing is left of p - q)
            mine = 0.0;
            if (tid < a.parts && w.minus) {
                mine = a.left[seq * a.parts + tid];
            } else if (tid < a.parts) {
                // a part has a weight where its largest score has one, by the same rule: its sum times a power may be a number where no code's weight is
                const float m = a.most[row * a.parts + tid], own = a.own[row * a.parts + tid];
                mine = m > kNegInf && (double)own - o.mp >= w.least_p ? a.sum[row * a.parts + tid] * exp2_wide(((double)m - o.mp) * a.c_target) : 0.0;
            }
            upto = chooser.scan(mine, 0.0, &total);
            if (total > 0.0 || !w.minus) break;
            w.minus = false;
            w.by_p = 1.0;
        }
        part_of[tid] = upto;
        const double goal = (double)v * total;
        int part = chooser.choose(mine > 0.0, upto, goal);
        if (part >= 0) {  // uniform
            const int at = part * kVerifyPart + tid * kVerifyEach;
            double y[kVerifyEach], sum = 0.0;
            lane_weights<T>(a, w, seq, o.accepted, at, y);
#pragma unroll
            for (int e = 0; e < kVerifyEach; ++e) sum += y[e];
            upto = chooser.scan(sum, part ? part_of[part - 1] : 0.0, &total);
            if (tid == chooser.choose(sum > 0.0, upto, goal)) next_of = at + among(y, upto - sum, goal);
        }
    }
    __syncthreads();
    if (wave) return;
    write_outcome(a, seq, o, code, next_of, lane);
}

// Rows of up to 2048 codes: a workgroup does all of a sequence, a wave per row, in one launch (62 sequences of 17 rows of 237 codes 23 us in
// three, 17 so).
constexpr int kVerifyFew = 2048;
template <typename T> __global__ void __launch_bounds__(256) k_verify_few(VerifyArgs a) {
    typedef typename T::Raw Raw;
    constexpr int EACH = kVerifyFew / 64;
    typedef Held<T, 64, EACH * (int)sizeof(Raw) / 16> H;
    __shared__ VerdictLds lds;
    __shared__ Choice choice;
    __shared__ int next_of;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int64_t seq = blockIdx.x;
    const float v = a.uniform[seq * a.ld_uniform + a.draft];
    int64_t code;
    const Verdict o = verdict<T>(a, seq, lds, &code, [&](int length) {
        const int rows = length + 1 + (a.drafts ? length : 0);
        for (int r = wave; r < rows; r += 4) {
            const bool draft = r > length;
            const int pos = draft ? r - length - 1 : r;
            H x;
            x.load(draft ? (const Raw *)a.drafts + (seq * a.draft + pos) * a.ld_draft : (const Raw *)a.target + (seq * (a.draft + 1) + pos) * a.ld_target, 0, a.k,
                   lane);
            const int out = !a.drafts && pos < length ? __shfl((int)code, pos) : -1;  // the row without its drafted code
            float m = kNegInf;
#pragma unroll
            for (int u = 0; u < EACH / H::VEC; ++u)
#pragma unroll
                for (int v = 0; v < H::VEC; ++v) {
                    if ((u * 64 + lane) * H::VEC + v == out) x.drop(u, v);
                    m = larger_or_nan(m, x.at(u, v));
                }
            m = __uint_as_float(over_group<64>(__float_as_uint(m), __float_as_uint(kNegInf), [](uint32_t p, uint32_t q) {
                return __float_as_uint(larger_or_nan(__uint_as_float(p), __uint_as_float(q)));
            }));
            const bool sound = m > kNegInf && m < __builtin_inff();  // uniform
            const double c = draft ? a.c_draft : a.c_target, from = sound ? m : 0.0f, least = -1000.0 / c;
            double sum = 0.0;
            if (sound) {
#pragma unroll
                for (int u = 0; u < EACH / H::VEC; ++u) {
                    if (u * 64 * H::VEC >= a.k) break;  // uniform
#pragma unroll
                    for (int v = 0; v < H::VEC; ++v) sum += exp2_of(fmax((double)x.at(u, v) - from, least), c);
                }
            }
            sum = wave_sum(sum);
            if (lane == 0) {
                lds.m[draft][pos] = m;
                lds.S[draft][pos] = m == kNegInf ? 0.0 : sound ? sum : __builtin_nan("");
            }
        }
    });
    Chooser chooser(choice);
    if (tid == 0) next_of = -1;
    if (!o.bad) {  // uniform
        Weights w = weights(a, o);
        double y[kVerifyEach], sum, upto, total;
        for (;;) {  // (a second time where nothing is left of p - q)
            lane_weights<T>(a, w, seq, o.accepted, tid * kVerifyEach, y);
            sum = 0.0;
#pragma unroll
            for (int e = 0; e < kVerifyEach; ++e) sum += y[e];
            upto = chooser.scan(sum, 0.0, &total);
            if (total > 0.0 || !w.minus) break;
            w.minus = false;
            w.by_p = 1.0;
        }
        const double goal = (double)v * total;
        if (tid == chooser.choose(sum > 0.0, upto, goal)) next_of = tid * kVerifyEach + among(y, upto - sum, goal);
    }
    __syncthreads();
    if (wave == 0) write_outcome(a, seq, o, code, next_of, lane);
}

}  // namespace vq
