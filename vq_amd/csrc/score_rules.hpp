// What the calls on 8-bit scores and log probabilities of codes take and refuse: rules on sizes, strides and addresses
// alone, without HIP, so that a CPU test can go through them.
#pragma once
#include <algorithm>
#include <cstdint>

#include "../../include/vq_hip.h"

namespace vq {

// Components of an 8-bit row: the sum of as many products of two bytes (at most 2^14 each) fits 32 bits.
constexpr int32_t kMaxDimI8 = 131071;
constexpr int32_t kMaxTop = 32;           // alternatives of a row
constexpr int32_t kMaxScoreCodes = 1 << 24;  // codes that rows are scored against
constexpr int32_t kMaxRowCodes = 1 << 20;    // codes of a row of scores whose probabilities are asked for

// Status and text of a refusal; VQ_OK: the call may run.
struct Refusal {
    int32_t status = VQ_OK;
    const char *text = "";
};
inline Refusal refuse(int32_t status, const char *what) { return {status, what}; }

inline int type_bytes(int32_t type) { return type == VQ_F32 ? 4 : type == VQ_F16 || type == VQ_BF16 ? 2 : 0; }

// The bytes of n rows of `row` bytes, `ld` bytes apart; [0, 0) for no rows.
struct Span {
    uintptr_t lo = 0, hi = 0;
    Span(const void *p, int64_t n, int64_t ld, int64_t row) {
        if (p && n > 0) lo = (uintptr_t)p, hi = lo + (uintptr_t)((n - 1) * ld + row);
    }
    bool meets(const Span &o) const { return lo < o.hi && o.lo < hi; }
};
// n rows of ld elements stay below 2^48 bytes, more than any memory
inline bool too_long(int64_t n, int64_t ld, int bytes) {
    return ld > 0 && n > (int64_t)(((uint64_t)1 << 48) / (uint64_t)bytes) / ld;
}
inline bool misaligned(const void *p, int bytes) { return ((uintptr_t)p & (uintptr_t)(bytes - 1)) != 0; }

inline Refusal check_rows_i8(int32_t type, const void *x, int64_t n, int64_t ld, int32_t dim, const void *q, int64_t ld_q,
                             const void *scale) {
    const int e = type_bytes(type);
    if (!e) return refuse(VQ_ERR_INVALID_ARG, "no such type");
    if (n < 0 || dim <= 0) return refuse(VQ_ERR_INVALID_ARG, "n must not be negative and dim must be greater than 0");
    if (dim > kMaxDimI8) return refuse(VQ_ERR_UNSUPPORTED, "dim must be at most 131071");
    if (ld < dim || ld_q < dim) return refuse(VQ_ERR_INVALID_ARG, "a row stride is below dim");
    if (too_long(n, ld, e) || too_long(n, ld_q, 1)) return refuse(VQ_ERR_INVALID_ARG, "rows and stride overflow");
    if (n == 0) return {};
    if (!x || !q || !scale) return refuse(VQ_ERR_INVALID_ARG, "null pointer");
    if (misaligned(x, e) || misaligned(scale, 4)) return refuse(VQ_ERR_INVALID_ARG, "misaligned pointer");
    const Span sx(x, n, ld * e, (int64_t)dim * e), sq(q, n, ld_q, dim), ss(scale, 1, 0, n * 4);
    if (sx.meets(sq) || sx.meets(ss) || sq.meets(ss)) return refuse(VQ_ERR_INVALID_ARG, "an output overlaps another array");
    return {};
}

inline Refusal check_scores_i8(const void *x, const void *xs, int64_t n, int64_t ld_x, const void *w, const void *ws, int32_t k,
                               int64_t ld_w, int32_t dim, const void *bias, int32_t out_type, const void *out, int64_t ld_out) {
    const int e = type_bytes(out_type);
    if (!e) return refuse(VQ_ERR_INVALID_ARG, "no such type");
    if (n < 0 || dim <= 0 || k <= 0) return refuse(VQ_ERR_INVALID_ARG, "n must not be negative, dim and k must be greater than 0");
    if (dim > kMaxDimI8) return refuse(VQ_ERR_UNSUPPORTED, "dim must be at most 131071");
    if (k > kMaxScoreCodes) return refuse(VQ_ERR_UNSUPPORTED, "k must be at most 16777216");
    if (ld_x < dim || ld_w < dim || ld_out < k) return refuse(VQ_ERR_INVALID_ARG, "a row stride is below the row's length");
    if (too_long(n, ld_x, 1) || too_long(k, ld_w, 1) || too_long(n, ld_out, e))
        return refuse(VQ_ERR_INVALID_ARG, "rows and stride overflow");
    if (n == 0) return {};
    if (!x || !xs || !w || !ws || !out) return refuse(VQ_ERR_INVALID_ARG, "null pointer");
    if (misaligned(xs, 4) || misaligned(ws, 4) || misaligned(bias, 4) || misaligned(out, e))
        return refuse(VQ_ERR_INVALID_ARG, "misaligned pointer");
    const Span so(out, n, ld_out * e, (int64_t)k * e);
    if (so.meets({x, n, ld_x, dim}) || so.meets({w, k, ld_w, dim}) || so.meets({xs, 1, 0, n * 4}) ||
        so.meets({ws, 1, 0, (int64_t)k * 4}) || so.meets({bias, 1, 0, (int64_t)k * 4}))
        return refuse(VQ_ERR_INVALID_ARG, "the scores overlap an input");
    return {};
}

// The scores, codes and sizes that both calls on log probabilities take.
inline Refusal check_scored_codes(int32_t type, const void *s, int64_t n, int64_t ld, int32_t k, float beta, int32_t code_bytes,
                                  const void *codes, int64_t code_stride) {
    const int e = type_bytes(type);
    if (!e) return refuse(VQ_ERR_INVALID_ARG, "no such type");
    if (n < 0 || k <= 0) return refuse(VQ_ERR_INVALID_ARG, "n must not be negative and k must be greater than 0");
    if (k > kMaxRowCodes) return refuse(VQ_ERR_UNSUPPORTED, "k must be at most 1048576");
    if (ld < k) return refuse(VQ_ERR_INVALID_ARG, "the row stride is below k");
    if (too_long(n, ld, e)) return refuse(VQ_ERR_INVALID_ARG, "rows and stride overflow");
    if (!(beta >= 1e-30f) || !(beta <= 1e30f)) return refuse(VQ_ERR_INVALID_ARG, "beta must be between 1e-30 and 1e30");
    if (codes) {
        if (code_bytes != 1 && code_bytes != 2 && code_bytes != 4) return refuse(VQ_ERR_INVALID_ARG, "codes have 1, 2 or 4 bytes");
        if (code_stride <= 0 || too_long(n, code_stride, code_bytes)) return refuse(VQ_ERR_INVALID_ARG, "stride of the codes");
        if (misaligned(codes, code_bytes)) return refuse(VQ_ERR_INVALID_ARG, "misaligned pointer");
    }
    if (n == 0) return {};
    if (!s) return refuse(VQ_ERR_INVALID_ARG, "null pointer");
    if (misaligned(s, e)) return refuse(VQ_ERR_INVALID_ARG, "misaligned pointer");
    return {};
}

inline Refusal check_code_logprobs(int32_t type, const void *s, int64_t n, int64_t ld, int32_t k, float beta, int32_t code_bytes,
                                   const void *codes, int64_t code_stride, int32_t top, const void *logprob, const void *max,
                                   const void *logsum, const void *entropy, const void *top_logprob, const void *top_code) {
    const Refusal r = check_scored_codes(type, s, n, ld, k, beta, code_bytes, codes, code_stride);
    if (r.status != VQ_OK) return r;
    if (top < 0) return refuse(VQ_ERR_INVALID_ARG, "top must not be negative");
    if (top > kMaxTop) return refuse(VQ_ERR_UNSUPPORTED, "top must be at most 32");
    if (n == 0) return {};
    if ((codes == nullptr) != (logprob == nullptr)) return refuse(VQ_ERR_INVALID_ARG, "codes and their log probabilities go together");
    if (top > 0 && (!top_logprob || !top_code)) return refuse(VQ_ERR_INVALID_ARG, "null pointer");
    const void *outs[] = {logprob, max, logsum, entropy, top ? top_logprob : nullptr, top ? top_code : nullptr};
    const int e = type_bytes(type);
    const Span in[] = {{s, n, ld * e, (int64_t)k * e}, {codes, n, code_stride * code_bytes, code_bytes}};
    for (int a = 0; a < 6; ++a) {
        if (misaligned(outs[a], 4)) return refuse(VQ_ERR_INVALID_ARG, "misaligned pointer");
        const Span oa(outs[a], 1, 0, n * 4 * (a < 4 ? 1 : top));
        for (int b = 0; b < a; ++b)
            if (oa.meets({outs[b], 1, 0, n * 4 * (b < 4 ? 1 : top)})) return refuse(VQ_ERR_INVALID_ARG, "an output overlaps another array");
        for (const Span &i : in)
            if (oa.meets(i)) return refuse(VQ_ERR_INVALID_ARG, "an output overlaps another array");
    }
    return {};
}

inline Refusal check_code_logprobs_grad(int32_t type, const void *s, int64_t n, int64_t ld, int32_t k, float beta,
                                        int32_t code_bytes, const void *codes, int64_t code_stride, const void *max,
                                        const void *logsum, const void *entropy, const void *g_logprob, const void *g_entropy,
                                        const void *grad, int64_t ld_grad) {
    const Refusal r = check_scored_codes(type, s, n, ld, k, beta, code_bytes, codes, code_stride);
    if (r.status != VQ_OK) return r;
    const int e = type_bytes(type);
    if (ld_grad < k || too_long(n, ld_grad, e)) return refuse(VQ_ERR_INVALID_ARG, "stride of the gradient");
    if (n == 0) return {};
    if (!max || !logsum || !grad || (!g_logprob && !g_entropy)) return refuse(VQ_ERR_INVALID_ARG, "null pointer");
    if (g_logprob && !codes) return refuse(VQ_ERR_INVALID_ARG, "a gradient of log probabilities without their codes");
    if (g_entropy && !entropy) return refuse(VQ_ERR_INVALID_ARG, "a gradient of entropies without the entropies");
    const void *rows[] = {max, logsum, entropy, g_logprob, g_entropy};
    const Span sg(grad, n, ld_grad * e, (int64_t)k * e);
    for (const void *p : rows) {
        if (misaligned(p, 4)) return refuse(VQ_ERR_INVALID_ARG, "misaligned pointer");
        if (sg.meets({p, 1, 0, n * 4})) return refuse(VQ_ERR_INVALID_ARG, "the gradient overlaps an input");
    }
    if (misaligned(grad, e)) return refuse(VQ_ERR_INVALID_ARG, "misaligned pointer");
    if (sg.meets({codes, n, code_stride * code_bytes, code_bytes})) return refuse(VQ_ERR_INVALID_ARG, "the gradient overlaps an input");
    // in place, or elsewhere
    if (!(grad == s && ld_grad == ld) && sg.meets({s, n, ld * e, (int64_t)k * e}))
        return refuse(VQ_ERR_INVALID_ARG, "the gradient overlaps the scores otherwise than in place");
    return {};
}

// How the rows of a call go through the GPU: `lanes` of a row, `per_lane` codes each (microseconds of the ways compared, calls in a row):
//   1, 4, 8 lanes  rows of up to 256 codes, several to a wave: the alternatives one after another (200,000 x 256, f32, 12 alternatives
//                  92, a wave each 107; 2000 x 256, 2 alternatives 5.4 and 5.5)
//   a wave, 8      up to 512 codes; of shorter rows those with many alternatives, which a wave lists and sorts at once: up to 16,384 rows with 8
//                  or more (2000 x 24, f32, 32 alternatives 5.3, in 4 lanes 18; x 256, 20: 5.4, in 8 lanes 19; the line is low for the
//                  most rows and the fewest alternatives, 16,384 x 24, f16, 8: 11.3 and 6.4), and above 128 codes those with 16 or more for
//                  which five lanes more than these hold codes (200,000 x 256, f32, 20: 112 and 145, 16: 110 and 119; x 128, 32: 240 and
//                  222; bf16, x 256, 20: 119 and 143, 32, which all the 32 lanes with codes would have to give: 310 and 220)
//   a wave         up to 4096 codes, 16 to 64 per lane (600 x 4000, bf16, 5 alternatives 6.1, a workgroup each 6.7; 10,000 x 2000, 5:
//                  15 and 32; 100,000 x 2000, 20: 109 and 360)
//   a workgroup    up to 16,384 codes, 32 or 64 per lane (8 x 16,384, f32, 20 alternatives 7.7, in two parts 11.7)
//   parts          longer rows: of 16,384 codes, or of 8192 where those would be fewer than 4096 workgroups and 64 parts are enough
//                  (777 x 50,021, f16, 5 alternatives 26.5 in parts of 8192, 28.3; 300 x 32,000, bf16, 8: 13.9 and 15.2; 8192 x 65,536, 8:
//                  214 and 198; about 1000 x 65,536 33.2 and 32.6)
constexpr int kMostParts = 64;
struct RowPlan {
    int lanes, per_lane;
    int32_t parts, codes;
};
static_assert(kMaxRowCodes <= kMostParts * 64 * 256, "64 codes per lane hold every row");
inline RowPlan plan_rows(int64_t n, int32_t k, int32_t top, int bytes = 4) {
    const bool many = (n <= 16384 && top >= 8) || (k > 128 && top >= 16 && k * bytes / 16 >= top + 5);
    if (k <= 512 && k >= 8 && (k > 256 || many)) return {64, 8, 1, k};
    if (k <= 256) return {k <= 16 ? 1 : k <= 64 ? 4 : 8, k <= 64 ? 16 : 32, 1, k};
    if (k <= 4096) return {64, k <= 1024 ? 16 : k <= 2048 ? 32 : 64, 1, k};
    const int64_t whole = (k + 16383) / 16384;
    const int e = k <= 8192 || (k > 16384 && n * whole < 4096 && k <= kMostParts * 8192) ? 32 : 64;
    return {256, e, (k + 256 * e - 1) / (256 * e), 256 * e};
}

// Rows of a launch: a grid has fewer than 2^32 lanes, and the parts' results (sums and lists) take at most 64 MiB.
constexpr int64_t kPartBytes = 64 << 20;
inline int64_t part_bytes(int32_t top) { return 12 + 8 * top; }
inline int64_t logprob_rows_of_a_launch(const RowPlan &plan, int32_t top) {
    if (plan.lanes < 256) return (int64_t)(1 << 23) * (256 / plan.lanes);
    return std::max<int64_t>(1, (plan.parts == 1 ? 1 << 23 : kPartBytes / part_bytes(top)) / plan.parts);
}
// Bytes of the parts' results that a call provides for: no fewer than its plan takes, and no fewer than any call of no more rows, codes
// and alternatives does, so that one of those may follow in a capture.  (A plan itself halves its parts' length, and so doubles their number,
// where rows or codes get fewer: 1024 rows of 65,536 codes have 4 parts each, 1023 have 8.)
inline int64_t part_workspace(int64_t n, int32_t k, int32_t top) {
    if (k <= 16384) return 0;
    const int64_t whole = (k + 16383) / 16384, halves = std::min<int64_t>(kMostParts, (k + 8191) / 8192);
    const int64_t most = kPartBytes / part_bytes(top) + 1, rows = std::min(n, most);  // (products stay small)
    return std::min(kPartBytes, std::max(rows * whole, std::min<int64_t>(rows * halves, 2 * 4095)) * part_bytes(top));
}

// How scores of aligned 8-bit rows are made (microseconds at n x dim x k, bf16 results, of the kernels compared):
//   FEW        16 x 16 per workgroup, the components shared out among its waves: up to 32 tiles of 64 x 64, or 16 rows and 256 of them
//              (32 x 4096 x 1024 6.0, T64 9.1; 14 x 3136 x 9152 8.4 and 9.3; 600 x 6000 x 600 25 and 17)
//   T64        64 x 64, 256 components per barrier, four steps in flight: one workgroup per compute unit at most
//              (1024 x 4096 x 1024 10.7, T64_MANY 17.6, T128 18.5)
//   T64_MANY   64 x 64, 128 components per barrier, two steps: several workgroups per compute unit, where 128 codes would be half
//              empty (84,654 x 188 x 24 8.7, T64_128 11.4, T128_MANY 10.8)
//   T64_128    64 rows x 128 codes, three steps: where they leave a compute unit one workgroup (1200 x 2000 x 1200 10.1, T64 14.6,
//              T128 13.5), and up to 64 rows (64 x 1280 x 65,536 19.8, T64_MANY 22.9, T128_MANY 21.3)
//   T128       128 x 128, four steps: one workgroup per compute unit (4099 x 1000 x 777 11.4, T64_MANY 13.1, T128_MANY 12.0)
//   T256       256 x 256: two per compute unit and more than 256 components, or one and many steps (8192 x 8192 x 8192 469,
//              T128_MANY 536; 4096 x 4096 x 4096 66 and 79; 100,000 x 384 x 1024 107 and 116)
//   T128_MANY  128 x 128, two steps, several workgroups per compute unit: the others (1247 x 27 x 16,682 16.4, T256 20.4;
//              1M x 128 x 256 173 and 179; 100,000 x 128 x 256 20.6 and 24.1)
// Places within a tile's rows are counted in 32 bits: strides up to 2^22.
enum ScoreWay { FEW, T64, T64_MANY, T64_128, T128, T256, T128_MANY };
constexpr int64_t kMaxTileStride = 1 << 22;
inline ScoreWay score_way(int64_t n, int32_t k, int32_t dim) {
    const auto tiles = [&](int r, int c) { return ((n + r - 1) / r) * ((k + c - 1) / c); };
    if (tiles(64, 64) <= 32 || (n <= 16 && tiles(64, 64) <= 256)) return FEW;
    if (tiles(64, 64) <= 256) return T64;
    if (k <= 64) return T64_MANY;
    if (n <= 64 || tiles(64, 128) <= 256) return T64_128;
    if (tiles(128, 128) <= 256) return T128;
    if (n > 128 && ((tiles(256, 256) >= 512 && dim > 256) || (tiles(256, 256) >= 256 && dim >= 1024))) return T256;
    return T128_MANY;
}
// Rows at other addresses or strides: through k_scores_any, which takes them as they are; where there is more than 2^28 to
// multiply and 32 rows and codes or more, they are copied to aligned rows first (4096 x 4099 x 4096 at a stride of 4099 282 us, 90 so; about
// 2^28: 256 x 1000 x 1000 at 1001 14.3 and 11.6, 512 x 100 x 5000 at 101 10.5 and 10.9), up to 1 GiB of codes, and of rows as many at a time
// as make 512 MiB.  The line at 32 is not where the two meet: of 1 to 31 rows at a stride of 1000 against 65,536 aligned codes the copy would
// take 2 to 3 us off 18 to 20, while 32 and 64 such rows against as many codes at that stride take 44, as they are 20 and 26.
constexpr int64_t kPackRows = 512 << 20, kPackCodes = 1 << 30;
inline int64_t packed_stride(int32_t dim) { return (dim + 15) / 16 * 16; }
inline bool score_pack(int64_t n, int32_t k, int32_t dim) {
    return n >= 32 && k >= 32 && k * packed_stride(dim) <= kPackCodes && (double)n * k * dim >= 0x1p28;
}
// Rows of a launch: fewer than 2^22 tiles of 64 x 64, and no more tiles of rows than a grid's second dimension holds.
inline int64_t score_rows_of_a_launch(int32_t k) {
    return 64 * std::min<int64_t>(65535, std::max<int64_t>(1, (1 << 22) / ((k + 63) / 64)));
}

// Lanes and vectors of 16 bytes per lane that hold a row of `length` values in registers: 4 lanes with one vector or four, 8 with four, 64 with
// one or four, a workgroup with eight; lanes 0: none does.  Short rows have few lanes, so that a wave shares what a row costs beside its values,
// two divisions most of all, among 16 or 8 of them (1M rows of 128 f32 102 us with 8 lanes, 202 with 64; of 24 bf16 23 with 4, 71 with 16).
struct LanePlan {
    int lanes, vectors;
};
inline LanePlan plan_lanes(int32_t length, int bytes) {
    const int vec = 16 / bytes;
    if (length < vec || length > 2048 * vec) return {0, 0};
    if (length <= 16 * vec) return {4, length <= 4 * vec ? 1 : 4};
    if (length <= 32 * vec) return {8, 4};
    if (length <= 256 * vec) return {64, length <= 64 * vec ? 1 : 4};
    return {256, 8};
}

}  // namespace vq
