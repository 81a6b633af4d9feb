// What the calls of models over codes (tables of vectors, distillation, verification of drafts) take and refuse, and how their
// work is shared out: rules on sizes, strides and addresses alone, without HIP, so that a CPU test can go through them.
#pragma once
#include "score_rules.hpp"

namespace vq {

constexpr int32_t kMaxStages = 64;      // codes of a position
constexpr int32_t kMaxEmbedDim = 1 << 20;
constexpr int32_t kMaxTeacher = 64;     // a teacher's alternatives of a row: a lane each
constexpr int32_t kMaxDraft = 63;       // drafted codes of a sequence: with the code that comes next a lane each

inline Refusal check_code_array(const void *codes, int32_t code_bytes, int64_t n, int64_t code_stride, int32_t row) {
    if (code_bytes != 1 && code_bytes != 2 && code_bytes != 4) return refuse(VQ_ERR_INVALID_ARG, "codes have 1, 2 or 4 bytes");
    if (code_stride < row || too_long(n, code_stride, code_bytes)) return refuse(VQ_ERR_INVALID_ARG, "stride of the codes");
    if (misaligned(codes, code_bytes)) return refuse(VQ_ERR_INVALID_ARG, "misaligned pointer");
    return {};
}

// Sizes of a table and of the rows that are read from it or summed into it.
inline Refusal check_table(int32_t type, int32_t out_type, int64_t n, int32_t k, int32_t dim, int32_t m, int64_t ld_table, int64_t ld_rows,
                           int table_bytes, int row_bytes, float scale) {
    if (!type_bytes(type) || !type_bytes(out_type)) return refuse(VQ_ERR_INVALID_ARG, "no such type");
    if (n < 0 || k <= 0 || dim <= 0 || m <= 0) return refuse(VQ_ERR_INVALID_ARG, "n must not be negative, k, dim and m must be greater than 0");
    if (k > kMaxRowCodes) return refuse(VQ_ERR_UNSUPPORTED, "k must be at most 1048576");
    if (dim > kMaxEmbedDim) return refuse(VQ_ERR_UNSUPPORTED, "dim must be at most 1048576");
    if (m > kMaxStages) return refuse(VQ_ERR_UNSUPPORTED, "m must be at most 64");
    if (ld_table < dim || ld_rows < dim) return refuse(VQ_ERR_INVALID_ARG, "a row stride is below dim");
    if (too_long((int64_t)m * k, ld_table, table_bytes) || too_long(n, ld_rows, row_bytes))
        return refuse(VQ_ERR_INVALID_ARG, "rows and stride overflow");
    if (!(scale >= -3.402823466e38f && scale <= 3.402823466e38f)) return refuse(VQ_ERR_INVALID_ARG, "scale must be finite");
    return {};
}

inline Refusal check_code_embed(int32_t type, const void *table, int32_t k, int64_t ld_table, int32_t dim, int32_t m, int32_t code_bytes,
                                const void *codes, int64_t n, int64_t code_stride, float scale, int32_t out_type, const void *out, int64_t ld_out) {
    const int e = type_bytes(type), o = type_bytes(out_type);
    Refusal r = check_table(type, out_type, n, k, dim, m, ld_table, ld_out, e, o, scale);
    if (r.status == VQ_OK) r = check_code_array(codes, code_bytes, n, code_stride, m);
    if (r.status != VQ_OK || n == 0) return r;
    if (!table || !codes || !out) return refuse(VQ_ERR_INVALID_ARG, "null pointer");
    if (misaligned(table, e) || misaligned(out, o)) return refuse(VQ_ERR_INVALID_ARG, "misaligned pointer");
    const Span so(out, n, ld_out * o, (int64_t)dim * o);
    if (so.meets({table, (int64_t)m * k, ld_table * e, (int64_t)dim * e}) || so.meets({codes, n, code_stride * code_bytes, (int64_t)m * code_bytes}))
        return refuse(VQ_ERR_INVALID_ARG, "the output overlaps an input");
    return {};
}

inline Refusal check_code_embed_grad(int32_t type, const void *g, int64_t n, int64_t ld_g, int32_t dim, int32_t m, int32_t code_bytes,
                                     const void *codes, int64_t code_stride, float scale, int32_t k, int32_t accumulate, int32_t grad_type,
                                     const void *grad, int64_t ld_grad) {
    const int e = type_bytes(type), o = type_bytes(grad_type);
    Refusal r = check_table(type, grad_type, n, k, dim, m, ld_grad, ld_g, o, e, scale);
    if (r.status == VQ_OK) r = check_code_array(codes, code_bytes, n, code_stride, m);
    if (r.status != VQ_OK) return r;
    if (n > ((int64_t)1 << 30) / m) return refuse(VQ_ERR_UNSUPPORTED, "n * m must be at most 2^30");
    if (accumulate != 0 && accumulate != 1) return refuse(VQ_ERR_INVALID_ARG, "accumulate is 0 or 1");
    if (n == 0 && accumulate) return {};
    if (!grad || (n > 0 && (!g || !codes))) return refuse(VQ_ERR_INVALID_ARG, "null pointer");
    if (misaligned(g, e) || misaligned(grad, o)) return refuse(VQ_ERR_INVALID_ARG, "misaligned pointer");
    const Span so(grad, (int64_t)m * k, ld_grad * o, (int64_t)dim * o);
    if (so.meets({g, n, ld_g * e, (int64_t)dim * e}) || so.meets({codes, n, code_stride * code_bytes, (int64_t)m * code_bytes}))
        return refuse(VQ_ERR_INVALID_ARG, "the gradient overlaps an input");
    return {};
}

// What both calls on a teacher's alternatives take.
inline Refusal check_teacher(int32_t type, const void *s, int64_t n, int64_t ld, int32_t k, float beta, int32_t top, const void *lp,
                             const void *code, int64_t ld_teacher, int32_t rest) {
    const Refusal r = check_scored_codes(type, s, n, ld, k, beta, 4, nullptr, 1);
    if (r.status != VQ_OK) return r;
    if (top <= 0) return refuse(VQ_ERR_INVALID_ARG, "top must be greater than 0");
    if (top > kMaxTeacher) return refuse(VQ_ERR_UNSUPPORTED, "top must be at most 64");
    if (ld_teacher < top || too_long(n, ld_teacher, 4)) return refuse(VQ_ERR_INVALID_ARG, "stride of the teacher's alternatives");
    if (rest != 0 && rest != 1) return refuse(VQ_ERR_INVALID_ARG, "rest is 0 or 1");
    if (n == 0) return {};
    if (!lp || !code) return refuse(VQ_ERR_INVALID_ARG, "null pointer");
    if (misaligned(lp, 4) || misaligned(code, 4)) return refuse(VQ_ERR_INVALID_ARG, "misaligned pointer");
    return {};
}
// The gradient of the scores: in place, or apart from all that is read (and, in the same call, from what else is written).
inline Refusal check_score_grad(int32_t type, const void *s, int64_t n, int64_t ld, int32_t k, int32_t top, const void *lp, const void *code,
                                int64_t ld_teacher, const void *g, const void *grad, int64_t ld_grad) {
    const int e = type_bytes(type);
    if (ld_grad < k || too_long(n, ld_grad, e)) return refuse(VQ_ERR_INVALID_ARG, "stride of the gradient");
    if (n == 0) return {};
    if (!g || !grad) return refuse(VQ_ERR_INVALID_ARG, "null pointer");
    if (misaligned(g, 4) || misaligned(grad, e)) return refuse(VQ_ERR_INVALID_ARG, "misaligned pointer");
    const Span sg(grad, n, ld_grad * e, (int64_t)k * e);
    if (sg.meets({lp, n, ld_teacher * 4, top * 4}) || sg.meets({code, n, ld_teacher * 4, top * 4}) || sg.meets({g, 1, 0, n * 4}))
        return refuse(VQ_ERR_INVALID_ARG, "the gradient overlaps an input");
    if (!(grad == s && ld_grad == ld) && sg.meets({s, n, ld * e, (int64_t)k * e}))
        return refuse(VQ_ERR_INVALID_ARG, "the gradient overlaps the scores otherwise than in place");
    return {};
}

inline Refusal check_code_distill(int32_t type, const void *s, int64_t n, int64_t ld, int32_t k, float beta, int32_t top, const void *lp,
                                  const void *code, int64_t ld_teacher, int32_t rest, const void *loss, const void *max, const void *logsum,
                                  const void *logrest, const void *g, const void *grad, int64_t ld_grad) {
    Refusal r = check_teacher(type, s, n, ld, k, beta, top, lp, code, ld_teacher, rest);
    if (r.status != VQ_OK) return r;
    if ((g == nullptr) != (grad == nullptr)) return refuse(VQ_ERR_INVALID_ARG, "a gradient and the gradients of the losses go together");
    if (grad) r = check_score_grad(type, s, n, ld, k, top, lp, code, ld_teacher, g, grad, ld_grad);
    if (r.status != VQ_OK || n == 0) return r;
    const int e = type_bytes(type);
    const void *outs[] = {loss, max, logsum, logrest};
    const Span in[] = {{s, n, ld * e, (int64_t)k * e}, {lp, n, ld_teacher * 4, top * 4}, {code, n, ld_teacher * 4, top * 4}, {g, 1, 0, n * 4},
                       {grad, n, ld_grad * e, (int64_t)k * e}};
    for (int a = 0; a < 4; ++a) {
        if (misaligned(outs[a], 4)) return refuse(VQ_ERR_INVALID_ARG, "misaligned pointer");
        const Span oa(outs[a], 1, 0, n * 4);
        for (int b = 0; b < a; ++b)
            if (oa.meets({outs[b], 1, 0, n * 4})) return refuse(VQ_ERR_INVALID_ARG, "an output overlaps another array");
        for (const Span &i : in)
            if (oa.meets(i)) return refuse(VQ_ERR_INVALID_ARG, "an output overlaps another array");
    }
    return {};
}

inline Refusal check_code_distill_grad(int32_t type, const void *s, int64_t n, int64_t ld, int32_t k, float beta, int32_t top, const void *lp,
                                       const void *code, int64_t ld_teacher, int32_t rest, const void *max, const void *logsum,
                                       const void *logrest, const void *g, const void *grad, int64_t ld_grad) {
    Refusal r = check_teacher(type, s, n, ld, k, beta, top, lp, code, ld_teacher, rest);
    if (r.status == VQ_OK) r = check_score_grad(type, s, n, ld, k, top, lp, code, ld_teacher, g, grad, ld_grad);
    if (r.status != VQ_OK || n == 0) return r;
    if (!max || !logsum || (rest && !logrest)) return refuse(VQ_ERR_INVALID_ARG, "null pointer");
    const int e = type_bytes(type);
    const Span sg(grad, n, ld_grad * e, (int64_t)k * e);
    for (const void *p : {max, logsum, rest ? logrest : nullptr}) {
        if (misaligned(p, 4)) return refuse(VQ_ERR_INVALID_ARG, "misaligned pointer");
        if (sg.meets({p, 1, 0, n * 4})) return refuse(VQ_ERR_INVALID_ARG, "the gradient overlaps an input");
    }
    return {};
}

inline Refusal check_code_verify(int32_t type, const void *target, int64_t ld_target, float beta, const void *drafts, int64_t ld_draft,
                                 float beta_draft, int64_t n, int32_t draft, int32_t k, int32_t code_bytes, const void *codes, int64_t code_stride,
                                 const void *uniform, int64_t ld_uniform, const void *accepted, const void *out, int64_t ld_out) {
    const int e = type_bytes(type);
    if (!e) return refuse(VQ_ERR_INVALID_ARG, "no such type");
    if (n < 0 || draft < 0 || k <= 0) return refuse(VQ_ERR_INVALID_ARG, "n and draft must not be negative and k must be greater than 0");
    if (k > kMaxRowCodes) return refuse(VQ_ERR_UNSUPPORTED, "k must be at most 1048576");
    if (draft > kMaxDraft) return refuse(VQ_ERR_UNSUPPORTED, "draft must be at most 63");
    if (n > (int64_t)1 << 30) return refuse(VQ_ERR_UNSUPPORTED, "n must be at most 2^30");
    if (ld_target < k || (drafts && ld_draft < k)) return refuse(VQ_ERR_INVALID_ARG, "the row stride is below k");
    if (too_long(n * (draft + 1), ld_target, e) || (drafts && too_long(n * (draft + 1), ld_draft, e)))
        return refuse(VQ_ERR_INVALID_ARG, "rows and stride overflow");
    if (!(beta >= 1e-30f) || !(beta <= 1e30f)) return refuse(VQ_ERR_INVALID_ARG, "beta must be between 1e-30 and 1e30");
    if (drafts && (!(beta_draft >= 1e-30f) || !(beta_draft <= 1e30f)))
        return refuse(VQ_ERR_INVALID_ARG, "beta of the drafts must be between 1e-30 and 1e30");
    if (draft > 0) {
        const Refusal r = check_code_array(codes, code_bytes, n, code_stride, draft);
        if (r.status != VQ_OK) return r;
    }
    if (ld_uniform < draft + 1 || ld_out < draft + 1 || too_long(n, ld_uniform, 4) || too_long(n, ld_out, 4))
        return refuse(VQ_ERR_INVALID_ARG, "stride of the random numbers or of the output");
    if (n == 0) return {};
    if (!target || !uniform || !accepted || !out || (draft > 0 && !codes)) return refuse(VQ_ERR_INVALID_ARG, "null pointer");
    if (misaligned(target, e) || misaligned(drafts, e) || misaligned(uniform, 4) || misaligned(accepted, 4) || misaligned(out, 4))
        return refuse(VQ_ERR_INVALID_ARG, "misaligned pointer");
    const Span in[] = {{target, n * (draft + 1), ld_target * e, (int64_t)k * e}, {drafts, n * draft, ld_draft * e, (int64_t)k * e},
                       {draft > 0 ? codes : nullptr, n, code_stride * code_bytes, (int64_t)draft * code_bytes}, {uniform, n, ld_uniform * 4, (draft + 1) * 4}};
    const Span sa(accepted, 1, 0, n * 4), so(out, n, ld_out * 4, (draft + 1) * 4);
    if (sa.meets(so)) return refuse(VQ_ERR_INVALID_ARG, "an output overlaps another array");
    for (const Span &i : in)
        if (sa.meets(i) || so.meets(i)) return refuse(VQ_ERR_INVALID_ARG, "an output overlaps another array");
    return {};
}

// ---- rows of a table -----------------------------------------------------------------------------------
// Slices of the columns of a lookup: eight, an XCD's each, where rows of the tables are read many times (twice at least, on average) and a slice has
// 128 bytes of a row or more; otherwise one.
inline int embed_slices(int64_t n, int32_t k, int32_t m, int vectors) { return n >= 2 * (int64_t)k && vectors >= 64 && (int64_t)k * m * vectors * 16 > 2 << 20 ? 8 : 1; }

// Pieces of 16 bytes of a row that a lane has: two where the additions of several stages count more than the number of waves (65,536 x 8 stages
// of 1024 bf16 54 us with one, 49 with two; 4 stages 38 and 33; 16,384 x 8 stages 14.9 and 14.5).
inline int embed_pieces(int64_t n, int32_t m, int pieces) { return m >= 4 && pieces >= 16 && n * pieces >= 1 << 18 ? 2 : 1; }

// ---- sums by code ------------------------------------------------------------------------------------
// The positions of each stage in the order of their codes, and where each code's positions begin: k + 1 numbers.  Workgroups of 16 waves
// list a bucket of codes each, of a share of the positions.  One share, and one launch, up to 32,768 positions; more positions in shares, in two
// launches, of at most 1024 workgroups, two to a compute unit by their 62 KB of LDS and 8 beside (363,313 x 4 codes of 8379: 3204 workgroups, one to a
// compute unit, 31 + 174 us, so 19 + 50).  Where the buckets of all stages are more than 512 already there is one share again, and a workgroup per bucket.
// The line, of whole gradients of 32 columns: 256 codes, 16,000 positions 11.5 us in one share, 18.8 in several; 48,000 16.9 and 20.4; 130,000 29.6 and
// 24.6.  It is low for many codes: 65,536 codes, 32,000 20 and 48; 130,000 37 and 69.
// Every bucket's workgroup reads all codes of its share, n * m * k / 480 of them in all: next to nothing for 256 codes or for the 65,536 of a batch, but 1M
// positions of 262,144 codes take 0.27 ms for the list alone, of 2^20 codes 0.72, and 8 stages of 262,144 codes 7.6, where the sums take 0.05, 0.1 and 0.4.
struct ListPlan {
    int32_t width, buckets;
    int32_t share, shares;
};
constexpr int kBucketMost = 480, kOneShareMost = 512;  // codes of a bucket
constexpr int kListBeside = 2 * 16 * 4 + 2 * 1024 * 4; // LDS of a workgroup beside list_lds
constexpr int kListQueue = 256;                        // positions of a bucket that a wave keeps
// 16 waves' counts, and (to write the list) positions and codes of each wave.
constexpr int list_lds(int width, bool place) { return (16 * width + 1) / 2 * 8 + (place ? 16 * kListQueue * 8 : 0); }
inline ListPlan plan_lists(int64_t n, int32_t k, int32_t m) {
    if (n <= 32768) {
        const int32_t width = std::min<int32_t>(kOneShareMost, (k + 255) / 256);
        return {width, (k + width - 1) / width, (int32_t)std::max<int64_t>(n, 1), 1};
    }
    const int32_t width = std::min<int32_t>(kBucketMost, k), buckets = (k + width - 1) / width;
    // shares of 4096 positions or more, at most 256 of them
    const int64_t most = std::max<int64_t>(1, std::min<int64_t>(256, 1024 / ((int64_t)buckets * m))), share = std::max<int64_t>(4096, (n + most - 1) / most);
    return {width, buckets, (int32_t)share, (int32_t)((n + share - 1) / share)};
}
// Up to so many positions the workgroups that sum make their lists themselves, for 4 codes each, or 16 or 64 where that would be more workgroups than
// 512 to read all codes, 1024 at most (333 x 100 f32, 1001 codes: 9.8 us in two launches, 6.8 so; 759 x 2 stages of 175 f16, 12,388 codes 24
// and 9).  0: the lists come first.
constexpr int kFewPositions = 1024, kFewCodes = 64;
inline int embed_few(int64_t n, int32_t k, int32_t m, int64_t across) {
    const auto groups = [&](int codes) { return (k + codes - 1) / codes * (int64_t)m * across; };
    return n > kFewPositions ? 0 : groups(4) <= 512 ? 4 : groups(16) <= 512 ? 16 : groups(kFewCodes) <= 1024 ? kFewCodes : 0;
}
// A code of more positions than this is summed in pieces of as many positions of the list, whose sums are joined afterwards.
constexpr int kLongCode = 1024;
constexpr int64_t embed_edges(int64_t n) { return (n + kLongCode - 1) / kLongCode; }  // pieces of the list
inline int64_t embed_chunks(int64_t n) { return n > kLongCode ? embed_edges(n) : 0; }
// Bytes of a call's workspace, in the order in which they lie there; their sum grows with each size.
struct EmbedWork {
    int64_t start, rows, edges, counts, below, partial, bytes;
};
inline EmbedWork embed_work(int64_t n, int32_t k, int32_t dim, int32_t m) {
    const auto up = [](int64_t b) { return (b + 255) / 256 * 256; };
    // (shares times codes: no plan has more than 256 shares, nor more than 1024 of share and bucket)
    const int64_t counts = n > 32768 ? std::min<int64_t>(256 * (int64_t)k, (int64_t)1024 * kBucketMost + k) : 0, belows = n > 32768 ? 4096 : 0;
    EmbedWork w;
    w.start = 0;
    w.rows = up((int64_t)m * (k + 1) * 4);
    w.edges = w.rows + up(m * n * 4);
    w.counts = w.edges + up(m * embed_edges(n) * 4);
    w.below = w.counts + up(m * counts * 4);
    w.partial = w.below + up(m * belows * 4);
    w.bytes = w.partial + up(m * embed_chunks(n) * 2 * ((dim + 15) / 16 * 16) * 4);
    return w;
}

// ---- rows of scores against a teacher ------------------------------------------------------------------
// How a row of k scores goes through the GPU: by `waves` waves that hold it whole, 64 * per_lane codes each, or (waves 0) in parts of
// 256 * per_lane codes, a workgroup each.
struct DistillPlan {
    int waves, per_lane;
    int32_t parts;
};
// Where the gradient comes along 64 rows or more have sixteen waves each: 65,536 bf16, 256 rows 16.8 us, 29.3 in parts; 64 rows 12.0 and 16.2.  The line is
// high: 48 rows 11.8 and 15.5, 16 rows 11.3 and 14.0, 8 rows 11.1 and 11.4; of 20,000 codes 8 rows 7.2 and 11.2.
inline DistillPlan plan_distill(int64_t n, int32_t k, bool grad) {
    if (k <= 4096) return {1, k <= 512 ? 8 : k <= 1024 ? 16 : k <= 2048 ? 32 : 64, 1};
    if (k <= 16384) return {4, k <= 8192 ? 32 : 64, 1};
    if (grad && k <= 65536 && n >= 64) return {16, k <= 32768 ? 32 : 64, 1};
    const int64_t whole = (k + 16383) / 16384;
    const int e = n * whole < 4096 && k <= kMostParts * 8192 ? 32 : 64;
    return {0, e, (k + 256 * e - 1) / (256 * e)};
}
// Rows of a launch (a grid has fewer than 2^32 lanes) and bytes of the parts' results, which lie beside one another for a launch's rows.
// (and, behind them, five numbers per row for the gradient)
constexpr int kDistillPartBytes = 8, kDistillRowBytes = 20;
inline int64_t distill_rows_of_a_launch(const DistillPlan &p) {
    return p.waves == 1 ? (int64_t)1 << 25 : p.waves ? ((int64_t)1 << 24) / (p.waves * 2) : std::max<int64_t>(1, (kPartBytes / kDistillPartBytes) / p.parts);
}
inline int64_t distill_work(int64_t n, int32_t k) {
    if (k <= 16384) return 0;
    const int64_t most = (k + 8191) / 8192;  // (no plan cuts a row into more, and none into fewer than two: a launch's rows have at most 2.25 kPartBytes)
    return std::min<int64_t>(3 * kPartBytes, std::min(n, kPartBytes) * (most * kDistillPartBytes + kDistillRowBytes));
}

// ---- drafts --------------------------------------------------------------------------------------------
// Rows of scores are cut into parts of 4096 codes, a workgroup each, or four to a workgroup where those are enough; a sequence has draft + 1 rows of its
// own and as many as drafts of its drafts'.
constexpr int kVerifyPart = 4096;
inline int32_t verify_parts(int32_t k) { return (k + kVerifyPart - 1) / kVerifyPart; }
// Rows of up to 2048 codes: a workgroup per sequence does everything, unless a few sequences have many rows each.
inline bool verify_few(int64_t n, int32_t draft, int32_t k) { return k <= 2048 && (draft <= 16 || n >= 512); }
// Four parts to a workgroup, 11 rows a sequence: 65,536 bf16, 32 sequences 36.1 us and 33.8 a part each; 64 52.6 and 53.9; 256 160 and 174.  Of 4097 to
// 8192 codes half of such a workgroup's lanes have none: 256 sequences 49 and 34.
inline bool verify_wide(int64_t rows, int32_t k) { return k > kVerifyPart && rows * ((k + 4 * kVerifyPart - 1) / (4 * kVerifyPart)) >= 2048; }
// Per row and part a sum in 64 bits and two maxima in 32; per sequence and part a sum more, and 64 bytes for what its drafts come to.
inline int64_t verify_bytes_of_a_sequence(int32_t draft, int32_t k) { return (int64_t)verify_parts(k) * ((2 * draft + 1) * 16 + 8) + 64; }
static_assert(kMaxRowCodes / kVerifyPart * ((2 * kMaxDraft + 1) * 16 + 8) + 64 <= kPartBytes * 4, "one sequence fits");
inline int64_t verify_sequences_of_a_launch(int32_t draft, int32_t k) {
    return std::max<int64_t>(1, std::min((kPartBytes * 4) / verify_bytes_of_a_sequence(draft, k), ((int64_t)1 << 23) / (verify_parts(k) * (2 * draft + 1))));
}
inline int64_t verify_work(int64_t n, int32_t draft, int32_t k) {
    return std::min(std::min(n, kPartBytes) * verify_bytes_of_a_sequence(draft, k), kPartBytes * 4);  // (at least one sequence's)
}

}  // namespace vq
