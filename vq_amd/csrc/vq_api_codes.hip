// C entry points of models over codes: tables of vectors, distillation, verification of drafts.
#include "code_distill.hpp"
#include "code_embed.hpp"
#include "code_rules.hpp"
#include "code_verify.hpp"
#include "score_calls.hpp"

using namespace vqh;

namespace {

// f(T, O) with the types of two arrays
template <typename F> void by_types(int32_t type, int32_t other, F f) {
    by_type(type, [&](auto t) { by_type(other, [&](auto o) { f(t, o); }); });
}

// f(integral constant) with the bytes of a code
template <typename F> void by_bytes(int32_t bytes, F f) {
    if (bytes == 1)
        f(std::integral_constant<int, 1>());
    else if (bytes == 2)
        f(std::integral_constant<int, 2>());
    else
        f(std::integral_constant<int, 4>());
}

// Sums by code: 16 bytes of a row per lane, or a value where a row has fewer.
template <typename T, typename O, bool FEW> void embed_sums(vq_ctx *ctx, const vq::SumArgs &a, unsigned groups, int m) {
    if (a.dim < vq::wide<T>())
        hipLaunchKernelGGL((vq::k_embed_sums<T, O, 1, FEW>), dim3(groups, 1, m), dim3(256), 0, ctx->stream, a);
    else
        hipLaunchKernelGGL((vq::k_embed_sums<T, O, vq::wide<T>(), FEW>), dim3(groups, 1, m), dim3(256), 0, ctx->stream, a);
}

// The alternatives' rows of a launch, from row r on.
vq::DistillArgs distill_slice(const vq::DistillArgs &a, int64_t r, int64_t rows, int e) {
    vq::DistillArgs s = a;
    const auto at = [&](float *p) { return p ? p + r : nullptr; };
    s.s = (const char *)a.s + r * a.ld * e;
    s.n = std::min(rows, a.n - r);
    s.lp = a.lp + r * a.ld_teacher;
    s.code = a.code + r * a.ld_teacher;
    s.loss = at(a.loss), s.max = at(a.max), s.logsum = at(a.logsum), s.logrest = at(a.logrest);
    s.rest_max = at(a.rest_max), s.rest_sum = at(a.rest_sum);
    s.g = a.g ? a.g + r : nullptr;
    s.grad = a.grad ? (char *)a.grad + r * a.ld_grad * e : nullptr;
    return s;
}

int32_t distill_grad(vq_ctx *ctx, int32_t type, const vq::DistillArgs &all) {
    const int64_t slice = (int64_t)1 << 22;  // rows per launch: a grid has fewer than 2^32 lanes
    for (int64_t r = 0; r < all.n; r += slice) {
        const vq::DistillArgs a = distill_slice(all, r, slice, vq::type_bytes(type));
        by_type(type, [&](auto t) {
            typedef decltype(t) T;
            constexpr int VEC = 16 / (int)sizeof(typename T::Raw);
            const auto waves = dim3((unsigned)cdiv64(a.n, 4));
            if (a.k <= 512)
                hipLaunchKernelGGL((vq::k_distill_grad<T, 1, 8 / VEC>), waves, dim3(256), 0, ctx->stream, a);
            else if (a.k <= 1024)
                hipLaunchKernelGGL((vq::k_distill_grad<T, 1, 16 / VEC>), waves, dim3(256), 0, ctx->stream, a);
            else if (a.k <= 2048)
                hipLaunchKernelGGL((vq::k_distill_grad<T, 1, 32 / VEC>), waves, dim3(256), 0, ctx->stream, a);
            else
                hipLaunchKernelGGL((vq::k_distill_grad<T, 4, 32 / VEC>), dim3((unsigned)a.n, (unsigned)cdiv(a.k, 256 * 32)), dim3(256), 0, ctx->stream, a);
        });
        VQ_HIP(ctx, hipGetLastError());
    }
    return VQ_OK;
}

}  // namespace

extern "C" {

int32_t vq_code_embed(vq_ctx *ctx, int32_t type, const void *d_table, int32_t k, int64_t ld_table, int32_t dim, int32_t m,
                      int32_t code_bytes, const void *d_codes, int64_t n, int64_t code_stride, float scale, int32_t out_type,
                      void *d_out, int64_t ld_out) {
    if (!ctx) return VQ_ERR_INVALID_ARG;
    bool go;
    VQ_TRY(admit(ctx, vq::check_code_embed(type, d_table, k, ld_table, dim, m, code_bytes, d_codes, n, code_stride, scale, out_type,
                                           d_out, ld_out), n, &go));
    if (!go) return VQ_OK;
    const int wide = 16 / vq::type_bytes(type), vectors = dim < wide ? dim : cdiv(dim, wide), slices = vq::embed_slices(n, k, m, vectors), pieces = cdiv(vectors, slices);
    const bool near = k <= 0xffffffffll / ld_table / vq::type_bytes(type) && ld_table * vq::type_bytes(type) < 1 << 24;  // (places in bytes of a stage's table fit 32 bits)
    const int each = near ? vq::embed_pieces(n, m, pieces) : 1;
    int shift = 0;
    while (shift < 8 && each << shift < pieces) ++shift;
    const unsigned across = cdiv(pieces, each << shift);
    const int64_t slice = std::max<int64_t>(256, ((int64_t)1 << 31) / ((int64_t)slices << shift));  // a grid has fewer than 2^32 lanes
    for (int64_t r = 0; r < n; r += slice) {
        const vq::EmbedArgs a{d_table, ld_table, k, dim, m, (const char *)d_codes + r * code_stride * code_bytes, code_bytes, std::min(slice, n - r),
                              code_stride, scale, (char *)d_out + r * ld_out * vq::type_bytes(out_type), ld_out};
        by_types(type, out_type, [&](auto t, auto o) {
            typedef decltype(t) T;
            typedef decltype(o) O;
            const dim3 grid((unsigned)cdiv64(a.n, 256 >> shift) * slices, across);
            const auto go = [&](auto bytes) {
                constexpr int BYTES = decltype(bytes)::value;
                if (dim < vq::wide<T>())
                    hipLaunchKernelGGL((vq::k_code_embed<T, O, 1, 1, BYTES, int64_t>), grid, dim3(256), 0, ctx->stream, a, shift, slices, pieces);
                else if (near && each == 2)
                    hipLaunchKernelGGL((vq::k_code_embed<T, O, vq::wide<T>(), 2, BYTES, uint32_t>), grid, dim3(256), 0, ctx->stream, a, shift, slices, pieces);
                else if (near)
                    hipLaunchKernelGGL((vq::k_code_embed<T, O, vq::wide<T>(), 1, BYTES, uint32_t>), grid, dim3(256), 0, ctx->stream, a, shift, slices, pieces);
                else
                    hipLaunchKernelGGL((vq::k_code_embed<T, O, vq::wide<T>(), 1, BYTES, int64_t>), grid, dim3(256), 0, ctx->stream, a, shift, slices, pieces);
            };
            by_bytes(code_bytes, go);
        });
        VQ_HIP(ctx, hipGetLastError());
    }
    return VQ_OK;
}

int32_t vq_code_embed_grad(vq_ctx *ctx, int32_t type, const void *d_g, int64_t n, int64_t ld_g, int32_t dim, int32_t m,
                           int32_t code_bytes, const void *d_codes, int64_t code_stride, float scale, int32_t k, int32_t accumulate,
                           int32_t grad_type, void *d_grad, int64_t ld_grad) {
    if (!ctx) return VQ_ERR_INVALID_ARG;
    bool go;
    // (without rows the gradient is still written)
    VQ_TRY(admit(ctx, vq::check_code_embed_grad(type, d_g, n, ld_g, dim, m, code_bytes, d_codes, code_stride, scale, k, accumulate,
                                                grad_type, d_grad, ld_grad), accumulate ? n : 1, &go));
    if (!go) return VQ_OK;
    const int wide = 16 / vq::type_bytes(type), columns = 16 * (dim < wide ? 1 : wide), across = cdiv(dim, columns);
    if (const int few = vq::embed_few(n, k, m, across)) {
        vq::SumArgs a{d_g, ld_g, (int)n, dim, k, scale, accumulate, d_grad, ld_grad, d_codes, code_bytes, code_stride, nullptr, nullptr, nullptr, nullptr,
                      0, 0, few, (int)cdiv(k, few), across, 0};
        by_types(type, grad_type, [&](auto t, auto o) {
            embed_sums<decltype(t), decltype(o), true>(ctx, a, a.groups * across, m);
        });
        VQ_HIP(ctx, hipGetLastError());
        return VQ_OK;
    }
    const vq::EmbedWork work = vq::embed_work(n, k, dim, m);
    VQ_TRY(ensure_kept(ctx, ctx->code_work, (size_t)work.bytes));
    char *w = (char *)ctx->code_work.p;
    const vq::ListPlan plan = vq::plan_lists(n, k, m);
    const vq::ListArgs l{d_codes, code_stride, (int)n, k, plan.width, plan.share, plan.shares, (int32_t *)(w + work.start),
                         (int32_t *)(w + work.rows), (int32_t *)(w + work.edges), (int32_t *)(w + work.counts), (int32_t *)(w + work.below)};
    const auto lists = [&](auto bytes) -> int32_t {
        constexpr int BYTES = decltype(bytes)::value;
        const dim3 grid(plan.buckets, plan.shares, m), wg(1024);
        const int lds = vq::list_lds(plan.width, true), count_lds = vq::list_lds(plan.width, false);
        const int bit = 1 << (2 * (BYTES >> 1) + (plan.shares == 1));
        if (!(ctx->list_lds_set & bit)) {  // more than 64 KB
            const auto kernel = plan.shares == 1 ? vq::k_code_lists<16, BYTES, true, true> : vq::k_code_lists<16, BYTES, false, true>;
            VQ_HIP(ctx, hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize,
                                            vq::list_lds(vq::kOneShareMost, true)));
            ctx->list_lds_set |= bit;
        }
        if (plan.shares == 1) {
            hipLaunchKernelGGL((vq::k_code_lists<16, BYTES, true, true>), grid, wg, lds, ctx->stream, l);
        } else {
            hipLaunchKernelGGL((vq::k_code_lists<16, BYTES, true, false>), grid, wg, count_lds, ctx->stream, l);
            hipLaunchKernelGGL((vq::k_code_lists<16, BYTES, false, true>), grid, wg, lds, ctx->stream, l);
        }
        VQ_HIP(ctx, hipGetLastError());
        return VQ_OK;
    };
    int32_t rc = VQ_OK;
    by_bytes(code_bytes, [&](auto bytes) { rc = lists(bytes); });
    VQ_TRY(rc);
    // codes of a workgroup: as many as leave 2048 workgroups, at most 128
    const int codes = (int)std::min<int64_t>(128, std::max<int64_t>(1, (int64_t)k * m * across / 2048));
    vq::SumArgs a{d_g, ld_g, (int)n, dim, k, scale, accumulate, d_grad, ld_grad, nullptr, 0, 0, l.start, l.rows, l.edges, (float *)(w + work.partial),
                  (int)vq::embed_chunks(n), (dim + 15) / 16 * 16, codes, (int)cdiv(k, codes), 0, 0};
    // the columns of some workgroups side by side, the others' in launches of their own: a grid has fewer than 2^32 lanes
    const int most = std::max(1, (1 << 23) / (a.groups + a.chunks));
    for (a.first = 0; a.first < across; a.first += most) {
        a.across = std::min(most, across - a.first);
        // rows without members, all columns of them, behind the last columns' sums
        const bool last = a.first + a.across == across;
        const unsigned zeros = last && !accumulate ? cdiv(k, vq::kZeroCodes) * cdiv((int64_t)dim * vq::type_bytes(grad_type), vq::kZeroBytes) : 0;
        by_types(type, grad_type, [&](auto t, auto o) {
            embed_sums<decltype(t), decltype(o), false>(ctx, a, (a.groups + a.chunks) * a.across + zeros, m);
        });
        VQ_HIP(ctx, hipGetLastError());
    }
    if (a.chunks) {
        by_type(grad_type, [&](auto o) {
            hipLaunchKernelGGL(vq::k_embed_join<decltype(o)>, dim3(a.chunks, cdiv(dim, 64), m), dim3(256), 0, ctx->stream, a);
        });
        VQ_HIP(ctx, hipGetLastError());
    }
    return VQ_OK;
}

int32_t vq_code_distill(vq_ctx *ctx, int32_t type, const void *d_scores, int64_t n, int64_t ld, int32_t k, float beta, int32_t top,
                        const float *d_teacher_logprob, const int32_t *d_teacher_code, int64_t ld_teacher, int32_t rest, float *d_loss,
                        float *d_max, float *d_logsum, float *d_logrest, const float *d_g_loss, void *d_grad, int64_t ld_grad) {
    if (!ctx) return VQ_ERR_INVALID_ARG;
    bool go;
    VQ_TRY(admit(ctx, vq::check_code_distill(type, d_scores, n, ld, k, beta, top, d_teacher_logprob, d_teacher_code, ld_teacher, rest,
                                             d_loss, d_max, d_logsum, d_logrest, d_g_loss, d_grad, ld_grad), n, &go));
    if (!go) return VQ_OK;
    const vq::DistillPlan plan = vq::plan_distill(n, k, d_grad != nullptr);
    vq::DistillArgs all{d_scores, n, ld, k, beta, top, d_teacher_logprob, d_teacher_code, ld_teacher, rest, rest || d_logrest, d_loss, d_max, d_logsum,
                        d_logrest, d_g_loss, d_grad, ld_grad, plan.parts, nullptr, nullptr, nullptr};
    float *stats = nullptr;
    const int64_t slice = vq::distill_rows_of_a_launch(plan);
    VQ_TRY(ensure_kept(ctx, ctx->code_work, (size_t)vq::distill_work(n, k)));  // (also where fewer rows only would go in parts: they may follow in a capture)
    if (plan.waves == 0) {
        // the gradient of a row in parts is a call of its own, from the sums that the caller need not have asked for
        all.sums = (float *)ctx->code_work.p;
        stats = all.sums + std::min(slice, n) * plan.parts * 2;
    }
    for (int64_t r = 0; r < n; r += slice) {
        vq::DistillArgs a = distill_slice(all, r, slice, vq::type_bytes(type));
        if (plan.waves == 0 && a.grad) {
            if (!a.max) a.max = stats;
            if (!a.logsum) a.logsum = stats + std::min(slice, n);
            if (!a.logrest && rest) a.logrest = stats + 2 * std::min(slice, n);
            if (rest) a.rest_max = stats + 3 * std::min(slice, n), a.rest_sum = stats + 4 * std::min(slice, n);
        }
        by_type(type, [&](auto t) {
            typedef decltype(t) T;
            constexpr int VEC = 16 / (int)sizeof(typename T::Raw);
            const dim3 waves((unsigned)cdiv64(a.n, 4)), rows((unsigned)a.n), wg(256);
            if (plan.waves == 1 && plan.per_lane == 8)
                hipLaunchKernelGGL((vq::k_distill_row<T, 1, 8 / VEC>), waves, wg, 0, ctx->stream, a);
            else if (plan.waves == 1 && plan.per_lane == 16)
                hipLaunchKernelGGL((vq::k_distill_row<T, 1, 16 / VEC>), waves, wg, 0, ctx->stream, a);
            else if (plan.waves == 1 && plan.per_lane == 32)
                hipLaunchKernelGGL((vq::k_distill_row<T, 1, 32 / VEC>), waves, wg, 0, ctx->stream, a);
            else if (plan.waves == 1)
                hipLaunchKernelGGL((vq::k_distill_row<T, 1, 64 / VEC>), waves, wg, 0, ctx->stream, a);
            else if (plan.waves == 4 && plan.per_lane == 32)
                hipLaunchKernelGGL((vq::k_distill_row<T, 4, 32 / VEC>), rows, wg, 0, ctx->stream, a);
            else if (plan.waves == 4)
                hipLaunchKernelGGL((vq::k_distill_row<T, 4, 64 / VEC>), rows, wg, 0, ctx->stream, a);
            else if (plan.waves == 16 && plan.per_lane == 32)
                hipLaunchKernelGGL((vq::k_distill_row<T, 16, 32 / VEC>), rows, dim3(1024), 0, ctx->stream, a);
            else if (plan.waves == 16)
                hipLaunchKernelGGL((vq::k_distill_row<T, 16, 64 / VEC>), rows, dim3(1024), 0, ctx->stream, a);
            else {
                const dim3 parts((unsigned)(a.n * plan.parts));
                if (plan.per_lane == 32)
                    hipLaunchKernelGGL((vq::k_distill_part<T, 32 / VEC>), parts, wg, 0, ctx->stream, a);
                else
                    hipLaunchKernelGGL((vq::k_distill_part<T, 64 / VEC>), parts, wg, 0, ctx->stream, a);
                hipLaunchKernelGGL(vq::k_distill_join<T>, waves, wg, 0, ctx->stream, a);
            }
        });
        VQ_HIP(ctx, hipGetLastError());
        if (plan.waves == 0 && a.grad) VQ_TRY(distill_grad(ctx, type, a));
    }
    return VQ_OK;
}

int32_t vq_code_distill_grad(vq_ctx *ctx, int32_t type, const void *d_scores, int64_t n, int64_t ld, int32_t k, float beta, int32_t top,
                             const float *d_teacher_logprob, const int32_t *d_teacher_code, int64_t ld_teacher, int32_t rest,
                             const float *d_max, const float *d_logsum, const float *d_logrest, const float *d_g_loss, void *d_grad,
                             int64_t ld_grad) {
    if (!ctx) return VQ_ERR_INVALID_ARG;
    bool go;
    VQ_TRY(admit(ctx, vq::check_code_distill_grad(type, d_scores, n, ld, k, beta, top, d_teacher_logprob, d_teacher_code, ld_teacher,
                                                  rest, d_max, d_logsum, d_logrest, d_g_loss, d_grad, ld_grad), n, &go));
    if (!go) return VQ_OK;
    const vq::DistillArgs a{d_scores, n, ld, k, beta, top, d_teacher_logprob, d_teacher_code, ld_teacher, rest, rest, nullptr, const_cast<float *>(d_max),
                            const_cast<float *>(d_logsum), const_cast<float *>(d_logrest), d_g_loss, d_grad, ld_grad, 1, nullptr, nullptr, nullptr};
    return distill_grad(ctx, type, a);
}

int32_t vq_code_verify(vq_ctx *ctx, int32_t type, const void *d_target, int64_t ld_target, float beta, const void *d_draft,
                       int64_t ld_draft, float beta_draft, int64_t n, int32_t draft, int32_t k, int32_t code_bytes,
                       const void *d_codes, int64_t code_stride, const float *d_uniform, int64_t ld_uniform, int32_t *d_accepted,
                       int32_t *d_out, int64_t ld_out) {
    if (!ctx) return VQ_ERR_INVALID_ARG;
    bool go;
    VQ_TRY(admit(ctx, vq::check_code_verify(type, d_target, ld_target, beta, d_draft, ld_draft, beta_draft, n, draft, k, code_bytes,
                                            d_codes, code_stride, d_uniform, ld_uniform, d_accepted, d_out, ld_out), n, &go));
    if (!go) return VQ_OK;
    static_assert(sizeof(vq::Verdict) <= 64, "as the workspace counts it");
    static_assert(vq::kVerifyFew <= 256 * vq::kVerifyEach, "a workgroup's lanes have all of a row's weights");
    const int e = vq::type_bytes(type);
    const int64_t slice = vq::verify_sequences_of_a_launch(draft, k);
    const bool few = vq::verify_few(n, draft, k);
    if (!vq::verify_few(1, draft, k)) VQ_TRY(ensure_kept(ctx, ctx->code_work, (size_t)vq::verify_work(n, draft, k)));
    const void *drafts = draft > 0 ? d_draft : nullptr;
    for (int64_t b = 0; b < n; b += slice) {
        const int64_t here = std::min(slice, n - b), rows = here * (draft + 1 + (drafts ? draft : 0));
        const bool wide = vq::verify_wide(rows, k);
        const int parts = vq::verify_parts(k);
        double *sum = (double *)ctx->code_work.p, *left = sum + rows * parts;
        vq::Verdict *verdicts = (vq::Verdict *)(left + here * parts);
        float *most = (float *)(verdicts + here), *own = most + rows * parts;
        const vq::VerifyArgs a{(const char *)d_target + b * (draft + 1) * ld_target * e, drafts ? (const char *)drafts + b * draft * ld_draft * e : nullptr,
                               ld_target, ld_draft, beta * vq::kLog2e64, beta_draft * vq::kLog2e64, (int)here, draft, k, parts,
                               draft ? (const char *)d_codes + b * code_stride * code_bytes : nullptr, code_bytes, code_stride,
                               d_uniform + b * ld_uniform, ld_uniform, d_accepted + b, d_out + b * ld_out, ld_out, most, sum, own, left, verdicts};
        by_type(type, [&](auto t) {
            typedef decltype(t) T;
            const dim3 all((unsigned)(rows * (wide ? cdiv(parts, 4) : parts))), some((unsigned)(here * parts)), each((unsigned)here), wg(256);
            if (few) {
                hipLaunchKernelGGL(vq::k_verify_few<T>, each, wg, 0, ctx->stream, a);
            } else if (wide) {
                hipLaunchKernelGGL((vq::k_verify_part<T, 64>), all, wg, 0, ctx->stream, a);
                hipLaunchKernelGGL(vq::k_verify_verdict<T>, each, wg, 0, ctx->stream, a);
                if (drafts) hipLaunchKernelGGL((vq::k_verify_left<T, true>), some, wg, 0, ctx->stream, a);
                hipLaunchKernelGGL((vq::k_verify_pick<T, true>), each, wg, 0, ctx->stream, a);
            } else {
                hipLaunchKernelGGL((vq::k_verify_part<T, 16>), all, wg, 0, ctx->stream, a);
                if (drafts) {
                    hipLaunchKernelGGL((vq::k_verify_left<T, false>), some, wg, 0, ctx->stream, a);
                    hipLaunchKernelGGL((vq::k_verify_pick<T, true>), each, wg, 0, ctx->stream, a);
                } else
                    hipLaunchKernelGGL((vq::k_verify_pick<T, false>), each, wg, 0, ctx->stream, a);
            }
        });
        VQ_HIP(ctx, hipGetLastError());
    }
    return VQ_OK;
}

}  // extern "C"
