// C entry points of the 8-bit scores and the log probabilities of codes.
#include <algorithm>

#include "ctx.hpp"
#include "logprobs.hpp"
#include "score_rules.hpp"
#include "scores_i8.hpp"

using namespace vqh;

namespace {

int64_t cdiv64(int64_t a, int64_t b) { return (a + b - 1) / b; }

// A workspace that captured graphs may hold the address of: it grows by a new allocation, at least twice the last, and the
// ones before stay.  While the stream is being captured it cannot grow, and the capture goes on.
int32_t ensure_kept(vq_ctx *ctx, DevBuf &b, size_t bytes) {
    if (bytes <= b.cap) return VQ_OK;
    hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
    VQ_HIP(ctx, hipStreamIsCapturing(ctx->stream, &st));
    if (st != hipStreamCaptureStatusNone)
        return fail(ctx, VQ_ERR_UNSUPPORTED, "a capture of this call needs the same call to have run before: its workspace cannot grow meanwhile");
    const size_t want = bytes > 2 * b.cap ? bytes + 256 : 2 * b.cap;
    try {  // (no exception leaves a C entry point)
        ctx->outgrown.reserve(ctx->outgrown.size() + 1);
    } catch (...) {
        return fail(ctx, VQ_ERR_OOM, "no host memory for a table of workspaces");
    }
    void *p = nullptr;
    VQ_HIP(ctx, hipMalloc(&p, want));
    if (b.p) ctx->outgrown.push_back(b.p);
    b.p = p;
    b.cap = want;
    return VQ_OK;
}

// Refusals and calls without rows end the call; `go` says whether it runs.
int32_t admit(vq_ctx *ctx, const vq::Refusal &r, int64_t n, bool *go) {
    *go = false;
    if (r.status != VQ_OK) return fail(ctx, r.status, "Invalid parameter: %s", r.text);
    if (n == 0) return VQ_OK;
    VQ_HIP(ctx, hipSetDevice(ctx->device));
    *go = true;
    return VQ_OK;
}

// f(T) with the type of the elements
template <typename F> void by_type(int32_t type, F f) {
    if (type == VQ_F32)
        f(vq::F32());
    else if (type == VQ_F16)
        f(vq::F16());
    else
        f(vq::BF16());
}

// One launch of tiles; the limit of the LDS above 64 KB is asked for once per context and instance.
template <typename T, int TR, int TC, int WR, int WC, int KS, int STAGES> int32_t score_tiles(vq_ctx *ctx, const vq::ScoresArgs &a, int bit) {
    static_assert(WR * WC * 32 * (TC / WC * (int)sizeof(typename T::Raw) + 16) <= STAGES * KS * (TR + TC) * 128, "blocks on their way out fit into the steps' LDS");
    const int lds = vq::tile_lds_bytes(TR, TC, WR * WC, WC, KS, STAGES, a.dim, (int)sizeof(typename T::Raw));
    const auto kernel = vq::k_scores_tile<T, TR, TC, WR, WC, KS, STAGES>;
    if (lds + TC * 8 > 65536 && !(ctx->scores_lds_set >> bit & 1)) {
        VQ_HIP(ctx, hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize,
                                        STAGES * KS * (TR + TC) * 128 + TC * 8));
        ctx->scores_lds_set |= 1u << bit;
    }
    const uint32_t rt = (uint32_t)cdiv64(a.n, TR), ct = (uint32_t)cdiv64(a.k, TC);
    hipLaunchKernelGGL(kernel, dim3(rt * ct), dim3(64 * WR * WC), lds + TC * 8, ctx->stream, a, rt, ct, lds);
    VQ_HIP(ctx, hipGetLastError());
    return VQ_OK;
}

// aligned: addresses and strides are multiples of 16, and the strides at most kMaxTileStride.
template <typename T> int32_t scores_slice(vq_ctx *ctx, const vq::ScoresArgs &a, int type, bool aligned) {
    if (!aligned) {
        hipLaunchKernelGGL(vq::k_scores_any<T>, dim3(cdiv(a.k, 64), cdiv(a.n, 64)), dim3(256), 0, ctx->stream, a);
        VQ_HIP(ctx, hipGetLastError());
        return VQ_OK;
    }
    const vq::ScoreWay way = vq::score_way(a.n, a.k, a.dim);
    const int bit = type * 8 + way;
    constexpr int WC = sizeof(typename T::Raw) == 4 ? 4 : 2;  // waves side by side: a wave's codes of a row are 128 bytes of results
    switch (way) {
    case vq::FEW:
        hipLaunchKernelGGL((vq::k_scores_few<T, 1, 1, 4>), dim3(cdiv(a.k, 16), cdiv(a.n, 16)), dim3(256), 0, ctx->stream, a);
        VQ_HIP(ctx, hipGetLastError());
        return VQ_OK;
    case vq::T64: return score_tiles<T, 64, 64, 2, 2, 2, 4>(ctx, a, bit);
    case vq::T64_MANY: return score_tiles<T, 64, 64, 2, 2, 1, 2>(ctx, a, bit);
    case vq::T64_128: return score_tiles<T, 64, 128, 2, WC, 1, 3>(ctx, a, bit);
    case vq::T128: return score_tiles<T, 128, 128, 8 / WC, WC, 1, 4>(ctx, a, bit);
    case vq::T256: return score_tiles<T, 256, 256, 2, 4, 1, 2>(ctx, a, bit);
    default: return score_tiles<T, 128, 128, 8 / WC, WC, 1, 2>(ctx, a, bit);
    }
}

// n 8-bit rows to aligned ones.
int32_t pack_i8(vq_ctx *ctx, const int8_t *x, int64_t n, int64_t ld, int32_t dim, int8_t *to) {
    const int64_t pieces = n * (vq::packed_stride(dim) / 16);
    hipLaunchKernelGGL(vq::k_pack_i8, dim3((unsigned)cdiv64(pieces, 256)), dim3(256), 0, ctx->stream, x, n, ld, dim, to);
    VQ_HIP(ctx, hipGetLastError());
    return VQ_OK;
}

template <typename T, bool TINY, int G, int E> void short_rows(vq_ctx *ctx, const vq::LogprobArgs &a) {
    hipLaunchKernelGGL((vq::k_logprobs_short<T, G, E, TINY>), dim3((unsigned)cdiv64(a.n, 256 / G)), dim3(256), 0, ctx->stream, a);
}
template <typename T> void row_parts(vq_ctx *ctx, const vq::PartArgs &p, int per_lane) {
    constexpr int VEC = 16 / (int)sizeof(typename T::Raw);
    const dim3 grid((unsigned)(p.a.n * p.parts)), wg(256);
    if (per_lane == 32)
        hipLaunchKernelGGL((vq::k_logprobs_part<T, 32 / VEC>), grid, wg, 0, ctx->stream, p);
    else
        hipLaunchKernelGGL((vq::k_logprobs_part<T, 64 / VEC>), grid, wg, 0, ctx->stream, p);
}

int32_t logprobs_slice(vq_ctx *ctx, int32_t type, const vq::LogprobArgs &a, const vq::RowPlan &plan) {
    if (plan.lanes < 256) {
        by_type(type, [&](auto t) {
            typedef decltype(t) T;
            if (a.k < 16 / (int)sizeof(typename T::Raw))
                short_rows<T, true, 1, 16>(ctx, a);
            else if (plan.lanes == 1)
                short_rows<T, false, 1, 16>(ctx, a);
            else if (plan.lanes == 4)
                short_rows<T, false, 4, 16>(ctx, a);
            else if (plan.lanes == 8)
                short_rows<T, false, 8, 32>(ctx, a);
            else if (plan.per_lane == 8)
                hipLaunchKernelGGL((vq::k_logprobs_wave<T, 8>), dim3((unsigned)cdiv64(a.n, 4)), dim3(256), 0, ctx->stream, a);
            else if (plan.per_lane == 16)
                hipLaunchKernelGGL((vq::k_logprobs_wave<T, 16>), dim3((unsigned)cdiv64(a.n, 4)), dim3(256), 0, ctx->stream, a);
            else if (plan.per_lane == 32)
                hipLaunchKernelGGL((vq::k_logprobs_wave<T, 32>), dim3((unsigned)cdiv64(a.n, 4)), dim3(256), 0, ctx->stream, a);
            else
                hipLaunchKernelGGL((vq::k_logprobs_wave<T, 64>), dim3((unsigned)cdiv64(a.n, 4)), dim3(256), 0, ctx->stream, a);
        });
        VQ_HIP(ctx, hipGetLastError());
        return VQ_OK;
    }
    vq::PartArgs p{a, (int)plan.parts, plan.codes, nullptr, nullptr};
    if (plan.parts > 1) {
        p.keys = (uint64_t *)ctx->score_parts.p;  // (the call has provided it)
        p.sums = (float *)(p.keys + (size_t)a.n * plan.parts * a.top);
    }
    by_type(type, [&](auto t) {
        row_parts<decltype(t)>(ctx, p, plan.per_lane);
        if (plan.parts > 1) {
            const int rows = plan.parts <= 8 ? 4 : 1;  // per workgroup: at most 32.5 KB of lists
            hipLaunchKernelGGL(vq::k_logprobs_join<decltype(t)>, dim3((unsigned)cdiv64(a.n, rows)), dim3(64 * rows),
                               rows * 8 * (2 * plan.parts * a.top + 8), ctx->stream, p);
        }
    });
    VQ_HIP(ctx, hipGetLastError());
    return VQ_OK;
}

}  // namespace

extern "C" {

int32_t vq_rows_i8(vq_ctx *ctx, int32_t type, const void *d_x, int64_t n, int64_t ld, int32_t dim, int8_t *d_q,
                   int64_t ld_q, float *d_scale) {
    if (!ctx) return VQ_ERR_INVALID_ARG;
    bool go;
    VQ_TRY(admit(ctx, vq::check_rows_i8(type, d_x, n, ld, dim, d_q, ld_q, d_scale), n, &go));
    if (!go) return VQ_OK;
    const int e = vq::type_bytes(type);
    const vq::LanePlan plan = vq::plan_lanes(dim, e);
    const int64_t slice = (int64_t)1 << 23;  // rows per launch: a grid has fewer than 2^32 lanes
    for (int64_t r = 0; r < n; r += slice) {
        const vq::RowsI8Args a{(const char *)d_x + r * ld * e, std::min(slice, n - r), ld, dim, d_q + r * ld_q, ld_q, d_scale + r};
        const auto grid = [&](int lanes) { return dim3((unsigned)cdiv64(a.n, 256 / lanes)); };
        by_type(type, [&](auto t) {
            typedef decltype(t) T;
            if (plan.lanes == 4 && plan.vectors == 1)
                hipLaunchKernelGGL((vq::k_rows_i8<T, 4, 1>), grid(4), dim3(256), 0, ctx->stream, a);
            else if (plan.lanes == 4)
                hipLaunchKernelGGL((vq::k_rows_i8<T, 4, 4>), grid(4), dim3(256), 0, ctx->stream, a);
            else if (plan.lanes == 8)
                hipLaunchKernelGGL((vq::k_rows_i8<T, 8, 4>), grid(8), dim3(256), 0, ctx->stream, a);
            else if (plan.lanes == 64 && plan.vectors == 1)
                hipLaunchKernelGGL((vq::k_rows_i8<T, 64, 1>), grid(64), dim3(256), 0, ctx->stream, a);
            else if (plan.lanes == 64)
                hipLaunchKernelGGL((vq::k_rows_i8<T, 64, 4>), grid(64), dim3(256), 0, ctx->stream, a);
            else if (plan.lanes == 256)
                hipLaunchKernelGGL((vq::k_rows_i8<T, 256, 8>), grid(256), dim3(256), 0, ctx->stream, a);
            else
                hipLaunchKernelGGL(vq::k_rows_i8_any<T>, dim3((unsigned)std::min<int64_t>(a.n, 1 << 20)), dim3(256), 0, ctx->stream, a);
        });
        VQ_HIP(ctx, hipGetLastError());
    }
    return VQ_OK;
}

int32_t vq_scores_i8(vq_ctx *ctx, const int8_t *d_x, const float *d_xs, int64_t n, int64_t ld_x, const int8_t *d_w,
                     const float *d_ws, int32_t k, int64_t ld_w, int32_t dim, const float *d_bias, int32_t out_type,
                     void *d_out, int64_t ld_out) {
    if (!ctx) return VQ_ERR_INVALID_ARG;
    bool go;
    VQ_TRY(admit(ctx, vq::check_scores_i8(d_x, d_xs, n, ld_x, d_w, d_ws, k, ld_w, dim, d_bias, out_type, d_out, ld_out), n, &go));
    if (!go) return VQ_OK;
    const auto fit = [](const void *p, int64_t ld) { return !vq::misaligned(p, 16) && ld % 16 == 0 && ld <= vq::kMaxTileStride; };
    bool ready_x = fit(d_x, ld_x), ready_w = fit(d_w, ld_w);
    vq::ScoresArgs a{d_x, d_xs, n, ld_x, d_w, d_ws, k, ld_w, dim, d_bias, d_out, ld_out};
    int64_t slice = vq::score_rows_of_a_launch(k);
    int8_t *packed_x = nullptr;
    if (!(ready_x && ready_w) && vq::score_pack(n, k, dim)) {
        const int64_t ld = vq::packed_stride(dim);
        if (!ready_x) slice = std::min(slice, std::max<int64_t>(64, vq::kPackRows / ld / 64 * 64));
        const int64_t rows = ready_x ? 0 : std::min(n, slice);
        VQ_TRY(ensure_kept(ctx, ctx->score_packed, (size_t)((rows + (ready_w ? 0 : k)) * ld)));
        int8_t *to = (int8_t *)ctx->score_packed.p;
        if (!ready_w) {
            VQ_TRY(pack_i8(ctx, d_w, k, ld_w, dim, to));
            a.w = to, a.ld_w = ld, ready_w = true;
        }
        if (!ready_x) packed_x = to + (a.w == to ? k * ld : 0), a.ld_x = ld, ready_x = true;
    }
    for (int64_t r = 0; r < n; r += slice) {
        a.n = std::min(n - r, slice);
        a.x = d_x + r * ld_x;
        a.xs = d_xs + r;
        a.out = (char *)d_out + r * ld_out * vq::type_bytes(out_type);
        if (packed_x) {
            VQ_TRY(pack_i8(ctx, a.x, a.n, ld_x, dim, packed_x));
            a.x = packed_x;
        }
        int32_t rc = VQ_OK;
        by_type(out_type, [&](auto t) { rc = scores_slice<decltype(t)>(ctx, a, out_type, ready_x && ready_w); });
        VQ_TRY(rc);
    }
    return VQ_OK;
}

int32_t vq_code_logprobs(vq_ctx *ctx, int32_t type, const void *d_scores, int64_t n, int64_t ld, int32_t k, float beta,
                         int32_t code_bytes, const void *d_codes, int64_t code_stride, int32_t top, float *d_logprob,
                         float *d_max, float *d_logsum, float *d_entropy, float *d_top_logprob, int32_t *d_top_code) {
    if (!ctx) return VQ_ERR_INVALID_ARG;
    bool go;
    VQ_TRY(admit(ctx, vq::check_code_logprobs(type, d_scores, n, ld, k, beta, code_bytes, d_codes, code_stride, top, d_logprob,
                                              d_max, d_logsum, d_entropy, d_top_logprob, d_top_code), n, &go));
    if (!go) return VQ_OK;
    const vq::RowPlan plan = vq::plan_rows(n, k, top, vq::type_bytes(type));
    const int64_t slice = vq::logprob_rows_of_a_launch(plan, top);
    if (plan.parts > 1) VQ_TRY(ensure_kept(ctx, ctx->score_parts, (size_t)vq::part_workspace(n, k, top)));
    const int e = vq::type_bytes(type);
    for (int64_t r = 0; r < n; r += slice) {
        vq::LogprobArgs a{(const char *)d_scores + r * ld * e, std::min(slice, n - r), ld, k, beta,
                          d_codes ? (const char *)d_codes + r * code_stride * code_bytes : nullptr, code_stride, code_bytes, top,
                          d_logprob ? d_logprob + r : nullptr, d_max ? d_max + r : nullptr, d_logsum ? d_logsum + r : nullptr,
                          d_entropy ? d_entropy + r : nullptr, top ? d_top_logprob + r * top : nullptr, top ? d_top_code + r * top : nullptr};
        VQ_TRY(logprobs_slice(ctx, type, a, plan));
    }
    return VQ_OK;
}

int32_t vq_code_logprobs_grad(vq_ctx *ctx, int32_t type, const void *d_scores, int64_t n, int64_t ld, int32_t k, float beta,
                              int32_t code_bytes, const void *d_codes, int64_t code_stride, const float *d_max,
                              const float *d_logsum, const float *d_entropy, const float *d_g_logprob,
                              const float *d_g_entropy, void *d_grad, int64_t ld_grad) {
    if (!ctx) return VQ_ERR_INVALID_ARG;
    bool go;
    VQ_TRY(admit(ctx, vq::check_code_logprobs_grad(type, d_scores, n, ld, k, beta, code_bytes, d_codes, code_stride, d_max,
                                                   d_logsum, d_entropy, d_g_logprob, d_g_entropy, d_grad, ld_grad), n, &go));
    if (!go) return VQ_OK;
    const int e = vq::type_bytes(type), vec = 16 / e;
    const int64_t slice = (int64_t)1 << 23;  // rows per launch: a grid has fewer than 2^32 lanes
    for (int64_t r = 0; r < n; r += slice) {
        const auto at = [&](const float *p) { return p ? p + r : nullptr; };
        const vq::GradArgs a{(const char *)d_scores + r * ld * e, std::min(slice, n - r), ld, k, beta,
                             d_codes ? (const char *)d_codes + r * code_stride * code_bytes : nullptr, code_stride, code_bytes,
                             at(d_max), at(d_logsum), at(d_entropy), at(d_g_logprob), at(d_g_entropy), (char *)d_grad + r * ld_grad * e, ld_grad};
        by_type(type, [&](auto t) {
            typedef decltype(t) T;
            if (k < vec)
                hipLaunchKernelGGL(vq::k_logprobs_grad_tiny<T>, dim3((unsigned)cdiv64(a.n, 256)), dim3(256), 0, ctx->stream, a);
            else if (k <= 16 * vec)
                hipLaunchKernelGGL((vq::k_logprobs_grad<T, 4, 4>), dim3((unsigned)cdiv64(a.n, 64)), dim3(256), 0, ctx->stream, a);
            else if (k <= 64 * vec)
                hipLaunchKernelGGL((vq::k_logprobs_grad<T, 16, 4>), dim3((unsigned)cdiv64(a.n, 16)), dim3(256), 0, ctx->stream, a);
            else if (k <= 256 * vec)
                hipLaunchKernelGGL((vq::k_logprobs_grad<T, 64, 4>), dim3((unsigned)cdiv64(a.n, 4)), dim3(256), 0, ctx->stream, a);
            else
                hipLaunchKernelGGL((vq::k_logprobs_grad<T, 256, 4>), dim3((unsigned)a.n, (unsigned)cdiv64(k, 1024 * vec)), dim3(256), 0, ctx->stream, a);
        });
        VQ_HIP(ctx, hipGetLastError());
    }
    return VQ_OK;
}

}  // extern "C"
