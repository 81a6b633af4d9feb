// What the C entry points of scores and of models over codes share.
#pragma once
#include <algorithm>

#include "ctx.hpp"
#include "logprobs.hpp"
#include "score_rules.hpp"

namespace vqh {

inline int64_t cdiv64(int64_t a, int64_t b) { return (a + b - 1) / b; }

// A workspace that captured graphs may hold the address of: it grows by a new allocation, at least twice the last, and the
// ones before stay.  While the stream is being captured it cannot grow, and the capture goes on.
inline int32_t ensure_kept(vq_ctx *ctx, DevBuf &b, size_t bytes) {
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
inline int32_t admit(vq_ctx *ctx, const vq::Refusal &r, int64_t n, bool *go) {
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

}  // namespace vqh
