// Rotary positions as an operator (include/zw_gpu.h, zwg_rope_*).
//
// The tables hold f32(m cos(p w_j)) and f32(m sin(p w_j)), formed in f64 on the device (2^17 positions of 64 pairs
// are 8.4 million sines and cosines, too many for the host at every load); the frequencies come from the host.
// The rotation reads each row once and writes it once: memory-bound (8192 tokens of 14 heads of 128: 122 MB in 20 us,
// 6.1 TB/s with what the caches still hold), and for few tokens bound by the launch (one token: 2.9 us).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <string>
#include <vector>

#include "kvq_plan.hpp"
#include "rope.hpp"
#include "zw_ctx.hpp"

using namespace zwg_host;

namespace {

constexpr int kRopeThreads = 256;

__global__ __launch_bounds__(256) void rope_table_kernel(const double *w, int half, int64_t n, double m, float *cos_t,
                                                         float *sin_t) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        const int64_t p = i / half;
        const double a = (double)p * w[i - p * half];
        cos_t[i] = (float)(m * cos(a));
        sin_t[i] = (float)(m * sin(a));
    }
}

struct RopeArgs {
    zwg::RopeView view;
    const float *x;
    float *out;
    int64_t x_stride, out_stride;
    const int32_t *pos_dev;
    int64_t pos0;
    int32_t n, n_head;
    int32_t pieces; // pieces of a head to go over: all, or in place the rotated ones alone
    int32_t tokens; // tokens per workgroup
};

// A workgroup takes `tokens` tokens and all their heads' pieces, neighbouring threads neighbouring pieces.
__global__ __launch_bounds__(kRopeThreads) void rope_kernel(RopeArgs a) {
    const int t0 = blockIdx.x * a.tokens;
    const int per = a.n_head * a.pieces;
    const int all = min(a.tokens, a.n - t0) * per;
    for (int i = threadIdx.x; i < all; i += kRopeThreads) {
        const int t = i / per, r = i - t * per;
        const int h = r / a.pieces, c = r - h * a.pieces;
        const int64_t tok = t0 + t;
        const int64_t pos = a.pos_dev ? (int64_t)a.pos_dev[tok] : a.pos0 + tok;
        if (pos < 0 || pos >= a.view.n_ctx) continue;
        const int64_t col = (int64_t)h * a.view.d;
        zwg::rope_piece(a.view, pos, c, a.x + tok * a.x_stride + col, a.out + tok * a.out_stride + col);
    }
}

const char *const kRopeClosed = "the rope's context is closed";

void release(zwg_rope *r) {
    if (r->ctx) {
        (void)hipSetDevice(r->ctx->device);
        (void)hipStreamSynchronize(r->ctx->stream);
    }
    r->tables.reset();
}

void detach_rope(void *obj) {
    auto *r = static_cast<zwg_rope *>(obj);
    release(r);
    r->ctx = nullptr;
}

int create(zwg_ctx *ctx, const zwg_rope_desc *desc, zwg_rope **out) {
    const std::string msg = zwg_planner::check_rope_desc(*desc);
    if (!msg.empty()) return fail(ctx, msg);
    hipError_t e = hipSetDevice(ctx->device);
    if (e != hipSuccess) return fail_hip(ctx, "hipSetDevice", e);
    const std::vector<double> w = zwg_planner::rope_frequencies(*desc);
    auto tables = std::make_shared<ZwgRopeTables>();
    tables->device = ctx->device;
    const int64_t n = (int64_t)(desc->n_ctx * w.size());
    void *wd = nullptr, *c = nullptr, *s = nullptr;
    e = hipMalloc(&wd, w.size() * sizeof(double));
    if (e == hipSuccess) e = hipMalloc(&c, (uint64_t)n * sizeof(float));
    tables->cos = static_cast<float *>(c);
    if (e == hipSuccess) e = hipMalloc(&s, (uint64_t)n * sizeof(float));
    tables->sin = static_cast<float *>(s);
    if (e == hipSuccess) e = hipMemcpyAsync(wd, w.data(), w.size() * sizeof(double), hipMemcpyHostToDevice, ctx->stream);
    if (e == hipSuccess) {
        const double m = zwg_planner::rope_mscale(*desc);
        rope_table_kernel<<<(unsigned)std::min<int64_t>((n + 255) / 256, 4096), 256, 0, ctx->stream>>>(
            static_cast<const double *>(wd), (int)w.size(), n, m, tables->cos, tables->sin);
        e = hipGetLastError();
    }
    const hipError_t es = hipStreamSynchronize(ctx->stream);
    if (wd) (void)hipFree(wd);
    if (e == hipSuccess) e = es;
    if (e != hipSuccess) return fail_hip(ctx, "rope tables", e);
    auto *r = new zwg_rope();
    r->ctx = ctx;
    r->desc = *desc;
    r->tables = std::move(tables);
    add_child(ctx, r, detach_rope);
    *out = r;
    return ZWG_OK;
}

int apply(zwg_rope *rope, const float *x, uint64_t n, uint64_t n_head, uint64_t x_stride, const int32_t *pos_dev,
          uint64_t pos0, float *out, uint64_t out_stride, uint32_t flags) {
    zwg_ctx *ctx = rope->ctx;
    const zwg_rope_desc &d = rope->desc;
    const std::string msg = zwg_planner::check_rope_apply(d, x, n, n_head, x_stride, pos_dev, pos0, out, out_stride, flags);
    if (!msg.empty()) return fail(ctx, msg);
    if (n == 0) return ZWG_OK;
    const bool in_place = x == out;
    hipError_t e = hipSetDevice(ctx->device);
    if (e != hipSuccess) return fail_hip(ctx, "hipSetDevice", e);
    RopeArgs a{};
    a.view = zwg::rope_view(d, *rope->tables, flags & ZWG_ROPE_INVERSE);
    a.x = x;
    a.out = out;
    a.x_stride = (int64_t)x_stride;
    a.out_stride = (int64_t)out_stride;
    a.pos_dev = pos_dev;
    a.pos0 = (int64_t)pos0;
    a.n = (int32_t)n;
    a.n_head = (int32_t)n_head;
    a.pieces = in_place ? zwg::rope_turned(a.view) : zwg::rope_pieces(a.view);
    const uint64_t per = n_head * (uint64_t)a.pieces; // at most 65535 * 1024
    a.tokens = (int32_t)std::max<uint64_t>(1, std::min<uint64_t>(n, 4 * kRopeThreads / per));
    const uint64_t blocks = (n + a.tokens - 1) / a.tokens;
    if (blocks * kRopeThreads > 0xffffffffull) return fail(ctx, "too many rows in one call"); // a launch's threads
    rope_kernel<<<(unsigned)blocks, kRopeThreads, 0, ctx->stream>>>(a);
    e = hipGetLastError();
    return e == hipSuccess ? ZWG_OK : fail_hip(ctx, "rope launch", e);
}

} // namespace

extern "C" {

int zwg_rope_create(zwg_ctx *ctx, const zwg_rope_desc *desc, zwg_rope **out) {
    if (!out) return fail(ctx, "null output pointer");
    *out = nullptr;
    if (!ctx || !desc) return fail(ctx, "null context or rope desc");
    return guarded(ctx, [&] { return create(ctx, desc, out); });
}

void zwg_rope_destroy(zwg_rope *rope) {
    if (!rope) return;
    if (rope->ctx) remove_child(rope->ctx, rope);
    release(rope);
    delete rope;
}

int zwg_rope_apply_dev(zwg_rope *rope, const float *x, uint64_t n, uint64_t n_head, uint64_t x_stride,
                       const int32_t *pos_dev, uint64_t pos0, float *out, uint64_t out_stride, uint32_t flags) {
    if (!rope) return fail(nullptr, "null rope");
    if (!rope->ctx) return fail(nullptr, kRopeClosed);
    return guarded(rope->ctx, [&] { return apply(rope, x, n, n_head, x_stride, pos_dev, pos0, out, out_stride, flags); });
}

} // extern "C"
