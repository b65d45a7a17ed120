// Rotary positions (include/zw_gpu.h, zwg_rope_*): the tables and the rotation of one piece of a head, shared
// by the operator (rope.hip) and the 8-bit caches' append (kv_quant.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <memory>

#include "zw_gpu.h"

// The tables of one zwg_rope in device memory; shared with the caches made with it, and freed by the last
// of their owners (each synchronises its context's stream before it lets go).
struct ZwgRopeTables {
    int device = 0;
    float *cos = nullptr; // [n_ctx][n_rot / 2]
    float *sin = nullptr;
    ~ZwgRopeTables() {
        (void)hipSetDevice(device);
        if (cos) (void)hipFree(cos);
        if (sin) (void)hipFree(sin);
    }
};

struct zwg_rope {
    zwg_ctx *ctx = nullptr;
    zwg_rope_desc desc{};
    std::shared_ptr<ZwgRopeTables> tables;
};

namespace zwg {

// How a head is cut into pieces that one thread rotates: in pieces of 4 pairs as 16-byte accesses
// (half layout, n_rot / 2 a multiple of 4), of 4 dims (interleaved, n_rot a multiple of 4), or pair by pair.
constexpr int kRopeHalf4 = 0, kRopeInter4 = 1, kRopePairs = 2;

struct RopeView {
    const float *cos, *sin; // nullptr: no rotation
    int32_t n_ctx, half, d; // half = n_rot / 2
    int32_t layout, mode;
    float sign;             // -1: the transposed rotation
};

inline RopeView rope_view(const zwg_rope_desc &d, const ZwgRopeTables &t, bool backward) {
    RopeView v{};
    v.cos = t.cos;
    v.sin = t.sin;
    v.n_ctx = (int32_t)d.n_ctx;
    v.half = (int32_t)(d.n_rot / 2);
    v.d = (int32_t)d.d;
    v.layout = (int32_t)d.layout;
    v.mode = d.layout == ZWG_ROPE_HALF ? (d.n_rot % 8 == 0 ? kRopeHalf4 : kRopePairs)
                                       : (d.n_rot % 4 == 0 ? kRopeInter4 : kRopePairs);
    v.sign = backward ? -1.0f : 1.0f;
    return v;
}

// Pieces of a head that hold rotated dims, and pieces in all (those behind are copied).
__host__ __device__ inline int rope_turned(const RopeView &v) {
    return v.mode == kRopeHalf4 ? v.half / 4 : v.mode == kRopeInter4 ? v.half / 2 : v.half;
}
__host__ __device__ inline int rope_pieces(const RopeView &v) {
    const int tail = v.d - 2 * v.half;
    return rope_turned(v) + (v.mode == kRopePairs ? tail : tail / 4);
}

#ifdef __HIPCC__
// Rotates piece `c` of the head at x (position `pos`) into the head at y, which may be x.  Each product and
// sum is rounded by itself, as the reference rounds them.
__device__ __forceinline__ void rope_piece(const RopeView &v, int64_t pos, int c, const float *x, float *y) {
#pragma clang fp contract(off)
    const int turned = rope_turned(v);
    const float *cs = v.cos + pos * v.half, *sn = v.sin + pos * v.half;
    if (v.mode == kRopeHalf4) {
        if (c < turned) {
            const int j = 4 * c;
            // two rows of a table are half floats apart, and half % 4 == 0: 16-byte loads
            const float4 co = *reinterpret_cast<const float4 *>(cs + j);
            float4 si = *reinterpret_cast<const float4 *>(sn + j);
            si = make_float4(si.x * v.sign, si.y * v.sign, si.z * v.sign, si.w * v.sign);
            const float4 a = *reinterpret_cast<const float4 *>(x + j);
            const float4 b = *reinterpret_cast<const float4 *>(x + j + v.half);
            *reinterpret_cast<float4 *>(y + j) = make_float4(a.x * co.x - b.x * si.x, a.y * co.y - b.y * si.y,
                                                             a.z * co.z - b.z * si.z, a.w * co.w - b.w * si.w);
            *reinterpret_cast<float4 *>(y + j + v.half) = make_float4(a.x * si.x + b.x * co.x, a.y * si.y + b.y * co.y,
                                                                      a.z * si.z + b.z * co.z, a.w * si.w + b.w * co.w);
            return;
        }
    } else if (v.mode == kRopeInter4) {
        if (c < turned) {
            const float2 co = *reinterpret_cast<const float2 *>(cs + 2 * c);
            const float2 s0 = *reinterpret_cast<const float2 *>(sn + 2 * c);
            const float2 si = make_float2(s0.x * v.sign, s0.y * v.sign);
            const float4 a = *reinterpret_cast<const float4 *>(x + 4 * c);
            *reinterpret_cast<float4 *>(y + 4 * c) = make_float4(a.x * co.x - a.y * si.x, a.x * si.x + a.y * co.x,
                                                                 a.z * co.y - a.w * si.y, a.z * si.y + a.w * co.y);
            return;
        }
    } else {
        if (c < turned) {
            const int i0 = v.layout == ZWG_ROPE_HALF ? c : 2 * c, i1 = v.layout == ZWG_ROPE_HALF ? c + v.half : 2 * c + 1;
            const float co = cs[c], si = sn[c] * v.sign, a = x[i0], b = x[i1];
            y[i0] = a * co - b * si;
            y[i1] = a * si + b * co;
        } else {
            y[v.half + c] = x[v.half + c]; // dim 2 half + (c - half)
        }
        return;
    }
    const int i = 2 * v.half + 4 * (c - turned);
    *reinterpret_cast<float4 *>(y + i) = *reinterpret_cast<const float4 *>(x + i);
}
#endif

} // namespace zwg
