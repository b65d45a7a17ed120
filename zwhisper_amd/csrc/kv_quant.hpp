// The 8-bit key/value caches (include/zw_gpu.h, zwg_kvq_*): their layout in HBM, shared by the kernels that write
// them (kv_quant.hip) and the attention that reads them (attn_kvq.hip).
//
// A unit is one (layer, sequence, KV head), u = (layer * n_seq + seq) * n_head_kv + head, of n_pad tokens (n_ctx
// rounded up to 64).  Per unit:
//   keys    n_pad * d bytes, values the same, in the order of kvq_at: a wave's 64 lanes read 1 KB on end, 16 bytes a lane,
//           and each half of these is an operand of a matrix instruction as it is; the values' order is the one in which
//           the attention's probabilities lie in the lanes' registers after the score products, so that they
//           feed the value products with no exchange between lanes
//   scales  [n_pad / block] f32 each for keys and values
//   the open block: its rows in f32 [block][d], keys and values, the block's index and filled rows, and
//           each row's largest magnitude
// Int8 codes are stored as code + 128, which turns into f16 by placing the byte under a constant exponent.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <memory>

#include "kvq_plan.hpp"
#include "rope.hpp"
#include "zw_gpu.h"

namespace zwg {

struct KvqView {
    uint8_t *codes[2]; // keys, values; unit u at + u * unit_bytes
    float *scales[2];  // unit u at + u * n_blocks
    float *rows[2];    // unit u's open block at + u * block * d
    KvqOpen *open;     // [unit][2]
    int64_t unit_bytes;
    int32_t n_blocks, block, n_ctx;
    int32_t d, n_head_kv, n_seq;
};

#ifdef __HIPCC__
// amax as its bit pattern -> the block's scale and what an element is multiplied by before rounding.
// Infinities and NaNs (patterns from 0x7f800000) give a NaN scale over zero codes; below 2^-100 zeros.
template <int FMT> __device__ __forceinline__ void kvq_scale(uint32_t top, float *scale, float *mul) {
    constexpr float Q = FMT == ZWG_KVQ_I8 ? 127.0f : 448.0f;
    const float amax = __builtin_bit_cast(float, top);
    const bool bad = top >= 0x7f800000u, none = top < ((127u - 100u) << 23);
    *scale = bad ? __builtin_nanf("") : none ? 0.0f : __fdiv_rn(amax, Q);
    *mul = bad || none ? 0.0f : __fdiv_rn(Q, amax);
}

// Four codes in one word.  The products are at most Q (1 + 2^-23) in magnitude, which rounds to Q.  With a zero
// multiplier every code is zero, whatever the element (an infinity times zero is no number).
template <int FMT> __device__ __forceinline__ uint32_t kvq_encode4(float a, float b, float c, float e, float mul) {
#pragma clang fp contract(off) // the product is rounded before the code is
    if (mul == 0.0f) return FMT == ZWG_KVQ_I8 ? 0x80808080u : 0u;
    a *= mul;
    b *= mul;
    c *= mul;
    e *= mul;
    if (FMT == ZWG_KVQ_I8) {
        // 3 * 2^22 + 128 + x: the sum is rounded to a whole number, ties to even, and its low byte is code + 128
        constexpr float kWhole = 12582912.0f + 128.0f;
        const uint32_t ua = __builtin_bit_cast(uint32_t, a + kWhole), ub = __builtin_bit_cast(uint32_t, b + kWhole);
        const uint32_t uc = __builtin_bit_cast(uint32_t, c + kWhole), ue = __builtin_bit_cast(uint32_t, e + kWhole);
        return __builtin_amdgcn_perm(__builtin_amdgcn_perm(ue, uc, 0x0c0c0400u), __builtin_amdgcn_perm(ub, ua, 0x0c0c0400u), 0x05040100u);
    }
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(c, e, w, true);
    return (uint32_t)w;
}

// The value of byte `i` of a word of codes, before the scale.
template <int FMT, int I> __device__ __forceinline__ float kvq_decode(uint32_t w) {
    if (FMT == ZWG_KVQ_I8) return (float)(int)((w >> (8 * I)) & 255u) - 128.0f;
    return __builtin_amdgcn_cvt_f32_fp8((int)w, I);
}
template <int FMT> __device__ __forceinline__ float kvq_decode_byte(uint8_t b) { return kvq_decode<FMT, 0>(b); }
#endif

} // namespace zwg

struct zwg_kvq {
    zwg_ctx *ctx = nullptr;
    zwg_kvq_desc desc{};
    bool has_rope = false;
    zwg_rope_desc rope{};
    std::shared_ptr<ZwgRopeTables> tables;
    void *mem = nullptr; // one allocation: codes, scales, open blocks
    zwg::KvqView view{};
    uint64_t n_pad = 0;
};
