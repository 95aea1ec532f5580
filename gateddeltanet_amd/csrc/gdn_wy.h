// gdn_wy.h -- FP32 products on the BF16 matrix cores, shared by the chunked
// prefill (gdn_batch.hip) and the delta-rule operators (gdn_delta.hip) of
// libgdn_amd.so.  Not part of the ABI.
//
// An FP32 operand enters as three BF16 terms whose sum it is (8 + 8 + 8
// significand bits).  v_mfma_f32_16x16x32_bf16 forms exact products and FP32
// sums at 16 times the rate of v_mfma_f32_16x16x4_f32, so three products (one
// operand is BF16) or six (both are split) still take a fifth (three eighths)
// of its time.
#ifndef GDN_WY_H
#define GDN_WY_H

#include "gdn_device.h"

namespace gdn {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ f32x4 mfma_bf16(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c,
                                                   0, 0, 0);
}

// x as three BF16 terms: p[0] + p[1] + p[2] = x (each rounded to nearest, the
// differences exact), four values packed in two words.  The first term is
// held to the largest finite BF16 value, so every finite x of 2^-110 and more
// is its terms' sum (rounded up to an infinity, that term would leave
// infinity - infinity behind); below, the last terms are BF16 subnormals.  An
// infinite or NaN x has a NaN term.
__device__ __forceinline__ void split3(const f32x4 x, u32x2 (&p)[3]) {
    constexpr float kMax = 0x1.fep127f;
    auto held = [](float v) { return __builtin_amdgcn_fmed3f(v, -kMax, kMax); };
    f32x4 r = x;
#pragma unroll
    for (int i = 0; i < 3; ++i) {
        p[i].x = i == 0 ? cvt_pk(held(r.x), held(r.y)) : cvt_pk(r.x, r.y);
        p[i].y = i == 0 ? cvt_pk(held(r.z), held(r.w)) : cvt_pk(r.z, r.w);
        if (i < 2) {
            r.x = r.x - u2f(p[i].x << 16);
            r.y = r.y - u2f(p[i].x & 0xffff0000u);
            r.z = r.z - u2f(p[i].y << 16);
            r.w = r.w - u2f(p[i].y & 0xffff0000u);
        }
    }
}

// The product of two split operands over one 32-wide k step, smallest terms
// first (the three terms below 2^-24 of the product are left out).
__device__ __forceinline__ f32x4 mfma_split(const u32x4 (&a)[3], const u32x4 (&b)[3], f32x4 c) {
    c = mfma_bf16(a[2], b[0], c);
    c = mfma_bf16(a[0], b[2], c);
    c = mfma_bf16(a[1], b[1], c);
    c = mfma_bf16(a[1], b[0], c);
    c = mfma_bf16(a[0], b[1], c);
    return mfma_bf16(a[0], b[0], c);
}

}  // namespace gdn
#endif
