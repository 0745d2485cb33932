// What the kernels of the paged attention share: their arguments, the scaling of q, the store of a result.
#pragma once

#include "paged_cache.cuh"

namespace b200 {
namespace paged {

struct AttendParams {
    uint16_t *out;
    const uint16_t *q;
    int64_t o_st, o_sh, q_st, q_sh;// strides of token and head
    const uint8_t *kp, *vp;
    const float *ks, *vs;
    const int32_t *table, *lens, *offs;
    int32_t rows, group;
    float scale_log2;// scale * log2(e)
    bool bf16, vec, q_vec, o_vec;
    FastDiv page_div;// by the page size
    CacheShape c;
    TableShape t;
};

// Power of two that brings the largest magnitude of a row of q (16-bit pattern without sign) to [2^14, 2^15) in fp16;
// 0 for rows of zeros and rows that hold infinities or NaN.
__device__ __forceinline__ int32_t query_shift(bool bf16, uint32_t top) {
    if (top == 0 || top >= (bf16 ? 0x7F80u : 0x7C00u)) return 0;
    const float f = bf16 ? __uint_as_float(top << 16) : f16_to_f32((uint16_t) top);
    const int32_t e = (int32_t) (__float_as_uint(f) >> 23) - 127;// (bf16 subnormals: -127, the clamp below holds)
    return max(-126, min(126, 14 - e));
}

__device__ __forceinline__ uint32_t round16x2(bool bf16, float lo, float hi) {
    uint32_t r;
    if (bf16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

// Elements d .. d + 3 of a row of out: y * 2^exponent / l, rounded once; rows that have seen no key get zeros.  The
// power of two may leave fp32's range on the way, so it is applied in two halves.
__device__ __forceinline__ void store_out(const AttendParams &p, uint16_t *out, int32_t d, float4 y, float l, float exponent) {
    float a = 0.f, b = 0.f;
    if (l != 0.f) {
        const float h = truncf(exponent * 0.5f);
        a = exp2f(h) / l, b = exp2f(exponent - h);
    }
    if (l == 0.f) y = make_float4(0.f, 0.f, 0.f, 0.f);
    const uint32_t lo = round16x2(p.bf16, y.x * a * b, y.y * a * b), hi = round16x2(p.bf16, y.z * a * b, y.w * a * b);
    if (p.o_vec) {
        if (d < p.c.dh) *reinterpret_cast<uint2 *>(out + d) = make_uint2(lo, hi);
        return;
    }
    if (d < p.c.dh) out[d] = (uint16_t) lo;
    if (d + 1 < p.c.dh) out[d + 1] = (uint16_t) (lo >> 16);
    if (d + 2 < p.c.dh) out[d + 2] = (uint16_t) hi;
    if (d + 3 < p.c.dh) out[d + 3] = (uint16_t) (hi >> 16);
}

}// namespace paged
}// namespace b200
