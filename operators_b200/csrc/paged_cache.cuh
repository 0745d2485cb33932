// What the operators on the paged 8-bit KV cache share: the checks of the cache's tensors (one set of rules for all
// four descriptors), the geometry that the kernels take, and the conversions of e4m3 codes.
#pragma once

#include "common.cuh"
#include "paged_index.h"

#include <algorithm>
#include <initializer_list>
#include <utility>

namespace b200 {
namespace paged {

// Pages, heads and tokens of one pool: element (n, h, p, d) at n * sn + h * sh + p * sp + d, the scale of page n and
// head h at n * cn + h * ch.  64-bit strides: a pool passes 2^32 elements long before it fills the GPU.
struct PoolStrides {
    int64_t sn, sh, sp, cn, ch;
};
struct CacheShape {
    int32_t pages, heads, page, dh;
    PoolStrides k, v;
};
// block table and lengths
struct TableShape {
    int32_t batch, cols, cap;// cap = cols * page size: tokens that a row can hold
    int64_t stride;
    bool offsets;// q_offsets are given
};

// Every dimension but the last: positive stride where it is more than one long; the last: unit stride.
static inline bool unit_rows(const TensorDescriptor *t) {
    for (uint64_t i = 0; i < t->ndim; ++i) {
        if (t->shape[i] > 1 && (i + 1 < t->ndim ? t->strides[i] <= 0 : t->strides[i] != 1)) return false;
    }
    return true;
}
// No two elements share an address (tensors that are written): sorted by stride, each dimension steps over all that
// the smaller ones span.
static inline bool disjoint(const TensorDescriptor *t) {
    std::pair<int64_t, uint64_t> dims[8];
    uint64_t n = 0;
    for (uint64_t i = 0; i < t->ndim && i < 8; ++i) {
        if (t->shape[i] == 0) return true;
        if (t->shape[i] > 1) dims[n++] = {t->strides[i], t->shape[i]};
    }
    std::sort(dims, dims + n);
    int64_t span = 1;
    for (uint64_t i = 0; i < n; ++i) {
        if (dims[i].first < span) return false;
        span += dims[i].first * (int64_t) (dims[i].second - 1);
    }
    return true;
}

// The pools and scales; fills `c`.
static inline infiniopStatus_t check_cache(const TensorDescriptor *kp, const TensorDescriptor *vp, const TensorDescriptor *ks,
                                           const TensorDescriptor *vs, CacheShape &c) {
    if (kp == nullptr || vp == nullptr || ks == nullptr || vs == nullptr) return STATUS_BAD_PARAM;
    if (kp->ndim != 4 || vp->ndim != 4 || ks->ndim != 2 || vs->ndim != 2) return STATUS_BAD_TENSOR_SHAPE;
    for (int i = 0; i < 4; ++i) {
        if (kp->shape[i] != vp->shape[i]) return STATUS_BAD_TENSOR_SHAPE;
    }
    for (int i = 0; i < 2; ++i) {
        if (ks->shape[i] != kp->shape[i] || vs->shape[i] != kp->shape[i]) return STATUS_BAD_TENSOR_SHAPE;
    }
    if (kp->shape[0] > 0x7FFFFFFFull || kp->shape[1] == 0 || kp->shape[1] > 0xFFFFull || kp->shape[2] == 0 ||
        kp->shape[2] > 0x3FFFFFull || kp->shape[3] == 0 || kp->shape[3] > 256) {
        return STATUS_BAD_TENSOR_SHAPE;
    }
    if (!dt_eq(kp->dt, F8E4M3) || !dt_eq(vp->dt, F8E4M3) || !dt_eq(ks->dt, F32) || !dt_eq(vs->dt, F32)) {
        return STATUS_BAD_TENSOR_DTYPE;
    }
    if (!unit_rows(kp) || !unit_rows(vp) || !disjoint(kp) || !disjoint(vp)) return STATUS_BAD_TENSOR_STRIDES;
    for (const TensorDescriptor *t : {ks, vs}) {
        for (int i = 0; i < 2; ++i) {
            if (t->shape[i] > 1 && t->strides[i] <= 0) return STATUS_BAD_TENSOR_STRIDES;
        }
        if (!disjoint(t)) return STATUS_BAD_TENSOR_STRIDES;
    }
    c.pages = (int32_t) kp->shape[0], c.heads = (int32_t) kp->shape[1], c.page = (int32_t) kp->shape[2], c.dh = (int32_t) kp->shape[3];
    c.k = {kp->strides[0], kp->strides[1], kp->strides[2], ks->strides[0], ks->strides[1]};
    c.v = {vp->strides[0], vp->strides[1], vp->strides[2], vs->strides[0], vs->strides[1]};
    return STATUS_SUCCESS;
}

// Block table and lengths; `offs` may be null.
static inline infiniopStatus_t check_tables(const TensorDescriptor *table, const TensorDescriptor *lens, const TensorDescriptor *offs,
                                            int32_t page, TableShape &t) {
    if (table == nullptr || lens == nullptr) return STATUS_BAD_PARAM;
    if (table->ndim != 2 || lens->ndim != 1 || (offs != nullptr && offs->ndim != 1)) return STATUS_BAD_TENSOR_SHAPE;
    const uint64_t batch = table->shape[0], cols = table->shape[1];
    if (lens->shape[0] != batch || (offs != nullptr && offs->shape[0] != batch + 1)) return STATUS_BAD_TENSOR_SHAPE;
    if (batch > 0xFFFFFFull || cols > 0x7FFFFFFFull || cols * (uint64_t) page > 0x7FFFFFFFull) return STATUS_BAD_TENSOR_SHAPE;
    if (!dt_eq(table->dt, I32) || !dt_eq(lens->dt, I32) || (offs != nullptr && !dt_eq(offs->dt, I32))) return STATUS_BAD_TENSOR_DTYPE;
    if (!unit_rows(table) || !unit_rows(lens) || (offs != nullptr && !unit_rows(offs))) return STATUS_BAD_TENSOR_STRIDES;
    t.batch = (int32_t) batch, t.cols = (int32_t) cols, t.cap = (int32_t) (cols * (uint64_t) page);
    t.stride = table->strides[0], t.offsets = offs != nullptr;
    return STATUS_SUCCESS;
}

// Every pointer is a multiple of `bytes` (a power of two): elements are read and written whole.
static inline bool aligned_to(uintptr_t bytes, std::initializer_list<const void *> pointers) {
    uintptr_t all = 0;
    for (const void *p : pointers) all |= reinterpret_cast<uintptr_t>(p);
    return (all & (bytes - 1)) == 0;
}

// New tokens' tensors [rows, heads, dh]: fp16 or bf16.
static inline infiniopStatus_t check_rows(const TensorDescriptor *x, uint64_t rows, uint64_t heads, uint64_t dh, DataLayout dt) {
    if (x->ndim != 3 || x->shape[0] != rows || x->shape[1] != heads || x->shape[2] != dh || rows > 0x7FFFFFFFull) return STATUS_BAD_TENSOR_SHAPE;
    if ((!dt_eq(x->dt, F16) && !dt_eq(x->dt, BF16)) || !dt_eq(x->dt, dt)) return STATUS_BAD_TENSOR_DTYPE;
    return unit_rows(x) ? STATUS_SUCCESS : STATUS_BAD_TENSOR_STRIDES;
}

// ---------------------------------------------------------------- device side --

// two codes (low byte first) <-> two values; the decoding is exact, the encoding rounds to nearest even and saturates
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint16_t c) {
    uint32_t r;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(c));
    return r;
}
// four codes of a word
__device__ __forceinline__ void e4m3x4_to_f16x4(uint32_t c, uint32_t &lo, uint32_t &hi) {
    asm("{\n\t.reg .b16 l, h;\n\t"
        "mov.b32 {l, h}, %2;\n\t"
        "cvt.rn.f16x2.e4m3x2 %0, l;\n\t"
        "cvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
        : "=r"(lo), "=r"(hi)
        : "r"(c));
}
__device__ __forceinline__ uint16_t f32x2_to_e4m3x2(float lo, float hi) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}

// a / b of values that mostly fit 32 bits (a 64-bit division takes a few hundred cycles)
__device__ __forceinline__ int64_t divide(int64_t a, int64_t b) {
    return ((a | b) >> 32) == 0 ? (int64_t) ((uint32_t) a / (uint32_t) b) : a / b;
}

// Largest finite magnitudes of two 16-bit floats, as bit patterns per half (the patterns of one sign are ordered like
// the values); infinities and NaN count as zero.
template<bool BF>
__device__ __forceinline__ uint32_t finite_abs2(uint32_t w) {
    const uint32_t inf = BF ? 0x7F807F80u : 0x7C007C00u, a = w & 0x7FFF7FFFu;
    return a & ~__vcmpgeu2(a, inf);
}
// max(top, |w|) per half; NaN in w is passed over
template<bool BF>
__device__ __forceinline__ uint32_t abs_max2(uint32_t top, uint32_t w) {
    uint32_t r;
    if (BF) asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(top), "r"(w & 0x7FFF7FFFu));
    else asm("max.f16x2 %0, %1, %2;" : "=r"(r) : "r"(top), "r"(w & 0x7FFF7FFFu));
    return r;
}
template<bool BF>
__device__ __forceinline__ float2 f16or_bf16x2(uint32_t w) {
    return unpack2_t<BF ? kBF16 : kF16>(w);
}

}// namespace paged
}// namespace b200
