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
    bool bf16, vec, q_vec, o_vec, o_vec8;// whole vectors: 16 bytes of codes, q and out, 8 bytes of out
    FastDiv page_div, group_div;// by the page size and by the q heads per kv head
    CacheShape c;
    TableShape t;
};

__device__ __forceinline__ uint4 lds128(uint32_t a) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
    return v;
}
// Copies to shared memory that the thread does not wait for; zeros where there is nothing to copy.
__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src, bool valid) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void *src, bool valid) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(valid ? 4 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template<int N>
__device__ __forceinline__ void cp_async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

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

// Keys that the rr-th query row (new token x q head of the group) of a sequence may see (pages may be missing among them).
__device__ __forceinline__ int32_t keys_of_row(const AttendParams &p, const Seq &s, uint32_t rr) {
    return max(0, min(s.len - s.n + (int32_t) p.group_div.div(rr) + 1, held(s.len, p.t.cap)));
}
// One of the first `keys` tokens of sequence b lies in a page.
__device__ __forceinline__ bool any_page(const AttendParams &p, int32_t b, int32_t keys) {
    const int32_t cols = keys > 0 ? (int32_t) p.page_div.div((uint32_t) keys - 1) + 1 : 0;
#pragma unroll 1
    for (int32_t i = 0; i < cols; ++i) {
        const int32_t id = p.table[(int64_t) b * p.t.stride + i];
        if (id >= 0 && id < p.c.pages) return true;
    }
    return false;
}
// A row's output is y * 2^exponent / l; the power of two may leave fp32's range on the way, so it is applied as two
// factors.  l = 0: a row that sees no key gets zeros; one whose scores are all -inf is 0 / 0.  (A score of NaN makes l
// NaN, also where the row has no reference for it: l is added up and scaled, never left out.)
__device__ __forceinline__ float2 out_factors(const AttendParams &p, int32_t b, int32_t keys, float l, float exponent) {
    if (l == 0.f) {
        const float none = any_page(p, b, keys) ? NAN : 0.f;
        return make_float2(none, none);
    }
    const float h = truncf(exponent * 0.5f);
    return make_float2(exp2f(h) / l, exp2f(exponent - h));
}
// Elements d .. d + 3 of a row of out, rounded once.
__device__ __forceinline__ void store_out(const AttendParams &p, uint16_t *out, int32_t d, float4 y, float2 f) {
    const float a = f.x, b = f.y;
    if (a == 0.f) y = make_float4(0.f, 0.f, 0.f, 0.f);
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

// Row of out of the rr-th query row (new token x q head of the group) of a sequence and kv head.
__device__ __forceinline__ uint16_t *row_of_out(const AttendParams &p, const Seq &s, int32_t kvh, uint32_t rr) {
    const int32_t tok = (int32_t) p.group_div.div(rr), hd = (int32_t) rr - tok * p.group;
    return p.out + (int64_t) (s.first + tok) * p.o_st + (int64_t) (kvh * p.group + hd) * p.o_sh;
}

// ---- equal stretches of work ------------------------------------------------------------------------------------
// The work of a call is a list of units, tiles of cached tokens, ordered by sequence, kv head, block of query rows,
// tile; CTA c takes units [c * each, (c + 1) * each).  An item (sequence, kv head, block of rows) that lies in one
// stretch is finished there; of any other, each CTA stores its part (unnormalised output and the rows' references) and
// join_kernel adds the parts in the order of the list.

__device__ __forceinline__ int64_t stretch_of(int64_t total, int64_t least) {
    const int64_t each = divide(total + gridDim.x - 1, gridDim.x);
    return each < least ? least : each;
}

// Sum over the CTA of a 64-bit value and the sum over the threads before; `slot`: WARPS words.
template<int WARPS>
__device__ __forceinline__ int64_t cta_exclusive_sum64(int64_t v, int64_t *slot, int64_t &total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int64_t incl = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t u = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += u;
    }
    __syncthreads();
    if (lane == 31) slot[warp] = incl;
    __syncthreads();
    int64_t before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
        if (w < warp) before += slot[w];
        total += slot[w];
    }
    return before + incl - v;
}

// log2 of a scale; exact and cheap for the powers of two that append writes.  Zero gives -inf.  All lanes call it.
__device__ __forceinline__ float log2_of(float v) {
    const uint32_t u = __float_as_uint(v);
    if (__any_sync(0xffffffffu, (u & 0x807FFFFFu) != 0 || u == 0)) return log2f(v);
    return (float) ((int32_t) (u >> 23) - 127);
}

// A row's part: sum over its keys of 2^(score - m) = l, and of 2^(score - w) * scale of the value * code = the output
struct PartHead {
    float m, l, w;
    int32_t keys;// decoding: keys_of_row
};
struct CtaMeta {
    int32_t b, kvh, rb;// the item that begins in this CTA's stretch and goes on behind it; b < 0: none
    int32_t last;      // the CTA whose stretch holds its end
};
struct SplitParams {
    AttendParams a;
    float *parts;   // [cta][2][rows][DHC]: the part of an item that began before the stretch, and of one that goes on
    PartHead *heads;// [cta][2][rows]
    CtaMeta *meta;  // [cta]
    uint32_t cluster;// decoding: CTAs of a cluster that share an item (0: equal stretches)
    bool one_poll;  // prompts: waits give up after their first poll (a test's)
};
static inline uint64_t split_bytes(uint64_t ctas, uint64_t rows, uint64_t dhc) {
    return ctas * (2 * rows * (sizeof(PartHead) + dhc * 4) + sizeof(CtaMeta));
}
static inline SplitParams split_params(const AttendParams &a, void *workspace, uint64_t ctas, uint64_t rows, uint64_t dhc) {
    SplitParams s{};
    s.a = a;
    s.parts = reinterpret_cast<float *>(workspace);
    s.heads = reinterpret_cast<PartHead *>(s.parts + ctas * 2 * rows * dhc);
    s.meta = reinterpret_cast<CtaMeta *>(s.heads + ctas * 2 * rows);
    return s;
}

// Joins the parts of the item that begins in stretch blockIdx.x and goes on behind it.  A decoding item (ROWS 8 or 16) may
// have dozens of parts: a block takes two rows, and for each, four groups of threads add every fourth part.  A block of
// prompt rows has few: eight rows per block, one group.  kBatch parts are loaded at a time (the loads' latency is all there
// is to this kernel), and everything is added in the order of the list.
template<int ROWS>
struct JoinShape {
    static constexpr int kRows = ROWS >= 128 ? 8 : 2, kGroups = ROWS >= 128 ? 1 : 4, kBatch = ROWS >= 128 ? 3 : 7;
};
template<int DHC, int ROWS>
__global__ void __launch_bounds__(JoinShape<ROWS>::kRows * JoinShape<ROWS>::kGroups * DHC / 4) join_kernel(const SplitParams dp) {
    constexpr int kJoinRows = JoinShape<ROWS>::kRows, kJoinGroups = JoinShape<ROWS>::kGroups, kBatch = JoinShape<ROWS>::kBatch;
    constexpr int kLanes = DHC / 4;
    __shared__ float4 acc[kJoinRows][kJoinGroups][kLanes];
    __shared__ float stat[kJoinRows][kJoinGroups][3];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const AttendParams &p = dp.a;
    const CtaMeta item = dp.meta[blockIdx.x];
    if (item.b < 0) return;
    const int ln = (int) threadIdx.x % kLanes, grp = (int) threadIdx.x / kLanes % kJoinGroups, sub = (int) threadIdx.x / (kLanes * kJoinGroups);
    const int r = (int) blockIdx.y * kJoinRows + sub, first = (int) blockIdx.x;
    const Seq s = seq_of(p.lens, p.offs, p.rows, item.b);
    const uint32_t rr = (uint32_t) item.rb * ROWS + (uint32_t) r;
    const bool have = rr < (uint32_t) s.n * (uint32_t) p.group;
    float m = -INFINITY, l = 0.f, w = -INFINITY;
    float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int32_t c0 = first + grp; have && c0 <= item.last; c0 += kJoinGroups * kBatch) {
        PartHead h[kBatch];
        float4 v[kBatch];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const int32_t c = c0 + i * kJoinGroups;
            const int64_t at = ((int64_t) c * 2 + (c == first ? 1 : 0)) * ROWS + r;
            h[i] = PartHead{-INFINITY, 0.f, -INFINITY, 0};
            v[i] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (c <= item.last) h[i] = dp.heads[at], v[i] = *reinterpret_cast<const float4 *>(dp.parts + at * DHC + ln * 4);
        }
        float m1 = m, w1 = w;
#pragma unroll
        for (int i = 0; i < kBatch; ++i) m1 = fmaxf(m1, h[i].m), w1 = fmaxf(w1, h[i].w);
        const float m0 = m1 == -INFINITY ? 0.f : m1;// (parts without a reference: their l is 0 or NaN)
        l *= fast_exp2(m - m0);// (from -inf: 0)
#pragma unroll
        for (int i = 0; i < kBatch; ++i) l += h[i].l * fast_exp2(h[i].m - m0);
        m = m1;
        if (w1 != -INFINITY) {
            const float f0 = fast_exp2(w - w1);
            y.x *= f0, y.y *= f0, y.z *= f0, y.w *= f0;
#pragma unroll
            for (int i = 0; i < kBatch; ++i) {
                const float f = fast_exp2(h[i].w - w1);
                y.x += v[i].x * f, y.y += v[i].y * f, y.z += v[i].z * f, y.w += v[i].w * f;
            }
            w = w1;
        }
    }
    acc[sub][grp][ln] = y;
    if (ln == 0) stat[sub][grp][0] = m, stat[sub][grp][1] = l, stat[sub][grp][2] = w;
    __syncthreads();
    if (grp != 0 || !have) return;
    m = w = -INFINITY, l = 0.f, y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int i = 0; i < kJoinGroups; ++i) m = fmaxf(m, stat[sub][i][0]), w = fmaxf(w, stat[sub][i][2]);
#pragma unroll
    for (int i = 0; i < kJoinGroups; ++i) {
        l += stat[sub][i][1] * fast_exp2(stat[sub][i][0] - (m == -INFINITY ? 0.f : m));
        if (stat[sub][i][2] != -INFINITY) {
            const float f = fast_exp2(stat[sub][i][2] - w);
            const float4 v = acc[sub][i][ln];
            y.x += f * v.x, y.y += f * v.y, y.z += f * v.z, y.w += f * v.w;
        }
    }
    store_out(p, row_of_out(p, s, item.kvh, rr), ln * 4, y, out_factors(p, item.b, keys_of_row(p, s, rr), l, w - m));
}

template<int DHC, int ROWS>
static inline cudaError_t launch_join(const SplitParams &sp, uint32_t ctas, cudaStream_t st) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ctas - 1, ROWS / JoinShape<ROWS>::kRows);
    cfg.blockDim = dim3(JoinShape<ROWS>::kRows * JoinShape<ROWS>::kGroups * DHC / 4);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr, cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, join_kernel<DHC, ROWS>, sp);
}

// Prompts and chunks (paged_prefill.cu): tiles of 64 cached tokens, items of 256 query rows (128 for head sizes beyond 128),
// one CTA per SM.
constexpr int kPrefillKeys = 64;
static inline int prefill_rows(int dhc) { return dhc <= 128 ? 256 : 128; }
constexpr int64_t kPrefillMaxBatch = 4096;// sequences whose unit counts fit the kernel's shared memory
cudaError_t launch_prefill(const AttendParams &a, void *workspace, int dhc, uint32_t ctas, int device_id, cudaStream_t st);

}// namespace paged
}// namespace b200
