// Attention over the paged 8-bit KV cache (no counterpart in the reference, whose attention composite reads one fp16
// cache per call, src/ops/attention/operator.cc:30-305):
//     out[t, h, :] = sum_j p_j v_j / sum_j p_j,   p_j = exp(scale * q[t, h, :] . k_j - max),   j <= position of t
// with k_j, v_j = code * scale of the page and kv head.
#include "paged_cache.cuh"

#include <cmath>
#include <new>

using namespace b200;
using namespace b200::paged;

namespace {

struct AttendParams {
    uint16_t *out;
    const uint16_t *q;
    int64_t o_st, o_sh, q_st, q_sh;// strides of token and head
    const uint8_t *kp, *vp;
    const float *ks, *vs;
    const int32_t *table, *lens, *offs;
    int32_t rows, q_heads, group;
    float scale;
    CacheShape c;
    TableShape t;
};

constexpr int kThreads = 128;

template<bool BF>
__device__ __forceinline__ uint16_t round16(float v) {
    if (BF) {
        uint16_t r;
        asm("cvt.rn.bf16.f32 %0, %1;" : "=h"(r) : "f"(v));
        return r;
    }
    return __half_as_ushort(__float2half_rn(v));
}
__device__ __forceinline__ float e4m3_to_f32(uint8_t c) { return unpack2(e4m3x2_to_f16x2(c)).x; }

// One CTA per new token and q head; a warp per cached token, a lane per 32nd element.
template<bool BF>
__global__ void __launch_bounds__(kThreads) attend_kernel(const AttendParams p) {
    __shared__ float part[4][256], stats[4][2];
    __shared__ int32_t owner;
    const int32_t row = (int32_t) blockIdx.x, head = (int32_t) blockIdx.y, kvh = head / p.group;
    if (threadIdx.x == 0) owner = -1;
    __syncthreads();
    for (int32_t b = threadIdx.x; b < p.t.batch; b += kThreads) {
        const Seq s = seq_of(p.lens, p.offs, p.rows, b);
        if (row >= s.first && row - s.first < s.n) owner = b;
    }
    __syncthreads();
    if (owner < 0) return;
    const int32_t b = owner;
    const Seq s = seq_of(p.lens, p.offs, p.rows, b);
    const int32_t pos = s.len - s.n + (row - s.first);
    const int32_t keys = pos < 0 ? 0 : held(pos + 1, p.t.cap), D = p.c.dh;
    const int32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    float q[8], acc[8], m = -INFINITY, l = 0.f;
    for (int i = 0; i < 8; ++i) {
        const int32_t d = lane + 32 * i;
        q[i] = d < D ? f16or_bf16x2<BF>(p.q[(int64_t) row * p.q_st + (int64_t) head * p.q_sh + d]).x : 0.f;
        acc[i] = 0.f;
    }
    for (int32_t j = warp; j < keys; j += 4) {
        const int32_t page = p.table[(int64_t) b * p.t.stride + j / p.c.page], at = j % p.c.page;
        if (page < 0 || page >= p.c.pages) continue;
        const uint8_t *k = p.kp + page * p.c.k.sn + kvh * p.c.k.sh + at * p.c.k.sp, *v = p.vp + page * p.c.v.sn + kvh * p.c.v.sh + at * p.c.v.sp;
        float x = 0.f;
        for (int i = 0; i < 8; ++i) {
            if (lane + 32 * i < D) x = fmaf(q[i], e4m3_to_f32(k[lane + 32 * i]), x);
        }
        x = warp_sum(x) * p.ks[page * p.c.k.cn + kvh * p.c.k.ch] * p.scale;
        const float m_new = fmaxf(m, x), shrink = m == -INFINITY ? 0.f : expf(m - m_new), w = m_new == -INFINITY ? 0.f : expf(x - m_new);
        const float wv = w * p.vs[page * p.c.v.cn + kvh * p.c.v.ch];
        l = l * shrink + w, m = m_new;
        for (int i = 0; i < 8; ++i) {
            if (lane + 32 * i < D) acc[i] = acc[i] * shrink + wv * e4m3_to_f32(v[lane + 32 * i]);
        }
    }
    for (int i = 0; i < 8; ++i) part[warp][lane + 32 * i] = acc[i];
    if (lane == 0) stats[warp][0] = m, stats[warp][1] = l;
    __syncthreads();
    float top = -INFINITY, sum = 0.f, w[4];
    for (int i = 0; i < 4; ++i) top = fmaxf(top, stats[i][0]);
    for (int i = 0; i < 4; ++i) {
        w[i] = stats[i][0] == -INFINITY ? 0.f : expf(stats[i][0] - top);
        sum += w[i] * stats[i][1];
    }
    for (int32_t d = threadIdx.x; d < D; d += kThreads) {
        float y = 0.f;
        for (int i = 0; i < 4; ++i) y += w[i] * part[i][d];
        p.out[(int64_t) row * p.o_st + (int64_t) head * p.o_sh + d] = round16<BF>(sum == 0.f ? 0.f : y / sum);
    }
}

struct AttendDesc {
    Device device;
    int device_id, sm_count;
    CacheShape c;
    TableShape t;
    int32_t rows, q_heads;
    bool bf16;
    int64_t o_st, o_sh, q_st, q_sh;
    float scale;
};

}// namespace

INFINIOP_API infiniopStatus_t infiniopCreatePagedAttentionDescriptor(
    infiniopHandle_t handle, infiniopPagedAttentionDescriptor_t *desc_ptr, infiniopTensorDescriptor_t out_desc,
    infiniopTensorDescriptor_t q_desc, infiniopTensorDescriptor_t k_pages_desc, infiniopTensorDescriptor_t v_pages_desc,
    infiniopTensorDescriptor_t k_scales_desc, infiniopTensorDescriptor_t v_scales_desc,
    infiniopTensorDescriptor_t block_table_desc, infiniopTensorDescriptor_t seq_lens_desc,
    infiniopTensorDescriptor_t q_offsets_desc, float scale) {
    if (handle == nullptr || handle->device != DevNvGpu) return STATUS_BAD_DEVICE;
    if (desc_ptr == nullptr) return STATUS_MEMORY_NOT_ALLOCATED;
    if (out_desc == nullptr || q_desc == nullptr || !std::isfinite(scale)) return STATUS_BAD_PARAM;
    AttendDesc d{};
    infiniopStatus_t st = check_cache(k_pages_desc, v_pages_desc, k_scales_desc, v_scales_desc, d.c);
    if (st != STATUS_SUCCESS) return st;
    st = check_tables(block_table_desc, seq_lens_desc, q_offsets_desc, d.c.page, d.t);
    if (st != STATUS_SUCCESS) return st;
    if (q_desc->ndim != 3) return STATUS_BAD_TENSOR_SHAPE;
    const uint64_t rows = q_desc->shape[0], heads = q_desc->shape[1];
    if (heads == 0 || heads > 0xFFFFull || heads % (uint64_t) d.c.heads != 0) return STATUS_BAD_TENSOR_SHAPE;
    for (auto *x : {q_desc, out_desc}) {
        st = check_rows(x, rows, heads, (uint64_t) d.c.dh, q_desc->dt);
        if (st != STATUS_SUCCESS) return st;
    }
    if (!disjoint(out_desc)) return STATUS_BAD_TENSOR_STRIDES;
    if (!d.t.offsets && rows != (uint64_t) d.t.batch) return STATUS_BAD_TENSOR_SHAPE;
    auto *h = reinterpret_cast<Handle *>(handle);
    d.device = DevNvGpu, d.device_id = h->device_id, d.sm_count = h->sm_count;
    d.rows = (int32_t) rows, d.q_heads = (int32_t) heads, d.bf16 = dt_eq(q_desc->dt, BF16), d.scale = scale;
    d.o_st = out_desc->strides[0], d.o_sh = out_desc->strides[1], d.q_st = q_desc->strides[0], d.q_sh = q_desc->strides[1];
    auto *r = new (std::nothrow) AttendDesc(d);
    if (r == nullptr) return STATUS_MEMORY_NOT_ALLOCATED;
    *desc_ptr = reinterpret_cast<infiniopPagedAttentionDescriptor_t>(r);
    return STATUS_SUCCESS;
}

INFINIOP_API infiniopStatus_t infiniopGetPagedAttentionWorkspaceSize(infiniopPagedAttentionDescriptor_t desc, uint64_t *size) {
    if (desc == nullptr || desc->device != DevNvGpu) return STATUS_BAD_DEVICE;
    if (size == nullptr) return STATUS_BAD_PARAM;
    *size = 0;
    return STATUS_SUCCESS;
}

INFINIOP_API infiniopStatus_t infiniopPagedAttention(infiniopPagedAttentionDescriptor_t desc, void *workspace,
                                                     uint64_t workspace_size, void *out, void const *q, void const *k_pages,
                                                     void const *v_pages, void const *k_scales, void const *v_scales,
                                                     void const *block_table, void const *seq_lens, void const *q_offsets,
                                                     void *stream) {
    (void) workspace;
    (void) workspace_size;
    if (desc == nullptr || desc->device != DevNvGpu) return STATUS_BAD_DEVICE;
    auto *d = reinterpret_cast<AttendDesc *>(desc);
    if (d->rows == 0 || d->t.batch == 0) return STATUS_SUCCESS;
    if (out == nullptr || q == nullptr || seq_lens == nullptr || d->t.offsets != (q_offsets != nullptr)) return STATUS_BAD_PARAM;
    // a table without columns or a pool without pages has no keys: every token gets zeros
    const bool empty = d->t.cols == 0 || d->c.pages == 0;
    if (!empty && (k_pages == nullptr || v_pages == nullptr || k_scales == nullptr || v_scales == nullptr || block_table == nullptr)) return STATUS_BAD_PARAM;
    DeviceGuard guard(d->device_id);
    AttendParams p{reinterpret_cast<uint16_t *>(out), reinterpret_cast<const uint16_t *>(q), d->o_st, d->o_sh, d->q_st, d->q_sh,
                   reinterpret_cast<const uint8_t *>(k_pages), reinterpret_cast<const uint8_t *>(v_pages),
                   reinterpret_cast<const float *>(k_scales), reinterpret_cast<const float *>(v_scales),
                   reinterpret_cast<const int32_t *>(block_table), reinterpret_cast<const int32_t *>(seq_lens),
                   reinterpret_cast<const int32_t *>(q_offsets), d->rows, d->q_heads, d->q_heads / d->c.heads, d->scale, d->c, d->t};
    if (empty) p.t.cap = 0;
    auto st = reinterpret_cast<cudaStream_t>(stream);
    const dim3 grid((unsigned) d->rows, (unsigned) d->q_heads);
    if (d->bf16) attend_kernel<true><<<grid, kThreads, 0, st>>>(p);
    else attend_kernel<false><<<grid, kThreads, 0, st>>>(p);
    return check_launch("paged attention");
}

INFINIOP_API infiniopStatus_t infiniopDestroyPagedAttentionDescriptor(infiniopPagedAttentionDescriptor_t desc) {
    if (desc == nullptr || desc->device != DevNvGpu) return STATUS_BAD_DEVICE;
    delete reinterpret_cast<AttendDesc *>(desc);
    return STATUS_SUCCESS;
}
