// Attention over the paged 8-bit KV cache for few new tokens per sequence (no counterpart in the reference, whose
// attention composite reads one fp16 cache per call, src/ops/attention/operator.cc:30-305):
//     out[t, h, :] = sum_j p_j v_j / sum_j p_j,   p_j = 2^(log2e * scale * q[t, h, :] . k_j - m),   j <= position of t
// with k_j, v_j = code * scale of the page and kv head.
//
// What bounds it: one read of the codes, 2 * dh bytes per cached token and kv head, whatever the number of q heads that
// share the kv head.  So a warp owns up to 8 or 16 query rows (the q heads of a group x the new tokens) and a tile of
// 32 cached tokens at a time, and everything else is arranged around keeping loads in flight:
//  * Work is a list of units = tiles of 32 tokens, ordered by sequence, kv head, block of query rows, tile.  Every
//    CTA takes an equal stretch of the list, whatever the lengths (they are read on the device, so a captured graph
//    follows the growing sequences); a stretch may end inside a sequence, and then the parts are joined by a second,
//    small kernel in the order of the list.  No CTA waits for another.
//  * A warp loads its own tiles with cp.async into a ring of its own in shared memory: no barrier in the loop.
//  * Products run on mma.m16n8k16 (fp16 in, fp32 accumulation) with 16 cached tokens (q . k) or 16 head elements
//    (p . v) as its rows and the query rows as its 8 columns: the contraction is far below a tcgen05 tile.  Codes
//    become fp16 exactly in registers.  The contraction index is only a label, so every lane reads 16 consecutive
//    bytes of a row; for p . v the bytes of two tokens are paired with one byte permutation per 4 elements.
//  * q in fp16 too: each bf16 row is multiplied by a power of two that brings its largest element to [2^14, 2^15), which
//    holds every element that is not 2^-29 of the largest exactly, and is undone in the score's factor.
//  * The running maximum m of a row moves only when a score exceeds it by more than a factor 2, so most tiles rescale
//    nothing.  The weight of a value is w_j = p_j * (scale of v_j): its own reference M keeps fp16 weights
//    between 2^15 and what is 2^-28 of the largest (2^-39 with subnormals), however the pages' scales differ.  Sums
//    of p and the output stay in fp32.
//  * Up to 8 query rows take one column block of the product, up to 16 take two: 16 sequences of 2000 tokens, 32 heads on 8
//    of 128 elements, 8 rows 27 us with one and 12 rows 33 us with two; more rows take further items, or the tcgen05 kernel
//    (prefill_is_faster).  Tiles that lie in one page (page sizes that are multiples of 32) read one page id and scale per
//    tile: 32 sequences of 2048 tokens 36 us with pages of 64, 41 us in the general form with pages of 16.
// Measured: 32 sequences of 1024 to 8192 tokens, 32 heads on 8 of 128 elements: 66 us, 4.75 TB/s; one sequence of 131072:
// 58 to 59 us, 4.6 TB/s.  The loop itself runs at 6.7 TB/s; the rest is the start (5 us), SMs that get less bandwidth than
// others (7 us), and the join (5 us).
#include "paged_cache.cuh"
#include "paged_attention.cuh"
#include "tc_ptx.cuh"

#include <atomic>
#include <cmath>
#include <new>

using namespace b200;
using namespace b200::paged;

namespace {

constexpr int kWarps = 4, kThreads = 32 * kWarps;
constexpr int kTile = 32;      // cached tokens per warp and step
constexpr int kMinUnits = 4;   // a CTA takes at least a tile per warp
// What the start and the end of an item cost, in tiles: with 4, 8 and 12 of them 12 sequences of up to 2500 tokens and 5 new
// ones, 40 heads on 8, take 23.1, 22.6, 22.6 us at a head size of 64, 31.9, 30.6, 30.7 at 128, 63.4, 60.2, 58.9 at 256; 32
// sequences of one new token differ by 1 %.
constexpr int kItemUnits = 8;
constexpr uint32_t kMaxCluster = 8;
constexpr int64_t kClusterRounds = 4;
constexpr float kSlack = 1.f;  // log2 by which a score may exceed its row's reference
constexpr float kLift = 14.f;  // weights are stored times 2^14: at most 2^(14 + slack) < 65504

// Resident CTAs per SM and stages of a warp's ring.  8 rows of a head size up to 128 leave registers for 12 to 16 warps
// per SM, which hide each other's latency better than deeper rings of fewer warps do.
__host__ __device__ constexpr int ctas_per_sm(int dhc, int nt) { return dhc == 256 ? 1 : dhc == 128 ? (nt == 1 ? 3 : 2) : (nt == 1 ? 4 : 3); }
__host__ __device__ constexpr int stages_of(int dhc, int nt) { return dhc == 128 && nt == 1 ? 2 : 3; }
// One stage of a warp's ring: K rows, V rows, their scales, the mask of valid tokens.
__host__ __device__ constexpr int stage_bytes(int dhc) { return 2 * kTile * dhc + 2 * kTile * 4 + 16; }
__host__ __device__ constexpr int smem_bytes(int dhc, int nt) { return kWarps * stages_of(dhc, nt) * stage_bytes(dhc); }

// Byte position of 16-byte chunk c of row r in a tile of rows of DHC bytes.  Chosen so that the lanes of a quarter warp
// hit different banks in both access patterns: 4 chunks of each of 2 neighbouring rows (q . k) and 2 chunks of each of
// 4 rows that are 2 apart (p . v).
template<int DHC>
__device__ __forceinline__ uint32_t chunk_at(uint32_t r, uint32_t c) {
    if (DHC == 128) return r * 128 + ((c ^ (r & 7u)) << 4);
    if (DHC == 64) return (r >> 1) * 128 + (((((r & 1u) << 2) | c) ^ ((r >> 1 & 3u) << 1)) << 4);
    return r * 256 + ((c ^ ((r >> 1 & 1u) | (((r ^ (r >> 2)) & 1u) << 2))) << 4);
}
// The chunk that lane t (of 4) of a row reads as its h-th in q . k.
template<int DHC>
__device__ __forceinline__ uint32_t key_chunk(uint32_t t, uint32_t h) {
    return DHC == 128 ? 2 * t + h : t + 4 * h;
}

__device__ __forceinline__ void mma_f16(float *c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}

__device__ __forceinline__ uint2 lds64(uint32_t a) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ float lds_f32(uint32_t a) {
    float v;
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ uint32_t lds_u32(uint32_t a) {
    uint32_t v;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
    return v;
}

__device__ __forceinline__ int64_t shfl64(int64_t v, int lane) { return __shfl_sync(0xffffffffu, v, lane); }

// Blocks of query rows and tiles of a sequence; its units are blocks x kv heads x tiles.
template<int ROWS>
__device__ __forceinline__ void extent_of(const AttendParams &p, const Seq &s, int32_t &blocks, int32_t &tiles) {
    blocks = (int32_t) (((uint32_t) s.n * (uint32_t) p.group + ROWS - 1) / ROWS);// (rows x group < 2^31)
    const int32_t keys = held(s.len, p.t.cap);
    tiles = keys > 0 ? (keys - 1) / kTile + 1 : 1;// a sequence without keys still writes zeros
}

// The state of a warp's ring while it walks tiles first, first + kWarps, .. of one item.
struct Walk {
    int32_t keys;
    const uint8_t *k, *v;// this kv head's pages
    const float *ks, *vs;
};

// DHC: head size rounded up to 64, 128 or 256; NT: 8 * NT query rows; ONE: a tile lies in one page (the page size is a
// multiple of 32) and its rows are whole aligned vectors, so one page id, two scales and a count describe it.
template<int DHC, int NT, bool ONE>
__global__ void __launch_bounds__(kThreads, ctas_per_sm(DHC, NT)) decode_kernel(const SplitParams dp) {
    constexpr int kRows = 8 * NT, kStages = stages_of(DHC, NT), kStage = stage_bytes(DHC), kChunks = DHC / 16;
    constexpr int kHalf = DHC / 64;  // chunks per lane and row in q . k
    constexpr int kSteps = DHC / 16; // mma steps of q . k, and m-tiles of p . v
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ int64_t slot[kWarps], found_base;
    __shared__ int32_t found_b;
    const AttendParams &p = dp.a;
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const uint32_t ring = (uint32_t) __cvta_generic_to_shared(smem) + warp * kStages * kStage;

    // ---- this CTA's stretch of the units
    // (with clusters: item blockIdx.x / CTAs of a cluster, and of its tiles this CTA's share)
    const uint32_t cl = dp.cluster, rank = cl > 0 ? blockIdx.x % cl : 0u;
    auto units_of = [&](int32_t b) -> int64_t {
        int32_t blocks, tiles;
        extent_of<kRows>(p, seq_of(p.lens, p.offs, p.rows, b), blocks, tiles);
        return (int64_t) blocks * (cl > 0 ? 1 : tiles + kItemUnits) * p.c.heads;
    };
    int64_t mine = 0, total;
    for (int32_t b = (int32_t) threadIdx.x; b < p.t.batch; b += kThreads) mine += units_of(b);
    cta_exclusive_sum64<kWarps>(mine, slot, total);
    const int64_t each = cl > 0 ? 1 : stretch_of(total, kMinUnits);
    int64_t u = cl > 0 ? (int64_t) (blockIdx.x / cl) : each * blockIdx.x;
    const int64_t u_end = u + each < total ? u + each : total;
    if (u >= u_end) {// (a cluster's CTAs leave together)
        if (cl > 0) return;
        if (threadIdx.x == 0) dp.meta[blockIdx.x] = CtaMeta{-1, 0, 0, 0};
        asm volatile("griddepcontrol.launch_dependents;");
        return;
    }
    {
        int64_t base = 0;
        for (int32_t b0 = 0; b0 < p.t.batch && base <= u; b0 += kThreads) {
            const int32_t b = b0 + (int32_t) threadIdx.x;
            const int64_t n = b < p.t.batch ? units_of(b) : 0;
            int64_t sum;
            const int64_t before = base + cta_exclusive_sum64<kWarps>(n, slot, sum);
            if (u >= before && u - before < n) found_b = b, found_base = before;
            base += sum;
        }
    }
    // head elements beyond dh: zeros in every stage, never written again
    if (p.c.dh < DHC) {
        for (uint32_t i = lane * 16; i < (uint32_t) (kStages * kStage); i += 512) {
            asm volatile("st.shared.v4.u32 [%0], {%1,%1,%1,%1};" ::"r"(ring + i), "r"(0) : "memory");
        }
    }
    __syncthreads();
    int32_t b = found_b;
    int64_t base = found_base;
    CtaMeta meta{-1, 0, 0, 0};// joined by the second kernel

    while (u < u_end) {
        Seq s = seq_of(p.lens, p.offs, p.rows, b);
        int32_t blocks, tiles;
        extent_of<kRows>(p, s, blocks, tiles);
        const int32_t size = tiles + kItemUnits;// the first kItemUnits units of an item hold no tile
        const int64_t units = (int64_t) blocks * (cl > 0 ? 1 : size) * p.c.heads;
        if (units == 0 || u - base >= units) {// on to the next sequence (u < total: there is one)
            base += units, ++b;
            continue;
        }
        const int64_t item = cl > 0 ? u - base : divide(u - base, size);
        int32_t t0, t1;
        if (cl > 0) {
            t0 = (int32_t) (rank * (uint32_t) tiles / cl), t1 = (int32_t) ((rank + 1) * (uint32_t) tiles / cl);
        } else {
            const int32_t at = (int32_t) (u - base - item * size), n = u_end - u < size - at ? (int32_t) (u_end - u) : size - at;
            t0 = max(0, at - kItemUnits), t1 = max(0, at + n - kItemUnits);
            u += n;
            if (t1 == t0) continue;
        }
        const int32_t kvh = (int32_t) divide(item, blocks), rb = (int32_t) (item - (int64_t) kvh * blocks);
        if (cl > 0) ++u;

        Walk w;
        w.keys = held(s.len, p.t.cap);
        w.k = p.kp + (int64_t) kvh * p.c.k.sh, w.v = p.vp + (int64_t) kvh * p.c.v.sh;
        w.ks = p.ks + (int64_t) kvh * p.c.k.ch, w.vs = p.vs + (int64_t) kvh * p.c.v.ch;
        const int32_t *row_table = p.table + (int64_t) b * p.t.stride;

        // page of this lane's token of a tile (-1: none), read one step ahead of its use
        auto page_of = [&](int32_t tile) -> int32_t {
            const int32_t tok = tile * kTile + (ONE ? 0 : (int32_t) lane);
            if (tile >= t1 || tok >= w.keys) return -1;
            const int32_t id = row_table[p.page_div.div((uint32_t) tok)];
            return id >= 0 && id < p.c.pages ? id : -1;
        };
        // loads of one tile into a stage.  Tokens without a page become zeros; their addresses stay inside the pool.
        auto fetch = [&](uint32_t st, int32_t tile, int32_t page) {
            const uint32_t at = ring + st * kStage, kat = at, vat = at + kTile * DHC, sat = vat + kTile * DHC;
            constexpr int kAtOnce = 32 / kChunks;// rows that the lanes load at a time, 16 bytes each
            const uint32_t c = lane % kChunks, r0 = lane / kChunks;
            const int32_t id = max(page, 0);
            if (ONE) {
                const int32_t first = tile * kTile, in_page = first - (int32_t) p.page_div.div((uint32_t) first) * p.c.page;
                const int32_t count = page < 0 ? 0 : min(kTile, w.keys - first);
                const uint8_t *k = w.k + (int64_t) id * p.c.k.sn + (int64_t) (in_page + (int32_t) r0) * p.c.k.sp + c * 16;
                const uint8_t *v = w.v + (int64_t) id * p.c.v.sn + (int64_t) (in_page + (int32_t) r0) * p.c.v.sp + c * 16;
                if (lane < 2) {
                    const float *s = lane == 0 ? w.ks + (int64_t) id * p.c.k.cn : w.vs + (int64_t) id * p.c.v.cn;
                    cp_async4(sat + lane * 4, s, page >= 0);// no page: scales of 0, log2 -inf
                }
                if (lane == 2) asm volatile("st.shared.u32 [%0], %1;" ::"r"(sat + 8), "r"(count) : "memory");
                if ((int32_t) c * 16 < p.c.dh) {
                    if (count == kTile) {
#pragma unroll
                        for (int i = 0; i < kTile / kAtOnce; ++i) {
                            const uint32_t to = chunk_at<DHC>(r0 + i * kAtOnce, c);
                            cp_async16(kat + to, k, true);
                            cp_async16(vat + to, v, true);
                            k += kAtOnce * p.c.k.sp, v += kAtOnce * p.c.v.sp;
                        }
                    } else {
#pragma unroll 1
                        for (int i = 0; i < kTile / kAtOnce; ++i) {
                            const uint32_t to = chunk_at<DHC>(r0 + i * kAtOnce, c);
                            const bool ok = (int32_t) r0 + i * kAtOnce < count;
                            cp_async16(kat + to, k, ok);
                            cp_async16(vat + to, v, ok);
                            k += kAtOnce * p.c.k.sp, v += kAtOnce * p.c.v.sp;
                        }
                    }
                }
            } else {
                const int32_t tok = tile * kTile + (int32_t) lane;
                const bool valid = page >= 0;
                const int32_t in_page = valid ? tok - (int32_t) p.page_div.div((uint32_t) tok) * p.c.page : 0;
                const int64_t koff = (int64_t) id * p.c.k.sn + (int64_t) in_page * p.c.k.sp;
                const int64_t voff = (int64_t) id * p.c.v.sn + (int64_t) in_page * p.c.v.sp;
                cp_async4(sat + lane * 4, w.ks + (int64_t) id * p.c.k.cn, valid);
                cp_async4(sat + 128 + lane * 4, w.vs + (int64_t) id * p.c.v.cn, valid);
                const uint32_t mask = __ballot_sync(0xffffffffu, valid);
                if (lane == 0) asm volatile("st.shared.u32 [%0], %1;" ::"r"(sat + 256), "r"(mask) : "memory");
                if (p.vec) {
                    const bool has = (int32_t) c * 16 < p.c.dh;
#pragma unroll 4
                    for (int i = 0; i < kTile / kAtOnce; ++i) {
                        const uint32_t r = r0 + i * kAtOnce, to = chunk_at<DHC>(r, c);
                        const int64_t kr = shfl64(koff, (int) r) + c * 16, vr = shfl64(voff, (int) r) + c * 16;
                        const bool ok = (mask >> r) & 1u;
                        if (has) {
                            cp_async16(kat + to, w.k + kr, ok);
                            cp_async16(vat + to, w.v + vr, ok);
                        }
                    }
                } else {
                    // rows that are no whole aligned vectors: a lane copies its token's bytes one by one
#pragma unroll 1
                    for (int32_t d = 0; d < p.c.dh; ++d) {
                        const uint32_t to = chunk_at<DHC>(lane, (uint32_t) d >> 4) + (d & 15);
                        const uint32_t kb = valid ? w.k[koff + d] : 0u, vb = valid ? w.v[voff + d] : 0u;
                        asm volatile("st.shared.u8 [%0], %1;" ::"r"(kat + to), "r"(kb) : "memory");
                        asm volatile("st.shared.u8 [%0], %1;" ::"r"(vat + to), "r"(vb) : "memory");
                    }
                }
            }
        };

        // ---- request q, start the ring, then look at q.  Lane (g, t) holds the elements of row g that its chunks of a key
        // row meet.  Row r of the block is new token (rb * kRows + r) / group, q head kvh * group + (..) % group.
        const int32_t n_rows = min(kRows, s.n * p.group - rb * kRows);
        uint32_t qf[NT][kSteps][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int32_t r = nt * 8 + (int32_t) g;
            const bool have = r < n_rows;
            const uint32_t rr = (uint32_t) rb * kRows + (uint32_t) r;
            const int32_t tok = have ? (int32_t) p.group_div.div(rr) : 0, hd = have ? (int32_t) rr - tok * p.group : 0;
            const uint16_t *q = p.q + (int64_t) (s.first + tok) * p.q_st + (int64_t) (kvh * p.group + hd) * p.q_sh;
#pragma unroll
            for (int h = 0; h < kHalf; ++h) {
                const int32_t d0 = (int32_t) key_chunk<DHC>(t, (uint32_t) h) * 16;
                uint32_t x[8];
                if (have && p.q_vec && d0 + 16 <= p.c.dh) {
                    const uint4 lo = *reinterpret_cast<const uint4 *>(q + d0), hi = *reinterpret_cast<const uint4 *>(q + d0 + 8);
                    x[0] = lo.x, x[1] = lo.y, x[2] = lo.z, x[3] = lo.w, x[4] = hi.x, x[5] = hi.y, x[6] = hi.z, x[7] = hi.w;
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const int32_t d = d0 + 2 * i;
                        const uint32_t a = have && d < p.c.dh ? q[d] : 0u, c = have && d + 1 < p.c.dh ? q[d + 1] : 0u;
                        x[i] = a | (c << 16);
                    }
                }
#pragma unroll
                for (int i = 0; i < 8; ++i) qf[nt][h * 4 + i / 2][i % 2] = x[i];
            }
        }
        int32_t ahead = t0 + (int32_t) warp, page = page_of(ahead);
        __syncwarp();
#pragma unroll 1
        for (int i = 0; i < kStages - 1; ++i) {
            const int32_t next = page_of(ahead + kWarps);
            if (ahead < t1) fetch((uint32_t) i, ahead, page);
            cp_async_commit();
            page = next, ahead += kWarps;
        }
        float factor[NT];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            uint32_t top = 0;
#pragma unroll
            for (int i = 0; i < kSteps; ++i) top = __vmaxu2(top, __vmaxu2(qf[nt][i][0] & 0x7FFF7FFFu, qf[nt][i][1] & 0x7FFF7FFFu));
            top = max(top & 0xFFFFu, top >> 16);
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const int32_t shift = query_shift(p.bf16, top);
            const float up = __uint_as_float(pow2_bits(shift));
            if (p.bf16) {// (fp16 elements go as they are)
#pragma unroll
                for (int i = 0; i < kSteps; ++i) {
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const float2 f = unpack2_t<kBF16>(qf[nt][i][j]);
                        const __half2 v = __floats2half2_rn(f.x * up, f.y * up);
                        qf[nt][i][j] = *reinterpret_cast<const uint32_t *>(&v);
                    }
                }
            }
            factor[nt] = (p.bf16 ? __uint_as_float(pow2_bits(-shift)) : 1.f) * p.scale_log2;
        }
        // scores come as (token g, rows 2t and 2t + 1): the factors and limits of those rows
        float rf[NT][2];
        int32_t limit[NT][2], least = w.keys;// keys that a row sees
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int32_t r = nt * 8 + (int32_t) (2 * t) + i;
                rf[nt][i] = __shfl_sync(0xffffffffu, factor[nt], (int) (2 * t + i) * 4);
                const int32_t pos = s.len - s.n + (int32_t) p.group_div.div((uint32_t) rb * kRows + (uint32_t) r);
                limit[nt][i] = r < n_rows ? max(0, min(pos + 1, w.keys)) : 0;
                if (r < n_rows) least = min(least, limit[nt][i]);
            }
        }
        least = __reduce_min_sync(0xffffffffu, least);

        // ---- the loop over this warp's tiles
        float o[NT][kSteps][4], m[NT][2], wm[NT][2], l[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            m[nt][0] = m[nt][1] = wm[nt][0] = wm[nt][1] = -INFINITY;
            l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
            for (int i = 0; i < kSteps; ++i) o[nt][i][0] = o[nt][i][1] = o[nt][i][2] = o[nt][i][3] = 0.f;
        }
        uint32_t st = 0, st_ahead = kStages - 1;
        for (int32_t tile = t0 + (int32_t) warp; tile < t1; tile += kWarps) {
            const int32_t next = page_of(ahead + kWarps);
            cp_async_wait<kStages - 2>();
            __syncwarp();// every lane's copies have landed, and every lane is done with the stage that is filled next
            if (ahead < t1) fetch(st_ahead, ahead, page);
            cp_async_commit();
            page = next, ahead += kWarps;
            if (++st_ahead == kStages) st_ahead = 0;

            const uint32_t kat = ring + st * kStage, vat = kat + kTile * DHC, sat = vat + kTile * DHC;
            if (++st == kStages) st = 0;
            // q . k
            float x[2][NT][4];
#pragma unroll
            for (int sub = 0; sub < 2; ++sub) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) x[sub][nt][0] = x[sub][nt][1] = x[sub][nt][2] = x[sub][nt][3] = 0.f;
            }
#pragma unroll
            for (int h = 0; h < kHalf; ++h) {
#pragma unroll
                for (int sub = 0; sub < 2; ++sub) {
                    const uint32_t c = key_chunk<DHC>(t, (uint32_t) h);
                    const uint4 lo = lds128(kat + chunk_at<DHC>(sub * 16 + g, c)), hi = lds128(kat + chunk_at<DHC>(sub * 16 + 8 + g, c));
                    const uint32_t a[4] = {lo.x, lo.y, lo.z, lo.w}, e[4] = {hi.x, hi.y, hi.z, hi.w};
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        uint32_t a0, a1, a2, a3;
                        e4m3x4_to_f16x4(a[i], a0, a2), e4m3x4_to_f16x4(e[i], a1, a3);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) mma_f16(x[sub][nt], a0, a1, a2, a3, qf[nt][h * 4 + i][0], qf[nt][h * 4 + i][1]);
                    }
                }
            }
            // scores in powers of two, masked; lv: log2 of the values' scales of tokens g, g + 8, g + 16, g + 24
            float lv[4];
            uint32_t mask;
            if (ONE) {
                const float ks = lds_f32(sat);
                lv[0] = lv[1] = lv[2] = lv[3] = log2_of(lds_f32(sat + 4));
                const uint32_t count = lds_u32(sat + 8);
                mask = count >= 32 ? 0xFFFFFFFFu : (1u << count) - 1u;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    const float f0 = ks * rf[nt][0], f1 = ks * rf[nt][1];
#pragma unroll
                    for (int i = 0; i < 4; ++i) x[i >> 1][nt][(i & 1) * 2] *= f0, x[i >> 1][nt][(i & 1) * 2 + 1] *= f1;
                }
            } else {
                mask = lds_u32(sat + 256);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float ks = lds_f32(sat + (i * 8 + g) * 4);
                    lv[i] = log2_of(lds_f32(sat + 128 + (i * 8 + g) * 4));
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        x[i >> 1][nt][(i & 1) * 2] *= ks * rf[nt][0];
                        x[i >> 1][nt][(i & 1) * 2 + 1] *= ks * rf[nt][1];
                    }
                }
            }
            if (mask != 0xFFFFFFFFu || tile * kTile + kTile > least) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int32_t tok = tile * kTile + i * 8 + (int32_t) g;
                    const bool ok = (mask >> (i * 8 + g)) & 1u;
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        if (!ok || tok >= limit[nt][0]) x[i >> 1][nt][(i & 1) * 2] = -INFINITY;
                        if (!ok || tok >= limit[nt][1]) x[i >> 1][nt][(i & 1) * 2 + 1] = -INFINITY;
                    }
                    if (!ONE && !ok) lv[i] = 0.f;
                }
            }
            // references: moved when a score or a weight exceeds its own by more than the slack
            bool over = false;
            float top[NT][2], wtop[NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float a0 = x[0][nt][i], a1 = x[0][nt][2 + i], a2 = x[1][nt][i], a3 = x[1][nt][2 + i];
                    top[nt][i] = fmaxf(fmaxf(a0, a1), fmaxf(a2, a3));
                    wtop[nt][i] = ONE ? top[nt][i] + lv[0] : fmaxf(fmaxf(a0 + lv[0], a1 + lv[1]), fmaxf(a2 + lv[2], a3 + lv[3]));
                    over = over || top[nt][i] > m[nt][i] + kSlack || wtop[nt][i] > wm[nt][i] + kSlack;
                }
            }
            if (__any_sync(0xffffffffu, over)) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
#pragma unroll
                        for (int d = 4; d < 32; d <<= 1) {
                            top[nt][i] = fmaxf(top[nt][i], __shfl_xor_sync(0xffffffffu, top[nt][i], d));
                            if (!ONE) wtop[nt][i] = fmaxf(wtop[nt][i], __shfl_xor_sync(0xffffffffu, wtop[nt][i], d));
                        }
                        if (ONE) wtop[nt][i] = top[nt][i] + lv[0];
                        if (top[nt][i] > m[nt][i] + kSlack) {
                            l[nt][i] *= fast_exp2(m[nt][i] - top[nt][i]);// from -inf: 0
                            m[nt][i] = top[nt][i];
                        }
                        if (wtop[nt][i] > wm[nt][i] + kSlack) {
                            const float f = fast_exp2(wm[nt][i] - wtop[nt][i]);
#pragma unroll
                            for (int j = 0; j < kSteps; ++j) o[nt][j][i] *= f, o[nt][j][2 + i] *= f;
                            wm[nt][i] = wtop[nt][i];
                        }
                    }
                }
            }
            // p to its sum, w in fp16 as operand B of p . v
            uint32_t bw[2][NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                // rows that have seen nothing yet: their scores are all -inf, any finite reference gives 0
                const float m0 = m[nt][0] == -INFINITY ? 0.f : m[nt][0], m1 = m[nt][1] == -INFINITY ? 0.f : m[nt][1];
                float w0 = wm[nt][0] == -INFINITY ? 0.f : wm[nt][0] - kLift, w1 = wm[nt][1] == -INFINITY ? 0.f : wm[nt][1] - kLift;
                if (ONE) w0 -= lv[0], w1 -= lv[0];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float a = x[i >> 1][nt][(i & 1) * 2], c = x[i >> 1][nt][(i & 1) * 2 + 1];
                    l[nt][0] += fast_exp2(a - m0), l[nt][1] += fast_exp2(c - m1);
                    const __half2 h = ONE ? __floats2half2_rn(fast_exp2(a - w0), fast_exp2(c - w1)) : __floats2half2_rn(fast_exp2(a - w0 + lv[i]), fast_exp2(c - w1 + lv[i]));
                    bw[i >> 1][nt][i & 1] = transpose8x8(*reinterpret_cast<const uint32_t *>(&h));
                }
            }
            // p . v: lane (g, t) holds DHC / 8 consecutive head elements of tokens 2t, 2t + 1, 2t + 8, 2t + 9
#pragma unroll
            for (int sub = 0; sub < 2; ++sub) {
                constexpr int kWords = DHC / 32;
                uint32_t v[4][kWords];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t r = sub * 16 + 2 * t + (i & 1) + (i >> 1) * 8;
                    if (DHC == 64) {
                        const uint2 a = lds64(vat + chunk_at<DHC>(r, g >> 1) + (g & 1) * 8);
                        v[i][0] = a.x, v[i][1] = a.y;
                    } else {
#pragma unroll
                        for (int c = 0; c < kWords / 4; ++c) {
                            const uint4 a = lds128(vat + chunk_at<DHC>(r, g * (kWords / 4) + c));
                            v[i][c * 4] = a.x, v[i][c * 4 + 1] = a.y, v[i][c * 4 + 2] = a.z, v[i][c * 4 + 3] = a.w;
                        }
                    }
                }
#pragma unroll
                for (int i = 0; i < kWords; ++i) {
                    // bytes of two tokens side by side: (a0 b0 a1 b1) and (a2 b2 a3 b3)
                    const uint32_t e0 = __byte_perm(v[0][i], v[1][i], 0x5140), e1 = __byte_perm(v[0][i], v[1][i], 0x7362);
                    const uint32_t f0 = __byte_perm(v[2][i], v[3][i], 0x5140), f1 = __byte_perm(v[2][i], v[3][i], 0x7362);
                    uint32_t a0, a1, a2, a3, c0, c1, c2, c3;
                    e4m3x4_to_f16x4(e0, a0, a1), e4m3x4_to_f16x4(f0, a2, a3), e4m3x4_to_f16x4(e1, c0, c1), e4m3x4_to_f16x4(f1, c2, c3);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        mma_f16(o[nt][2 * i], a0, a1, a2, a3, bw[sub][nt][0], bw[sub][nt][1]);
                        mma_f16(o[nt][2 * i + 1], c0, c1, c2, c3, bw[sub][nt][0], bw[sub][nt][1]);
                    }
                }
            }
        }

        // ---- the warps' results meet in shared memory: [warp][row][DHC] and the rows' references
        cp_async_wait<0>();
        __syncthreads();
        float *so = reinterpret_cast<float *>(smem);
        PartHead *sh = reinterpret_cast<PartHead *>(so + kWarps * kRows * DHC);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int r = nt * 8 + 2 * (int) t + i;
                float sum = l[nt][i];
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
                if (g == 0) sh[warp * kRows + r] = PartHead{m[nt][i], sum, wm[nt][i], limit[nt][i]};
                // elements g * DHC / 8 .. of this row; 16-byte groups rotated by the row, so that the four rows of a
                // store spread over the banks
                float *dst = so + (warp * kRows + r) * DHC;
#pragma unroll
                for (int j = 0; j < kSteps; j += 2) {
                    const uint32_t grp = g * (DHC / 32) + j / 2;
                    *reinterpret_cast<float4 *>(dst + ((grp ^ (uint32_t) (r & 7)) << 2)) = make_float4(o[nt][j][i], o[nt][j][2 + i], o[nt][j + 1][i], o[nt][j + 1][2 + i]);
                }
            }
        }
        __syncthreads();
        const bool whole = cl > 0 ? cl == 1 : t0 == 0 && t1 == tiles;
        const int part = t0 > 0 ? 0 : 1;
        float *po = reinterpret_cast<float *>(sh + kWarps * kRows);// this CTA's part, for its cluster
        PartHead *ph = reinterpret_cast<PartHead *>(po + kRows * DHC);
        const int64_t slot0 = ((int64_t) blockIdx.x * 2 + part) * kRows;
        for (int r = (int) warp; r < n_rows; r += kWarps) {
            float mr = -INFINITY, wr = -INFINITY, lr = 0.f, f[kWarps];
#pragma unroll
            for (int i = 0; i < kWarps; ++i) mr = fmaxf(mr, sh[i * kRows + r].m), wr = fmaxf(wr, sh[i * kRows + r].w);
            const float m0 = mr == -INFINITY ? 0.f : mr;// (warps without a reference: their l is 0 or NaN)
#pragma unroll
            for (int i = 0; i < kWarps; ++i) {
                const PartHead h = sh[i * kRows + r];
                lr += h.l * fast_exp2(h.m - m0);
                f[i] = h.w == -INFINITY ? 0.f : fast_exp2(h.w - wr);
            }
            uint16_t *out = row_of_out(p, s, kvh, (uint32_t) rb * kRows + (uint32_t) r);
            if (!whole && lane == 0) (cl > 0 ? ph[r] : dp.heads[slot0 + r]) = PartHead{mr, lr, wr - kLift, sh[r].keys};
#pragma unroll
            for (int j = 0; j < (DHC + 127) / 128; ++j) {
                const uint32_t grp = lane + 32 * j;
                if (DHC == 64 && grp >= 16) break;
                float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int i = 0; i < kWarps; ++i) {
                    const float4 a = *reinterpret_cast<const float4 *>(so + (i * kRows + r) * DHC + ((grp ^ (uint32_t) (r & 7)) << 2));
                    if (f[i] != 0.f) y.x += f[i] * a.x, y.y += f[i] * a.y, y.z += f[i] * a.z, y.w += f[i] * a.w;
                }
                if (whole) store_out(p, out, (int32_t) grp * 4, y, out_factors(p, b, sh[r].keys, lr, wr - kLift - mr));
                else *reinterpret_cast<float4 *>(cl > 0 ? po + r * DHC + grp * 4 : dp.parts + (slot0 + r) * DHC + grp * 4) = y;
            }
        }
        if (cl > 1) {
            // the CTAs of the cluster meet: each adds the parts of its share of the rows, in the order of the tiles
            cluster_sync_all();
            const uint32_t po_at = (uint32_t) __cvta_generic_to_shared(po), ph_at = (uint32_t) __cvta_generic_to_shared(ph);
            for (int r = (int) (rank + cl * warp); r < n_rows; r += (int) (cl * kWarps)) {
                float mr = -INFINITY, wr = -INFINITY, lr = 0.f;
                PartHead h[kMaxCluster];
#pragma unroll
                for (uint32_t i = 0; i < kMaxCluster; ++i) {
                    h[i] = PartHead{-INFINITY, 0.f, -INFINITY, 0};
                    if (i < cl) {
                        const float4 v = tc::ld_cluster_f4(tc::mapa_u32(ph_at + (uint32_t) r * 16u, i));
                        h[i] = PartHead{v.x, v.y, v.z, __float_as_int(v.w)};
                    }
                    mr = fmaxf(mr, h[i].m), wr = fmaxf(wr, h[i].w);
                }
#pragma unroll
                for (uint32_t i = 0; i < kMaxCluster; ++i) lr += h[i].l * fast_exp2(h[i].m - (mr == -INFINITY ? 0.f : mr));
                uint16_t *out = row_of_out(p, s, kvh, (uint32_t) rb * kRows + (uint32_t) r);
#pragma unroll
                for (int j = 0; j < (DHC + 127) / 128; ++j) {
                    const uint32_t grp = lane + 32 * j;
                    if (DHC == 64 && grp >= 16) break;
                    float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                    for (uint32_t i = 0; i < kMaxCluster; ++i) {
                        if (i < cl && h[i].w != -INFINITY) {
                            const float f = fast_exp2(h[i].w - wr);
                            const float4 a = tc::ld_cluster_f4(tc::mapa_u32(po_at + ((uint32_t) r * DHC + grp * 4) * 4u, i));
                            y.x += f * a.x, y.y += f * a.y, y.z += f * a.z, y.w += f * a.w;
                        }
                    }
                    store_out(p, out, (int32_t) grp * 4, y, out_factors(p, b, sh[r].keys, lr, wr - mr));
                }
            }
            cluster_sync_all();// nobody leaves while its part may still be read
            return;
        }
        if (!whole && part == 1) {
            meta.b = b, meta.kvh = kvh, meta.rb = rb;
            meta.last = (int32_t) divide(base + (item + 1) * size - 1, each);
        }
        if (u < u_end) {
            __syncthreads();// the ring is loaded again
            if (p.c.dh < DHC) {// .. and the zeros beyond dh were written over
                for (uint32_t i = lane * 16; i < (uint32_t) (kStages * kStage); i += 512) {
                    asm volatile("st.shared.v4.u32 [%0], {%1,%1,%1,%1};" ::"r"(ring + i), "r"(0) : "memory");
                }
                __syncwarp();
            }
        }
    }
    if (cl > 0) return;
    asm volatile("griddepcontrol.launch_dependents;");
    if (threadIdx.x == 0) dp.meta[blockIdx.x] = meta;
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
    int dhc;      // head size rounded up to 64, 128 or 256
    int block;    // query rows per item: 8 or 16 (mma.sync), 128 or 256 (tcgen05)
    uint32_t ctas;
    uint32_t cluster;// CTAs that share an item over distributed shared memory; 0: equal stretches, joined by a second kernel
};

uint64_t workspace_of_desc(const AttendDesc &d) { return d.cluster > 0 ? 0 : split_bytes(d.ctas, (uint64_t) d.block, (uint64_t) d.dhc); }

// Whether the tcgen05 kernel takes a call with rows_each query rows per sequence and kv head, from what both cost in ns
// x SMs if every sequence fills its table.  Measured over 1 and 16 sequences of 2000 to 30000 tokens and 2 to 64 new ones:
// this kernel takes 130, 270 or 600 ns for 16 rows and 32 cached tokens at a head size of 64, 128 or 256, the other one
// 950, 950 or 1250 ns for a block of rows and 64 cached tokens and 6 us more to start and end.  32 heads on 8 of 128
// elements, 16 sequences of 8000 tokens: 8 new tokens 122 us here and 130 us there, 16 new tokens 220 us and 132 us; one
// sequence of 2000 tokens: 12 new ones 15 us and 21 us, 64 new ones 33 us and 28 us.
bool prefill_is_faster(const AttendDesc &d, int64_t rows_each) {
    if (rows_each <= 16 || d.t.batch > kPrefillMaxBatch) return false;
    const auto cost = [&](int64_t block, int64_t keys, int64_t each) {
        return (double) d.t.batch * (double) d.c.heads * (double) ((rows_each + block - 1) / block) * (double) (((int64_t) d.t.cap + keys - 1) / keys) * (double) each;
    };
    return cost(16, kTile, d.dhc == 64 ? 130 : d.dhc == 128 ? 270 : 600) > cost(prefill_rows(d.dhc), kPrefillKeys, d.dhc == 256 ? 1250 : 950) + 6000. * d.sm_count;
}

template<int DHC, int NT, bool ONE>
cudaError_t launch_decode_as(const AttendDesc &d, const AttendParams &a, void *workspace, cudaStream_t st) {
    constexpr int kSmem = smem_bytes(DHC, NT);
    static_assert((kWarps + 1) * 8 * NT * (DHC * 4 + (int) sizeof(PartHead)) <= kSmem, "the warps' results and their sum fit the rings");
    static_assert(stage_bytes(DHC) % 16 == 0, "stages start on 16 bytes");
    SplitParams dp = split_params(a, workspace, d.ctas, 8 * NT, DHC);
    dp.cluster = d.cluster;
    // more shared memory than the default: asked for once per device (again, where two threads come first)
    static std::atomic<uint64_t> ready{0};
    const uint64_t bit = d.device_id < 64 ? 1ull << d.device_id : 0;
    cudaError_t e = cudaSuccess;
    if ((ready.load(std::memory_order_relaxed) & bit) == 0) {
        e = cudaFuncSetAttribute(decode_kernel<DHC, NT, ONE>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
        if (e != cudaSuccess) return e;
        ready.fetch_or(bit, std::memory_order_relaxed);
    }
    if (d.cluster > 0) return launch_cluster_smem(decode_kernel<DHC, NT, ONE>, d.ctas, kThreads, d.cluster, kSmem, st, dp);
    decode_kernel<DHC, NT, ONE><<<d.ctas, kThreads, kSmem, st>>>(dp);
    e = cudaGetLastError();
    if (e != cudaSuccess || d.ctas == 1) return e;
    return launch_join<DHC, 8 * NT>(dp, d.ctas, st);
}
template<int DHC, int NT>
cudaError_t launch_decode(const AttendDesc &d, const AttendParams &a, void *workspace, cudaStream_t st) {
    return a.vec && a.c.page % kTile == 0 ? launch_decode_as<DHC, NT, true>(d, a, workspace, st) : launch_decode_as<DHC, NT, false>(d, a, workspace, st);
}

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
    d.dhc = d.c.dh <= 64 ? 64 : d.c.dh <= 128 ? 128 : 256;
    const int64_t group = d.q_heads / d.c.heads;
    if ((int64_t) d.rows * group > 0x7FFFFFFF) return STATUS_BAD_TENSOR_SHAPE;
    // query rows per sequence on average (only the device knows each one's)
    const int64_t rows_each = d.t.batch > 0 ? (int64_t) d.rows * group / d.t.batch : 0;
    const bool prefill = prefill_is_faster(d, rows_each);
    d.block = prefill ? prefill_rows(d.dhc) : rows_each > 8 ? 16 : 8;
    // every CTA that fits the GPU at once, but no more than there can be units for
    const int64_t blocks = ((int64_t) d.rows * group + d.block - 1) / d.block + d.t.batch, keys = prefill ? kPrefillKeys : kTile;
    const int64_t tiles = std::max<int64_t>(1, ((int64_t) d.t.cap + keys - 1) / keys);
    const int64_t places = (int64_t) d.sm_count * (prefill ? 1 : ctas_per_sm(d.dhc, d.block / 8));
    d.ctas = (uint32_t) places;
    if (blocks * d.c.heads < places * kMinUnits) {
        d.ctas = (uint32_t) std::max<int64_t>(1, std::min(places, (blocks * d.c.heads * tiles + kMinUnits - 1) / kMinUnits));
    }
    // Few items over a table of few columns: a cluster of CTAs per item, one launch.  A CTA of four warps takes up to
    // kClusterRounds tiles per warp; beyond that equal stretches over all SMs are faster although they take a second launch.
    // (One query over 777 tokens: 8.3 us with clusters, 10.3 us with stretches, which a table with room for 32768 takes.)
    d.cluster = 0;
    if (!prefill) {
        const int64_t exact = d.t.offsets ? blocks : (int64_t) d.t.batch * ((group + d.block - 1) / d.block);
        const int64_t items = exact * d.c.heads;
        uint32_t c = 1;
        while (c < kMaxCluster && items * c * 2 <= places && tiles > (int64_t) c * kWarps) c *= 2;
        if (items <= places && tiles <= (int64_t) c * kWarps * kClusterRounds) d.cluster = c, d.ctas = (uint32_t) (items * c);
    }
    auto *r = new (std::nothrow) AttendDesc(d);
    if (r == nullptr) return STATUS_MEMORY_NOT_ALLOCATED;
    *desc_ptr = reinterpret_cast<infiniopPagedAttentionDescriptor_t>(r);
    return STATUS_SUCCESS;
}

INFINIOP_API infiniopStatus_t infiniopGetPagedAttentionWorkspaceSize(infiniopPagedAttentionDescriptor_t desc, uint64_t *size) {
    if (desc == nullptr || desc->device != DevNvGpu) return STATUS_BAD_DEVICE;
    if (size == nullptr) return STATUS_BAD_PARAM;
    *size = workspace_of_desc(*reinterpret_cast<AttendDesc *>(desc));
    return STATUS_SUCCESS;
}

INFINIOP_API infiniopStatus_t infiniopPagedAttention(infiniopPagedAttentionDescriptor_t desc, void *workspace,
                                                     uint64_t workspace_size, void *out, void const *q, void const *k_pages,
                                                     void const *v_pages, void const *k_scales, void const *v_scales,
                                                     void const *block_table, void const *seq_lens, void const *q_offsets,
                                                     void *stream) {
    if (desc == nullptr || desc->device != DevNvGpu) return STATUS_BAD_DEVICE;
    auto *d = reinterpret_cast<AttendDesc *>(desc);
    if (d->rows == 0 || d->t.batch == 0) return STATUS_SUCCESS;
    if (out == nullptr || q == nullptr || seq_lens == nullptr || d->t.offsets != (q_offsets != nullptr)) return STATUS_BAD_PARAM;
    // a table without columns or a pool without pages has no keys: every token gets zeros
    const bool empty = d->t.cols == 0 || d->c.pages == 0;
    if (!empty && (k_pages == nullptr || v_pages == nullptr || k_scales == nullptr || v_scales == nullptr || block_table == nullptr)) return STATUS_BAD_PARAM;
    const uint64_t need = workspace_of_desc(*d);
    if (need > 0 && (workspace == nullptr || workspace_size < need)) return STATUS_MEMORY_NOT_ALLOCATED;
    if ((need > 0 && !aligned16(workspace)) || !aligned_to(2, {out, q}) || !aligned_to(4, {k_scales, v_scales, block_table, seq_lens, q_offsets})) {
        return STATUS_BAD_PARAM;
    }
    DeviceGuard guard(d->device_id);
    AttendParams p{};
    p.out = reinterpret_cast<uint16_t *>(out), p.q = reinterpret_cast<const uint16_t *>(q);
    p.o_st = d->o_st, p.o_sh = d->o_sh, p.q_st = d->q_st, p.q_sh = d->q_sh;
    p.kp = reinterpret_cast<const uint8_t *>(k_pages), p.vp = reinterpret_cast<const uint8_t *>(v_pages);
    p.ks = reinterpret_cast<const float *>(k_scales), p.vs = reinterpret_cast<const float *>(v_scales);
    p.table = reinterpret_cast<const int32_t *>(block_table), p.lens = reinterpret_cast<const int32_t *>(seq_lens);
    p.offs = reinterpret_cast<const int32_t *>(q_offsets);
    p.rows = d->rows, p.group = d->q_heads / d->c.heads;
    p.scale_log2 = (float) ((double) d->scale * 1.4426950408889634);
    p.page_div = FastDiv((uint32_t) d->c.page), p.group_div = FastDiv((uint32_t) p.group);
    p.c = d->c, p.t = d->t, p.bf16 = d->bf16;
    if (empty) p.t.cap = 0;
    // whole 16-byte vectors: rows of codes, rows of q; 8-byte pieces of out's rows
    p.vec = d->c.dh % 16 == 0 && aligned16(k_pages) && aligned16(v_pages);
    for (int64_t s : {d->c.k.sn, d->c.k.sh, d->c.k.sp, d->c.v.sn, d->c.v.sh, d->c.v.sp}) p.vec = p.vec && s % 16 == 0;
    p.q_vec = aligned16(q) && d->q_st % 8 == 0 && d->q_sh % 8 == 0;
    p.o_vec = (uintptr_t) out % 8 == 0 && d->o_st % 4 == 0 && d->o_sh % 4 == 0 && d->c.dh % 4 == 0;
    p.o_vec8 = aligned16(out) && d->o_st % 8 == 0 && d->o_sh % 8 == 0 && d->c.dh % 8 == 0;
    auto st = reinterpret_cast<cudaStream_t>(stream);
    cudaError_t e;
    if (d->block >= 128) {
        e = launch_prefill(p, workspace, d->dhc, d->ctas, d->device_id, st);
    } else {
        const bool few = d->block == 8;
        if (d->dhc == 64) e = few ? launch_decode<64, 1>(*d, p, workspace, st) : launch_decode<64, 2>(*d, p, workspace, st);
        else if (d->dhc == 128) e = few ? launch_decode<128, 1>(*d, p, workspace, st) : launch_decode<128, 2>(*d, p, workspace, st);
        else e = few ? launch_decode<256, 1>(*d, p, workspace, st) : launch_decode<256, 2>(*d, p, workspace, st);
    }
    if (e != cudaSuccess) {
        cudaGetLastError();
        fprintf(stderr, "infiniop[b200]: paged attention launch failed: %s\n", cudaGetErrorString(e));
        return STATUS_EXECUTION_FAILED;
    }
    return check_launch("paged attention");
}

INFINIOP_API infiniopStatus_t infiniopDestroyPagedAttentionDescriptor(infiniopPagedAttentionDescriptor_t desc) {
    if (desc == nullptr || desc->device != DevNvGpu) return STATUS_BAD_DEVICE;
    delete reinterpret_cast<AttendDesc *>(desc);
    return STATUS_SUCCESS;
}
