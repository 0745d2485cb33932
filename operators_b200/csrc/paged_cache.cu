// The paged 8-bit KV cache: appending tokens, copying pages, freeing and compacting.  Attention over it is in
// paged_attention.cu.  No counterpart in the reference, whose cache is one fp16 tensor per sequence that its attention
// composite writes with rearrange (src/ops/attention/operator.cc:87-91).
//
// Append.  A block (page x kv head, K and V apart) has one scale s, a power of two:
//     s = max(s_old if rows of the page are kept, 2^x, 2^-40),  x = min { x : max|x_new| <= 448 * 2^x }
//     code = e4m3(x_new / s),  kept codes: e4m3(code * s_old / s)
// e4m3 carries its own exponent, so a power of two costs no precision against an exact 448 / max (the step relative to
// the value is the same in every binade), division by it is exact, and when the scale of a half-filled page grows the
// kept codes only move in their exponent: nothing is lost but bits of codes that become subnormal, however often it
// happens.  One CTA owns the K and the V block of a page and head (the page is looked up once, and both blocks' loads are
// under way together): it reads the new rows once into registers, takes the maxima, and writes codes.  256 threads, 128 where
// every sequence has one new token.  Prompts of 9000 tokens in all, 8 heads of 128 elements: 16.5 us, 3.3 TB/s of what it reads
// and writes; the conversions keep the issue slots 65 % busy, and the first loads wait for the search of the page.
//
// Copy and compact move whole pages; compact first finds the live pages (one cluster, a bitmap in the workspace).  Bound by
// memory: 700 pairs of pages of 8 heads, 64 tokens, 128 elements 30.7 us, 6.0 TB/s; 1024 moved pages of that size 59.8 us, of
// which the plan takes 9.
#include "paged_cache.cuh"

#include <new>

using namespace b200;
using namespace b200::paged;

namespace {

// ------------------------------------------------------------------------------------------------------- append --

struct AppendParams {
    const uint16_t *k, *v;
    int64_t k_st, k_sh, v_st, v_sh;// strides of token and head
    uint8_t *kp, *vp;
    float *ks, *vs;
    const int32_t *table, *lens, *offs;
    int32_t rows;
    FastDiv per_row, page_div;// by the vectors of a row and by the page size
    CacheShape c;
    TableShape t;
};

constexpr int kAppendThreads = 256;
constexpr int kHeld = 4;// vectors of new elements that a thread keeps between the maximum and the encoding

// Exclusive sum over the CTA; `total` = sum over all threads.  `slot`: 33 words of shared memory.
__device__ __forceinline__ int32_t cta_exclusive_sum(int32_t v, int32_t *slot, int32_t &total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    int32_t incl = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int32_t u = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += u;
    }
    __syncthreads();
    if (lane == 31) slot[warp] = incl;
    __syncthreads();
    int32_t before = 0, all = 0;
    for (int w = 0; w < warps; ++w) {
        if (w < warp) before += slot[w];
        all += slot[w];
    }
    total = all;
    return before + incl - v;
}

// VEC new elements of one row at a time: 8 (16-byte loads, 8-byte stores of codes) or 1.
template<bool BF, int VEC>
__global__ void __launch_bounds__(kAppendThreads) append_kernel(const AppendParams p) {
    __shared__ uint32_t wmax[2][kAppendThreads / 32];
    const int32_t item = (int32_t) blockIdx.x, head = (int32_t) blockIdx.y;
    const int32_t P = p.c.page, D = p.c.dh, lane = (int32_t) (threadIdx.x & 31);

    const auto page_of = [&](int32_t token) -> int32_t { return (int32_t) p.page_div.div((uint32_t) token); };
    // the item-th touched page of the call: sequence b, its nth page.  Every warp looks for it by itself (no barrier ahead
    // of the loads), a sequence per lane, four where there are many.
    int32_t b = item, nth = 0;// one token, one page per sequence
    if (p.offs == nullptr) {
        if (b >= p.t.batch) return;
    } else {
        const int32_t each = p.t.batch <= 32 ? 1 : 4;
        int32_t base = 0;
        bool hit = false;
        for (int32_t b0 = 0; b0 < p.t.batch && !hit; b0 += 32 * each) {
            int32_t count[4], mine = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int32_t x = b0 + lane * each + i;
                count[i] = 0;
                if (i < each && x < p.t.batch) {
                    int32_t lo, hi;
                    written(seq_of(p.lens, p.offs, p.rows, x), p.t.cap, lo, hi);
                    count[i] = pages_touched(lo, hi, page_of);
                }
                mine += count[i];
            }
            int32_t incl = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int32_t u = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= o) incl += u;
            }
            const int32_t before = base + incl - mine;
            const uint32_t who = __ballot_sync(0xffffffffu, item >= before && item - before < mine);
            if (who != 0) {
                int32_t f = 0, k = item - before;
#pragma unroll
                for (int i = 0; i < 3; ++i) {
                    if (f == i && k >= count[i]) k -= count[i], f = i + 1;
                }
                const int src = __ffs((int) who) - 1;
                b = b0 + src * each + __shfl_sync(0xffffffffu, f, src), nth = __shfl_sync(0xffffffffu, k, src);
                hit = true;
            }
            base += __shfl_sync(0xffffffffu, incl, 31);
        }
        if (!hit) return;
    }
    const Seq s = seq_of(p.lens, p.offs, p.rows, b);
    int32_t lo, hi;
    written(s, p.t.cap, lo, hi);
    if (hi <= lo) return;
    const int32_t col = page_of(lo) + nth, page0 = col * P;
    const int32_t p0 = lo > page0 ? lo : page0, p1 = hi - page0 < P ? hi : page0 + P;
    const int32_t page = p.table[(int64_t) b * p.t.stride + col];// (looked at once the new rows are on their way)
    const int32_t kept = p0 - page0, m = p1 - p0;

    const int64_t row0 = s.first + (p0 - (s.len - s.n));
    const uint16_t *x[2] = {p.k + row0 * p.k_st + (int64_t) head * p.k_sh, p.v + row0 * p.v_st + (int64_t) head * p.v_sh};
    const int64_t x_st[2] = {p.k_st, p.v_st};

    // the new rows: into registers, and their largest magnitudes.  (A block has fewer than 2^31 elements.)
    const uint32_t per_row = (uint32_t) (D / VEC), nv = (uint32_t) m * per_row, step = blockDim.x;
    uint4 held_v[2][kHeld];
    auto load = [&](int side, uint32_t i) -> uint4 {
        const uint32_t r = p.per_row.div(i);
        const uint16_t *src = x[side] + (int64_t) r * x_st[side] + (i - r * per_row) * VEC;
        if (VEC == 8) return *reinterpret_cast<const uint4 *>(src);
        return make_uint4(*src, 0u, 0u, 0u);
    };
    uint32_t top[2] = {0u, 0u};
    auto grow = [&](int side, uint4 w) {
        top[side] = abs_max2<BF>(top[side], w.x);
        if (VEC == 8) top[side] = abs_max2<BF>(abs_max2<BF>(abs_max2<BF>(top[side], w.y), w.z), w.w);
    };
#pragma unroll
    for (int j = 0; j < kHeld; ++j) {
        const uint32_t i = threadIdx.x + (uint32_t) j * step;
#pragma unroll
        for (int side = 0; side < 2; ++side) held_v[side][j] = i < nv ? load(side, i) : make_uint4(0u, 0u, 0u, 0u);
    }
    if (page < 0 || page >= p.c.pages) return;
    uint8_t *codes[2] = {p.kp + (int64_t) page * p.c.k.sn + (int64_t) head * p.c.k.sh, p.vp + (int64_t) page * p.c.v.sn + (int64_t) head * p.c.v.sh};
    const int64_t sp[2] = {p.c.k.sp, p.c.v.sp};
    float *scale[2] = {p.ks + (int64_t) page * p.c.k.cn + (int64_t) head * p.c.k.ch, p.vs + (int64_t) page * p.c.v.cn + (int64_t) head * p.c.v.ch};
    const float old[2] = {kept > 0 ? *scale[0] : 0.f, kept > 0 ? *scale[1] : 0.f};
#pragma unroll
    for (int side = 0; side < 2; ++side) {
#pragma unroll
        for (int j = 0; j < kHeld; ++j) grow(side, held_v[side][j]);
        for (uint32_t i = threadIdx.x + kHeld * step; i < nv; i += step) grow(side, load(side, i));
    }
    const uint32_t kInf = BF ? 0x7F80u : 0x7C00u;
    auto block_max = [&]() {// patterns of one sign are ordered like their values
#pragma unroll
        for (int side = 0; side < 2; ++side) {
            const uint32_t t = __reduce_max_sync(0xffffffffu, max(top[side] & 0xFFFFu, top[side] >> 16));
            if (lane == 0) wmax[side][threadIdx.x >> 5] = t;
        }
        __syncthreads();
        const uint32_t w = (uint32_t) lane < step / 32 ? (uint32_t) lane : 0u;
#pragma unroll
        for (int side = 0; side < 2; ++side) top[side] = __reduce_max_sync(0xffffffffu, wmax[side][w]);
    };
    block_max();
    if (max(top[0], top[1]) >= kInf) {
        // an infinity (NaN is passed over by the maximum): once more, finite elements only
        __syncthreads();
#pragma unroll
        for (int side = 0; side < 2; ++side) {
            uint32_t t = 0;
            for (uint32_t i = threadIdx.x; i < nv; i += step) {
                const uint4 w = load(side, i);
                t = __vmaxu2(t, finite_abs2<BF>(w.x));
                if (VEC == 8) t = __vmaxu2(__vmaxu2(t, finite_abs2<BF>(w.y)), __vmaxu2(finite_abs2<BF>(w.z), finite_abs2<BF>(w.w)));
            }
            top[side] = t;
        }
        block_max();
    }
#pragma unroll
    for (int side = 0; side < 2; ++side) {
        const float amax = BF ? __uint_as_float(top[side] << 16) : f16_to_f32((uint16_t) top[side]);
        const float fresh = __uint_as_float(pow2_bits(scale_exponent(__float_as_uint(amax)))), now = fmaxf(old[side], fresh);

        // rows that stay, where the scale has grown
        if (kept > 0 && now != old[side]) {
            const float ratio = old[side] / now;
            const uint32_t n = (uint32_t) kept * per_row;
            for (uint32_t i = threadIdx.x; i < n; i += step) {
                const uint32_t r = p.per_row.div(i);
                uint8_t *at = codes[side] + (int64_t) r * sp[side] + (i - r * per_row) * VEC;
                if (VEC == 8) {
                    uint2 w = *reinterpret_cast<uint2 *>(at);
                    uint32_t out[2] = {w.x, w.y};
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const float2 a = unpack2(e4m3x2_to_f16x2((uint16_t) out[j])), c = unpack2(e4m3x2_to_f16x2((uint16_t) (out[j] >> 16)));
                        out[j] = (uint32_t) f32x2_to_e4m3x2(a.x * ratio, a.y * ratio) | ((uint32_t) f32x2_to_e4m3x2(c.x * ratio, c.y * ratio) << 16);
                    }
                    *reinterpret_cast<uint2 *>(at) = make_uint2(out[0], out[1]);
                } else {
                    const float2 a = unpack2(e4m3x2_to_f16x2((uint16_t) *at));
                    *at = (uint8_t) f32x2_to_e4m3x2(a.x * ratio, 0.f);
                }
            }
        }
        // the new rows
        uint8_t *first = codes[side] + (int64_t) kept * sp[side];
        auto store = [&](uint32_t i, uint4 w, auto code2) {// `code2`: two elements to two codes
            const uint32_t r = p.per_row.div(i);
            uint8_t *at = first + (int64_t) r * sp[side] + (i - r * per_row) * VEC;
            if (VEC == 8) *reinterpret_cast<uint2 *>(at) = make_uint2(code2(w.x) | (code2(w.y) << 16), code2(w.z) | (code2(w.w) << 16));
            else *at = (uint8_t) code2(w.x);
        };
        if ((__float_as_uint(now) & 0x7FFFFFu) == 0) {
            const float inv = 1.f / now;// exact, and so are the products
            auto code2 = [&](uint32_t w) -> uint32_t {
                const float2 f = f16or_bf16x2<BF>(w);
                return f32x2_to_e4m3x2(f.x * inv, f.y * inv);
            };
#pragma unroll
            for (int j = 0; j < kHeld; ++j) {
                const uint32_t i = threadIdx.x + (uint32_t) j * step;
                if (i < nv) store(i, held_v[side][j], code2);
            }
            for (uint32_t i = threadIdx.x + kHeld * step; i < nv; i += step) store(i, load(side, i), code2);
        } else {// an old scale that is no power of two
            for (uint32_t i = threadIdx.x; i < nv; i += step) {
                store(i, load(side, i), [&](uint32_t w) -> uint32_t {
                    const float2 f = f16or_bf16x2<BF>(w);
                    return f32x2_to_e4m3x2(f.x / now, f.y / now);
                });
            }
        }
        if (threadIdx.x == 0) *scale[side] = now;// (every read of the old scale lies before the barrier)
    }
}

struct AppendDesc {
    Device device;
    int device_id;
    CacheShape c;
    TableShape t;
    int32_t rows;
    bool bf16;
    int64_t k_st, k_sh, v_st, v_sh;
};

// ------------------------------------------------------------------------------------------------ copying pages --

// A page of one pool as runs of consecutive bytes: `runs` = n0 x n1 of them, `len` bytes each.
struct PageRuns {
    int64_t page, s0, s1, cn, ch;// strides: page, runs (n1 fastest), scales
    int32_t n0, n1, len;
};
struct MoveParams {
    uint8_t *kp, *vp;
    float *ks, *vs;
    PageRuns k, v;
    int32_t pages, heads;
    int64_t k_pieces, v_pieces;// of a page
};

constexpr int kMoveThreads = 256;

PageRuns page_runs(const CacheShape &c, const PoolStrides &s) {
    PageRuns r{s.sn, s.sh, s.sp, s.cn, s.ch, c.heads, c.page, c.dh};
    if (r.n0 > 1 && r.n1 > 1 && r.s0 < r.s1) std::swap(r.s0, r.s1), std::swap(r.n0, r.n1);// the smaller stride inside
    if (r.n1 == 1) std::swap(r.s0, r.s1), std::swap(r.n0, r.n1);
    for (int i = 0; i < 2 && r.n1 > 1 && r.s1 == r.len && (int64_t) r.n1 * r.len < ((int64_t) 1 << 31); ++i) {
        r.len *= r.n1;// the runs of the inner dimension follow each other
        r.n1 = r.n0, r.s1 = r.s0, r.n0 = 1, r.s0 = 0;
    }
    return r;
}
// Widest unit (bytes) that every run can be moved in.
int run_unit(const PageRuns &r, const void *base) {
    uint64_t all = (uint64_t) (uintptr_t) base | (uint64_t) r.len | 16u;
    if (r.n0 > 1) all |= (uint64_t) r.s0;
    if (r.n1 > 1) all |= (uint64_t) r.s1;
    all |= (uint64_t) r.page;
    return (all & 15u) == 0 ? 16 : (all & 3u) == 0 ? 4 : 1;
}

// Units [begin, begin + 4 * threads) of one page of one pool, and with the first of them the page's scales.  ONE: a page
// is one run of bytes.
template<typename U, bool ONE>
__device__ __forceinline__ void move_piece(uint8_t *pool, float *scales, const PageRuns &r, int32_t heads, int64_t src, int64_t dst, int64_t begin) {
    const int64_t per_run = r.len / (int32_t) sizeof(U), units = ONE ? per_run : per_run * r.n1 * r.n0;
    const uint8_t *from = pool + src * r.page;
    uint8_t *to = pool + dst * r.page;
    U v[4];
    int64_t at[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int64_t u = begin + threadIdx.x + (int64_t) j * kMoveThreads;
        at[j] = -1;
        if (u < units) {
            if (ONE) {
                at[j] = u * (int64_t) sizeof(U);
            } else {
                const int64_t run = divide(u, per_run), outer = divide(run, r.n1);
                at[j] = outer * r.s0 + (run - outer * r.n1) * r.s1 + (u - run * per_run) * (int64_t) sizeof(U);
            }
            v[j] = *reinterpret_cast<const U *>(from + at[j]);
        }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if (at[j] >= 0) *reinterpret_cast<U *>(to + at[j]) = v[j];
    }
    if (begin == 0) {
        for (int32_t h = threadIdx.x; h < heads; h += kMoveThreads) scales[dst * r.cn + h * r.ch] = scales[src * r.cn + h * r.ch];
    }
}
template<typename U>
int64_t pieces_of(const PageRuns &r) {
    const int64_t units = (int64_t) (r.len / (int32_t) sizeof(U)) * r.n1 * r.n0;
    return (units + 4 * kMoveThreads - 1) / (4 * kMoveThreads);
}
bool one_run(const MoveParams &m) { return m.k.n0 * m.k.n1 == 1 && m.v.n0 * m.v.n1 == 1; }

// A block moves 16 KB (U 16 bytes): piece blockIdx.x of pool blockIdx.y of the pairs blockIdx.z ..
template<typename U, bool ONE>
__global__ void __launch_bounds__(kMoveThreads) copy_pairs_kernel(const MoveParams p, const int32_t *pairs, int64_t stride, int64_t count) {
    const bool is_v = blockIdx.y != 0;
    for (int64_t i = blockIdx.z; i < count; i += gridDim.z) {
        const int32_t src = pairs[i * stride], dst = pairs[i * stride + 1];
        if (src < 0 || src >= p.pages || dst < 0 || dst >= p.pages || src == dst) continue;
        for (int64_t piece = blockIdx.x; piece < (is_v ? p.v_pieces : p.k_pieces); piece += gridDim.x) {
            move_piece<U, ONE>(is_v ? p.vp : p.kp, is_v ? p.vs : p.ks, is_v ? p.v : p.k, p.heads, src, dst, piece * 4 * kMoveThreads);
        }
    }
}

struct CopyDesc {
    Device device;
    int device_id, sm_count;
    CacheShape c;
    int64_t count, stride;
};

MoveParams move_params(const CacheShape &c, void *kp, void *vp, void *ks, void *vs) {
    return MoveParams{reinterpret_cast<uint8_t *>(kp), reinterpret_cast<uint8_t *>(vp), reinterpret_cast<float *>(ks),
                      reinterpret_cast<float *>(vs), page_runs(c, c.k), page_runs(c, c.v), c.pages, c.heads, 0, 0};
}

// ---------------------------------------------------------------------------------------------------- compacting --

constexpr uint32_t kPlanCtas = 8, kPlanThreads = 1024;

// Workspace: header, bitmap of live pages, sources and destinations of the moves.
struct PlanHeader {
    int32_t live, moves, pad[2];
};
struct PlanView {
    PlanHeader *head;
    uint32_t *bits;
    int32_t *src, *dst;
};
uint64_t plan_words(uint64_t pages) { return (pages + 31) / 32; }
uint64_t plan_bytes(uint64_t pages) { return sizeof(PlanHeader) + 4 * ((plan_words(pages) + 3) / 4 * 4) + 8 * (pages / 2 + 1); }
PlanView plan_view(void *ws, uint64_t pages) {
    PlanView v;
    v.head = reinterpret_cast<PlanHeader *>(ws);
    v.bits = reinterpret_cast<uint32_t *>(v.head + 1);
    v.src = reinterpret_cast<int32_t *>(v.bits + (plan_words(pages) + 3) / 4 * 4);
    v.dst = v.src + (pages / 2 + 1);
    return v;
}

struct CompactParams {
    const int32_t *table, *lens;
    int32_t *new_table, *page_map, *live;
    int64_t new_stride;
    TableShape t;
    int32_t pages, page;
    PlanView plan;
};

// One cluster finds the live pages and the moves.
__global__ void __launch_bounds__(kPlanThreads) compact_plan_kernel(const CompactParams p) {
    __shared__ int32_t slot[33];
    __shared__ int32_t below;// live pages below the count
    const int32_t words = (p.pages + 31) / 32;
    const uint32_t rank = cluster_rank(), gtid = rank * kPlanThreads + threadIdx.x;
    for (int32_t w = (int32_t) gtid; w < words; w += (int32_t) (kPlanCtas * kPlanThreads)) p.plan.bits[w] = 0;
    cluster_sync_all();
    // marks: the warps of the cluster share out the rows, several warps to a row where rows are few
    {
        const int32_t warps = kPlanCtas * kPlanThreads / 32, warp = (int32_t) (gtid / 32), lane = (int32_t) (gtid & 31);
        const int32_t per_row = p.t.batch >= warps ? 1 : warps / (p.t.batch > 0 ? p.t.batch : 1);
        for (int64_t u = warp; u < (int64_t) p.t.batch * per_row; u += warps) {
            const int32_t b = (int32_t) (u / per_row), part = (int32_t) (u % per_row);
            const int32_t len = held(p.lens[b] > 0 ? p.lens[b] : 0, p.t.cap), used = len > 0 ? (len - 1) / p.page + 1 : 0;
            const int32_t *row = p.table + (int64_t) b * p.t.stride;
            for (int64_t i = (int64_t) part * 32 + lane; i < used; i += (int64_t) per_row * 32) {
                const int32_t id = row[i];
                if (id >= 0 && id < p.pages) atomicOr(&p.plan.bits[id >> 5], 1u << (id & 31));
            }
        }
    }
    cluster_sync_all();
    if (rank != 0) return;
    // ranks of live pages and holes: a stretch of words per thread
    const int32_t each = (words + (int32_t) kPlanThreads - 1) / (int32_t) kPlanThreads;
    const int32_t w0 = min((int32_t) threadIdx.x * each, words), w1 = min(w0 + each, words);
    int32_t mine = 0;
    for (int32_t w = w0; w < w1; ++w) mine += __popc(p.plan.bits[w]);
    int32_t live;
    const int32_t before = cta_exclusive_sum(mine, slot, live);
    if (threadIdx.x == 0) below = 0;
    __syncthreads();
    int32_t seen = before;
    for (int32_t w = w0; w < w1; ++w) {
        const uint32_t bits = p.plan.bits[w];
        if (live / 32 == w) below = seen + __popc(bits & ((1u << (live & 31)) - 1u));
        seen += __popc(bits);
    }
    if (threadIdx.x == 0 && live / 32 >= words) below = live;// every page is live and the last word is full
    __syncthreads();
    seen = before;
    for (int32_t w = w0; w < w1; ++w) {
        const uint32_t bits = p.plan.bits[w];
        // holes: dead pages below `live`; the j-th of them has j dead ones before it
        uint32_t holes = ~bits;
        if ((w + 1) * 32 > live) holes &= live > w * 32 ? (1u << (live - w * 32)) - 1u : 0u;
        while (holes != 0) {
            const int32_t i = __ffs((int) holes) - 1;
            holes &= holes - 1;
            p.plan.dst[w * 32 + i - (seen + __popc(bits & ((1u << i) - 1u)))] = w * 32 + i;
        }
        uint32_t movers = bits;
        if (w * 32 < live) movers &= live - w * 32 >= 32 ? 0u : ~((1u << (live - w * 32)) - 1u);
        while (movers != 0) {
            const int32_t i = __ffs((int) movers) - 1;
            movers &= movers - 1;
            p.plan.src[seen + __popc(bits & ((1u << i) - 1u)) - below] = w * 32 + i;
        }
        seen += __popc(bits);
    }
    __syncthreads();
    const int32_t moves = live - below;
    for (int32_t j = (int32_t) threadIdx.x; j < moves; j += (int32_t) kPlanThreads) p.page_map[p.plan.src[j]] = p.plan.dst[j];
    if (threadIdx.x == 0) {
        p.plan.head->live = live, p.plan.head->moves = moves;
        *p.live = live;
    }
}

// Renames the table's entries, fills the map and moves the pages.  Sources lie at or above the live count,
// destinations below it, so no page is both.
template<typename U, bool ONE>
__global__ void __launch_bounds__(kMoveThreads, 5) compact_apply_kernel(const CompactParams p, const MoveParams m) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int32_t live = p.plan.head->live;
    const int64_t moves = p.plan.head->moves;
    const int64_t gtid = (int64_t) blockIdx.x * kMoveThreads + threadIdx.x, threads = (int64_t) gridDim.x * kMoveThreads;
    for (int64_t i = gtid; i < p.pages; i += threads) {
        const bool is_live = (p.plan.bits[i >> 5] >> (i & 31)) & 1u;
        if (!is_live) p.page_map[i] = -1;
        else if (i < live) p.page_map[i] = (int32_t) i;
    }
    for (int64_t i = gtid; i < (int64_t) p.t.batch * p.t.cols; i += threads) {
        const int32_t b = (int32_t) (i / p.t.cols), col = (int32_t) (i - (int64_t) b * p.t.cols);
        const int32_t len = held(p.lens[b] > 0 ? p.lens[b] : 0, p.t.cap);
        int32_t id = p.table[(int64_t) b * p.t.stride + col];
        if ((int64_t) col * p.page < len && id >= live && id < p.pages) id = p.page_map[id];// a mover: written by the plan
        p.new_table[(int64_t) b * p.new_stride + col] = id;
    }
    const int64_t each = m.k_pieces + m.v_pieces;
    for (int64_t w = blockIdx.x; w < moves * each; w += gridDim.x) {
        const int64_t i = divide(w, each), rest = w - i * each;
        const bool is_v = rest >= m.k_pieces;
        move_piece<U, ONE>(is_v ? m.vp : m.kp, is_v ? m.vs : m.ks, is_v ? m.v : m.k, m.heads, p.plan.src[i], p.plan.dst[i],
                           (is_v ? rest - m.k_pieces : rest) * 4 * kMoveThreads);
    }
}

struct CompactDesc {
    Device device;
    int device_id, sm_count;
    CacheShape c;
    TableShape t;
    int64_t new_stride;
};

}// namespace

// ------------------------------------------------------------------------------------------------- entry points --

INFINIOP_API infiniopStatus_t infiniopCreatePagedCacheAppendDescriptor(
    infiniopHandle_t handle, infiniopPagedCacheAppendDescriptor_t *desc_ptr, infiniopTensorDescriptor_t k_desc,
    infiniopTensorDescriptor_t v_desc, infiniopTensorDescriptor_t k_pages_desc, infiniopTensorDescriptor_t v_pages_desc,
    infiniopTensorDescriptor_t k_scales_desc, infiniopTensorDescriptor_t v_scales_desc,
    infiniopTensorDescriptor_t block_table_desc, infiniopTensorDescriptor_t seq_lens_desc,
    infiniopTensorDescriptor_t q_offsets_desc) {
    if (handle == nullptr || handle->device != DevNvGpu) return STATUS_BAD_DEVICE;
    if (desc_ptr == nullptr) return STATUS_MEMORY_NOT_ALLOCATED;
    if (k_desc == nullptr || v_desc == nullptr) return STATUS_BAD_PARAM;
    AppendDesc d{};
    infiniopStatus_t st = check_cache(k_pages_desc, v_pages_desc, k_scales_desc, v_scales_desc, d.c);
    if (st != STATUS_SUCCESS) return st;
    st = check_tables(block_table_desc, seq_lens_desc, q_offsets_desc, d.c.page, d.t);
    if (st != STATUS_SUCCESS) return st;
    if (k_desc->ndim != 3) return STATUS_BAD_TENSOR_SHAPE;
    const uint64_t rows = k_desc->shape[0];
    for (auto *x : {k_desc, v_desc}) {
        st = check_rows(x, rows, (uint64_t) d.c.heads, (uint64_t) d.c.dh, k_desc->dt);
        if (st != STATUS_SUCCESS) return st;
    }
    if (!d.t.offsets && rows != (uint64_t) d.t.batch) return STATUS_BAD_TENSOR_SHAPE;
    auto *h = reinterpret_cast<Handle *>(handle);
    d.device = DevNvGpu, d.device_id = h->device_id, d.rows = (int32_t) rows, d.bf16 = dt_eq(k_desc->dt, BF16);
    d.k_st = k_desc->strides[0], d.k_sh = k_desc->strides[1], d.v_st = v_desc->strides[0], d.v_sh = v_desc->strides[1];
    auto *r = new (std::nothrow) AppendDesc(d);
    if (r == nullptr) return STATUS_MEMORY_NOT_ALLOCATED;
    *desc_ptr = reinterpret_cast<infiniopPagedCacheAppendDescriptor_t>(r);
    return STATUS_SUCCESS;
}

INFINIOP_API infiniopStatus_t infiniopGetPagedCacheAppendWorkspaceSize(infiniopPagedCacheAppendDescriptor_t desc, uint64_t *size) {
    if (desc == nullptr || desc->device != DevNvGpu) return STATUS_BAD_DEVICE;
    if (size == nullptr) return STATUS_BAD_PARAM;
    *size = 0;
    return STATUS_SUCCESS;
}

INFINIOP_API infiniopStatus_t infiniopPagedCacheAppend(infiniopPagedCacheAppendDescriptor_t desc, void *workspace,
                                                       uint64_t workspace_size, void const *k, void const *v, void *k_pages,
                                                       void *v_pages, void *k_scales, void *v_scales,
                                                       void const *block_table, void const *seq_lens, void const *q_offsets,
                                                       void *stream) {
    (void) workspace;
    (void) workspace_size;
    if (desc == nullptr || desc->device != DevNvGpu) return STATUS_BAD_DEVICE;
    auto *d = reinterpret_cast<AppendDesc *>(desc);
    if (d->rows == 0 || d->t.batch == 0 || d->t.cols == 0 || d->c.pages == 0) return STATUS_SUCCESS;
    if (k == nullptr || v == nullptr || k_pages == nullptr || v_pages == nullptr || k_scales == nullptr || v_scales == nullptr ||
        block_table == nullptr || seq_lens == nullptr || d->t.offsets != (q_offsets != nullptr)) {
        return STATUS_BAD_PARAM;
    }
    if (!aligned_to(2, {k, v}) || !aligned_to(4, {k_scales, v_scales, block_table, seq_lens, q_offsets})) return STATUS_BAD_PARAM;
    DeviceGuard guard(d->device_id);
    AppendParams p{reinterpret_cast<const uint16_t *>(k), reinterpret_cast<const uint16_t *>(v), d->k_st, d->k_sh, d->v_st, d->v_sh,
                   reinterpret_cast<uint8_t *>(k_pages), reinterpret_cast<uint8_t *>(v_pages), reinterpret_cast<float *>(k_scales),
                   reinterpret_cast<float *>(v_scales), reinterpret_cast<const int32_t *>(block_table),
                   reinterpret_cast<const int32_t *>(seq_lens), reinterpret_cast<const int32_t *>(q_offsets), d->rows, FastDiv(1), FastDiv((uint32_t) d->c.page), d->c, d->t};
    // 8 elements at a time where every row of the new tokens starts on 16 bytes and every row of codes on 8
    bool vec = d->c.dh % 8 == 0 && aligned16(k) && aligned16(v) && ((uintptr_t) k_pages | (uintptr_t) v_pages) % 8 == 0;
    for (int64_t s : {d->k_st, d->k_sh, d->v_st, d->v_sh, d->c.k.sn, d->c.k.sh, d->c.k.sp, d->c.v.sn, d->c.v.sh, d->c.v.sp}) vec = vec && s % 8 == 0;
    p.per_row = FastDiv((uint32_t) (vec ? d->c.dh / 8 : d->c.dh));
    const int64_t items = d->t.offsets ? pages_bound(d->rows, d->t.batch, d->c.page) : d->rows;
    const dim3 grid((unsigned) items, (unsigned) d->c.heads);
    // one token per sequence is 16 vectors of 8: a small block leaves the SM to more of them
    const unsigned threads = d->t.offsets ? kAppendThreads : 128;
    auto st = reinterpret_cast<cudaStream_t>(stream);
    if (d->bf16) {
        if (vec) append_kernel<true, 8><<<grid, threads, 0, st>>>(p);
        else append_kernel<true, 1><<<grid, threads, 0, st>>>(p);
    } else {
        if (vec) append_kernel<false, 8><<<grid, threads, 0, st>>>(p);
        else append_kernel<false, 1><<<grid, threads, 0, st>>>(p);
    }
    return check_launch("paged cache append");
}

INFINIOP_API infiniopStatus_t infiniopDestroyPagedCacheAppendDescriptor(infiniopPagedCacheAppendDescriptor_t desc) {
    if (desc == nullptr || desc->device != DevNvGpu) return STATUS_BAD_DEVICE;
    delete reinterpret_cast<AppendDesc *>(desc);
    return STATUS_SUCCESS;
}

INFINIOP_API infiniopStatus_t infiniopCreatePagedCacheCopyDescriptor(
    infiniopHandle_t handle, infiniopPagedCacheCopyDescriptor_t *desc_ptr, infiniopTensorDescriptor_t k_pages_desc,
    infiniopTensorDescriptor_t v_pages_desc, infiniopTensorDescriptor_t k_scales_desc, infiniopTensorDescriptor_t v_scales_desc,
    infiniopTensorDescriptor_t pairs_desc) {
    if (handle == nullptr || handle->device != DevNvGpu) return STATUS_BAD_DEVICE;
    if (desc_ptr == nullptr) return STATUS_MEMORY_NOT_ALLOCATED;
    if (pairs_desc == nullptr) return STATUS_BAD_PARAM;
    CopyDesc d{};
    const infiniopStatus_t st = check_cache(k_pages_desc, v_pages_desc, k_scales_desc, v_scales_desc, d.c);
    if (st != STATUS_SUCCESS) return st;
    if (pairs_desc->ndim != 2 || pairs_desc->shape[1] != 2 || pairs_desc->shape[0] > 0x7FFFFFFFull) return STATUS_BAD_TENSOR_SHAPE;
    if (!dt_eq(pairs_desc->dt, I32)) return STATUS_BAD_TENSOR_DTYPE;
    if (!unit_rows(pairs_desc)) return STATUS_BAD_TENSOR_STRIDES;
    auto *h = reinterpret_cast<Handle *>(handle);
    d.device = DevNvGpu, d.device_id = h->device_id, d.sm_count = h->sm_count;
    d.count = (int64_t) pairs_desc->shape[0], d.stride = pairs_desc->strides[0];
    auto *r = new (std::nothrow) CopyDesc(d);
    if (r == nullptr) return STATUS_MEMORY_NOT_ALLOCATED;
    *desc_ptr = reinterpret_cast<infiniopPagedCacheCopyDescriptor_t>(r);
    return STATUS_SUCCESS;
}

INFINIOP_API infiniopStatus_t infiniopGetPagedCacheCopyWorkspaceSize(infiniopPagedCacheCopyDescriptor_t desc, uint64_t *size) {
    if (desc == nullptr || desc->device != DevNvGpu) return STATUS_BAD_DEVICE;
    if (size == nullptr) return STATUS_BAD_PARAM;
    *size = 0;
    return STATUS_SUCCESS;
}

INFINIOP_API infiniopStatus_t infiniopPagedCacheCopy(infiniopPagedCacheCopyDescriptor_t desc, void *workspace, uint64_t workspace_size,
                                                     void *k_pages, void *v_pages, void *k_scales, void *v_scales,
                                                     void const *pairs, void *stream) {
    (void) workspace;
    (void) workspace_size;
    if (desc == nullptr || desc->device != DevNvGpu) return STATUS_BAD_DEVICE;
    auto *d = reinterpret_cast<CopyDesc *>(desc);
    if (d->count == 0 || d->c.pages == 0) return STATUS_SUCCESS;
    if (k_pages == nullptr || v_pages == nullptr || k_scales == nullptr || v_scales == nullptr || pairs == nullptr) return STATUS_BAD_PARAM;
    if (!aligned_to(4, {k_scales, v_scales, pairs})) return STATUS_BAD_PARAM;
    DeviceGuard guard(d->device_id);
    MoveParams m = move_params(d->c, k_pages, v_pages, k_scales, v_scales);
    const int unit = std::min(run_unit(m.k, k_pages), run_unit(m.v, v_pages));
    auto st = reinterpret_cast<cudaStream_t>(stream);
    const auto *list = reinterpret_cast<const int32_t *>(pairs);
    auto run = [&](auto u, auto *whole, auto *runs) {
        using U = decltype(u);
        m.k_pieces = pieces_of<U>(m.k), m.v_pieces = pieces_of<U>(m.v);
        const dim3 grid((unsigned) std::min<int64_t>(std::max(m.k_pieces, m.v_pieces), 1 << 20), 2, (unsigned) std::min<int64_t>(d->count, 65535));
        if (one_run(m)) whole<<<grid, kMoveThreads, 0, st>>>(m, list, d->stride, d->count);
        else runs<<<grid, kMoveThreads, 0, st>>>(m, list, d->stride, d->count);
    };
    if (unit == 16) run(uint4{}, copy_pairs_kernel<uint4, true>, copy_pairs_kernel<uint4, false>);
    else if (unit == 4) run(uint32_t{}, copy_pairs_kernel<uint32_t, true>, copy_pairs_kernel<uint32_t, false>);
    else run(uint8_t{}, copy_pairs_kernel<uint8_t, true>, copy_pairs_kernel<uint8_t, false>);
    return check_launch("paged cache copy");
}

INFINIOP_API infiniopStatus_t infiniopDestroyPagedCacheCopyDescriptor(infiniopPagedCacheCopyDescriptor_t desc) {
    if (desc == nullptr || desc->device != DevNvGpu) return STATUS_BAD_DEVICE;
    delete reinterpret_cast<CopyDesc *>(desc);
    return STATUS_SUCCESS;
}

INFINIOP_API infiniopStatus_t infiniopCreatePagedCacheCompactDescriptor(
    infiniopHandle_t handle, infiniopPagedCacheCompactDescriptor_t *desc_ptr, infiniopTensorDescriptor_t k_pages_desc,
    infiniopTensorDescriptor_t v_pages_desc, infiniopTensorDescriptor_t k_scales_desc, infiniopTensorDescriptor_t v_scales_desc,
    infiniopTensorDescriptor_t new_table_desc, infiniopTensorDescriptor_t block_table_desc, infiniopTensorDescriptor_t seq_lens_desc,
    infiniopTensorDescriptor_t page_map_desc, infiniopTensorDescriptor_t live_desc) {
    if (handle == nullptr || handle->device != DevNvGpu) return STATUS_BAD_DEVICE;
    if (desc_ptr == nullptr) return STATUS_MEMORY_NOT_ALLOCATED;
    if (new_table_desc == nullptr || page_map_desc == nullptr || live_desc == nullptr) return STATUS_BAD_PARAM;
    CompactDesc d{};
    infiniopStatus_t st = check_cache(k_pages_desc, v_pages_desc, k_scales_desc, v_scales_desc, d.c);
    if (st != STATUS_SUCCESS) return st;
    st = check_tables(block_table_desc, seq_lens_desc, nullptr, d.c.page, d.t);
    if (st != STATUS_SUCCESS) return st;
    if (new_table_desc->ndim != 2 || page_map_desc->ndim != 1 || live_desc->ndim != 1) return STATUS_BAD_TENSOR_SHAPE;
    if (new_table_desc->shape[0] != (uint64_t) d.t.batch || new_table_desc->shape[1] != (uint64_t) d.t.cols ||
        page_map_desc->shape[0] != (uint64_t) d.c.pages || live_desc->shape[0] != 1 || d.c.pages > (1 << 27)) {
        return STATUS_BAD_TENSOR_SHAPE;
    }
    for (auto *x : {new_table_desc, page_map_desc, live_desc}) {
        if (!dt_eq(x->dt, I32)) return STATUS_BAD_TENSOR_DTYPE;
    }
    for (auto *x : {new_table_desc, page_map_desc, live_desc}) {
        if (!unit_rows(x) || !disjoint(x)) return STATUS_BAD_TENSOR_STRIDES;
    }
    auto *h = reinterpret_cast<Handle *>(handle);
    d.device = DevNvGpu, d.device_id = h->device_id, d.sm_count = h->sm_count, d.new_stride = new_table_desc->strides[0];
    auto *r = new (std::nothrow) CompactDesc(d);
    if (r == nullptr) return STATUS_MEMORY_NOT_ALLOCATED;
    *desc_ptr = reinterpret_cast<infiniopPagedCacheCompactDescriptor_t>(r);
    return STATUS_SUCCESS;
}

INFINIOP_API infiniopStatus_t infiniopGetPagedCacheCompactWorkspaceSize(infiniopPagedCacheCompactDescriptor_t desc, uint64_t *size) {
    if (desc == nullptr || desc->device != DevNvGpu) return STATUS_BAD_DEVICE;
    if (size == nullptr) return STATUS_BAD_PARAM;
    *size = plan_bytes((uint64_t) reinterpret_cast<CompactDesc *>(desc)->c.pages);
    return STATUS_SUCCESS;
}

INFINIOP_API infiniopStatus_t infiniopPagedCacheCompact(infiniopPagedCacheCompactDescriptor_t desc, void *workspace,
                                                        uint64_t workspace_size, void *k_pages, void *v_pages, void *k_scales,
                                                        void *v_scales, void *new_table, void const *block_table,
                                                        void const *seq_lens, void *page_map, void *live, void *stream) {
    if (desc == nullptr || desc->device != DevNvGpu) return STATUS_BAD_DEVICE;
    auto *d = reinterpret_cast<CompactDesc *>(desc);
    const bool no_pages = d->c.pages == 0, no_rows = d->t.batch == 0 || d->t.cols == 0;
    if (live == nullptr) return STATUS_BAD_PARAM;
    if (!no_pages && (k_pages == nullptr || v_pages == nullptr || k_scales == nullptr || v_scales == nullptr || page_map == nullptr)) return STATUS_BAD_PARAM;
    if (!no_rows && (new_table == nullptr || block_table == nullptr || seq_lens == nullptr)) return STATUS_BAD_PARAM;
    if (workspace == nullptr || workspace_size < plan_bytes((uint64_t) d->c.pages)) return STATUS_MEMORY_NOT_ALLOCATED;
    if (!aligned16(workspace) || !aligned_to(4, {k_scales, v_scales, new_table, block_table, seq_lens, page_map, live})) return STATUS_BAD_PARAM;
    DeviceGuard guard(d->device_id);
    auto st = reinterpret_cast<cudaStream_t>(stream);
    CompactParams p{};
    p.table = reinterpret_cast<const int32_t *>(block_table), p.lens = reinterpret_cast<const int32_t *>(seq_lens);
    p.new_table = reinterpret_cast<int32_t *>(new_table), p.page_map = reinterpret_cast<int32_t *>(page_map);
    p.live = reinterpret_cast<int32_t *>(live);
    p.new_stride = d->new_stride, p.t = d->t, p.pages = d->c.pages, p.page = d->c.page;
    if (no_rows) p.t.batch = 0;
    p.plan = plan_view(workspace, (uint64_t) d->c.pages);
    if (launch_cluster(compact_plan_kernel, kPlanCtas, kPlanThreads, kPlanCtas, st, p) != cudaSuccess) return check_launch("paged cache compact (plan)");
    MoveParams m = move_params(d->c, k_pages, v_pages, k_scales, v_scales);
    const int unit = std::min(run_unit(m.k, k_pages), run_unit(m.v, v_pages));
    auto run = [&](auto u, auto *whole, auto *runs) {
        using U = decltype(u);
        m.k_pieces = pieces_of<U>(m.k), m.v_pieces = pieces_of<U>(m.v);
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned) d->sm_count * 5);
        cfg.blockDim = dim3(kMoveThreads);
        cfg.stream = st;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = attr, cfg.numAttrs = 1;
        return one_run(m) ? cudaLaunchKernelEx(&cfg, whole, p, m) : cudaLaunchKernelEx(&cfg, runs, p, m);
    };
    const cudaError_t e = unit == 16 ? run(uint4{}, compact_apply_kernel<uint4, true>, compact_apply_kernel<uint4, false>)
        : unit == 4                 ? run(uint32_t{}, compact_apply_kernel<uint32_t, true>, compact_apply_kernel<uint32_t, false>)
                                    : run(uint8_t{}, compact_apply_kernel<uint8_t, true>, compact_apply_kernel<uint8_t, false>);
    (void) e;// reported by the check below
    return check_launch("paged cache compact");
}

INFINIOP_API infiniopStatus_t infiniopDestroyPagedCacheCompactDescriptor(infiniopPagedCacheCompactDescriptor_t desc) {
    if (desc == nullptr || desc->device != DevNvGpu) return STATUS_BAD_DEVICE;
    delete reinterpret_cast<CompactDesc *>(desc);
    return STATUS_SUCCESS;
}
