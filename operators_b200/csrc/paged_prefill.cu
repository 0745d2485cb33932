// Attention over the paged 8-bit KV cache for prompts, chunks of prompts and long drafts: tcgen05.
//
// A block is 128 query rows (new tokens x the q heads that share a kv head, row = token * group + head), one TMEM lane
// each; a tile is 64 cached tokens.  Per tile: S = q k^T into TMEM, weights in fp16 back into TMEM over S (operand A of
// the second product), O += W v in TMEM.  The operands of kind::f16 are fp16: q is scaled per row by a power of two
// (see paged_attention.cu), the codes become fp16 exactly on their way into shared memory, once per pair of blocks.
//
// Softmax in one pass: p = 2^(s f - m) with f the row's and the page's factor and m the row's reference, at first the largest
// score of its first tile.  The weight of a value is w = p * 2^c with 2^c = 2^(m - M + 2) * (scale of the values' page) and M
// the weights' own reference.  No tile is looked through for its largest score: sums of 16 weights, formed anyway, tell when a
// weight may have grown beyond fp16.  Then M follows by the power of two that brings the tile's largest weight back to
// [2^2, 2^3), and the tile's weights (still in fp32 in registers) and O are divided by it, exactly.  (Looking for the maximum
// and forming the weights anew took 187 us where this takes 162, in heads whose scores spread widely.)  m is no part of that:
// weights also grow with the scales of the values' pages, which the sum of p must not follow.  m moves to the tile's largest
// score, and M to its largest weight, where the tile would add more than 2^64 to the sum or weights pass 2^100.  fp16
// holds weights down to 2^-16 of the reference with all their bits, smaller ones to 2^-27 of it.  One exponential gives w;
// the sum of p takes the tile's sum of w times 2^-c.  c is kept above -90: such weights are zero in fp16 either way (p < 2^64),
// and their sum must not underflow.
//
// What bounds it: per tile and block 64 x 128 exponentials (16 a cycle and SM: 512 cycles) stand against 2 x 64 x 128 x dh
// multiply-adds (at dh 128: 256 cycles at full rate; S with its 64 columns runs at two thirds of it, 640 in all).  One CTA per SM
// works on two blocks at a time (head sizes beyond 128: one), so that one's exponentials run beside the other's products and
// both share the converted tiles.  Measured: 2000 cycles per pair of blocks and tile, of which the tensor pipe is busy 1280
// and the exponentials 1024; the softmax warps' chain (S from TMEM, exponentials, weights to TMEM, barriers) is what is left.
//
// Roles (512 threads; 384 with one block): a warpgroup per block for softmax and epilogue, a thread per row; two warps
// convert the codes of K, two those of V (their loads run a tile ahead in registers); of the last warpgroup one warp allocates
// TMEM and issues the products (the warp as one, see umma_f16_ss).  Shared memory: q of this item and (head sizes up to 128)
// of the next, copied and made ready while this one is worked on (160 -> 150 us for a chunk, 170 -> 152 us for prompts); two
// tiles of K, two of V (128-byte swizzled rows as TMA would lay them).  S is double-buffered: S of tile j + 1 is issued before
// W v of tile j.
//
// Work is divided into equal stretches as in paged_attention.cu; an item is a pair of blocks, stops where its last row's
// mask begins, and counts kItemUnits tiles more for what its start and end cost.  All roles walk the stretch's items by
// themselves.
//
// A product's completion is waited for only where O is touched, so it has a barrier for even and one for odd tiles: a row
// that has seen S of tile n knows that W v of tile n - 2 (issued before it) is done, not that of tile n - 1, and one
// barrier's parity could not tell the two apart.
// Every wait is bounded: a role that gives up raises the CTA's abort flag, all roles leave, and TMEM and shared memory are
// given back when the products and copies that were under way have ended.
//
// 512 new tokens over 16384 cached ones, 32 heads on 8 of 128 elements, bf16: 152 to 157 us on different GPUs, 920 to 890
// TFLOP/s.  Two prompts of up to 4096 tokens, nothing cached before them, fp16: 149 to 154 us, 700 to 680 TFLOP/s of the
// visible products.
#include "paged_attention.cuh"
#include "tc_ptx.cuh"

#include <atomic>

namespace b200 {
namespace paged {

namespace {

using namespace tc;

constexpr int kRows = 128, kKeys = kPrefillKeys;
constexpr float kSlack = 13.f, kLift = 2.f;// kSlack: of the general form, w <= 2^15 there
constexpr float kLeast = -90.f;
constexpr long long kDrainTicks = 2000000;// about a millisecond; a tile's products take a microsecond
constexpr float kMostWeight = 65504.f, kFarWeight = 0x1p100f;// sums of 16 weights that fp16 or fp32 may not hold
constexpr float kFarGain = 0x1p64f;// what a tile may add to a row's sum: 2^25 such tiles stay below 2^90
// What the start and the end of an item cost, in tiles: with 4, 6 and 8 of them two prompts of up to 4096 tokens (bf16) take
// 133, 131, 134 us at a head size of 64, 169, 160, 158 at 128, 367, 333, 310 at 256; 512 new tokens over 16384 differ by 1 %.
constexpr int kItemUnits = 6;
constexpr int kMinUnits = 8;
constexpr uint32_t kSuspendNs = 20000;// up to which the hardware may keep a waiting thread suspended
constexpr int kScaleSets = 4;// a set is rewritten four tiles later, when the rows of its tile are long done

__host__ __device__ constexpr int blocks_at_once(int dhc) { return dhc <= 128 ? 2 : 1; }
__host__ __device__ constexpr int threads_of(int nb) { return 128 * nb + 256; }
// Registers per thread: at launch (all of the SM's), and after the warpgroups have traded: the softmax holds the 64 scores of
// a row's tile and their weights.  Whole warpgroups only: a 17th warp would cost the launch 32 registers per thread.
__host__ __device__ constexpr int launch_regs(int nb) { return nb == 2 ? 128 : 168; }
__host__ __device__ constexpr int softmax_regs(int nb) { return nb == 2 ? 184 : 240; }
__host__ __device__ constexpr int convert_regs(int nb) { return nb == 2 ? 88 : 152; }
__host__ __device__ constexpr int issue_regs(int nb) { return nb == 2 ? 56 : 112; }
__host__ __device__ constexpr bool split_fits(int nb) {
    return nb * softmax_regs(nb) + convert_regs(nb) + issue_regs(nb) <= (nb + 2) * launch_regs(nb) && threads_of(nb) * launch_regs(nb) <= 65536;
}
static_assert(split_fits(1) && split_fits(2), "the registers' split fits what the launch gave");

// TMEM columns of a block: S (and the weights over it) [0, 64) and [64, 128), O from 128; the second block from 256.
constexpr uint32_t kTmemCols = 512;

// barriers; the second block's own follow the first's
enum Bar { kKFull, kKFull1, kKEmpty, kKEmpty1, kVFull, kVFull1, kVEmpty, kVEmpty1, kDrained, kScFull, kBlock = kScFull + kScaleSets,
           kQFull = 0, kSFull, kSFull1, kWFull, kWFull1, kPvDone, kPvDone1, kBlockBars, kBars = kBlock + 2 * kBlockBars };

struct TileScales {
    float ks[kKeys], lv[kKeys];// scales of the keys, log2 of the values'
    uint32_t mask[2], pad[2];             // tokens that exist
};

__host__ __device__ constexpr uint32_t q_bytes(int dhc) { return (uint32_t) dhc * 2 * kRows; }// of one block
__host__ __device__ constexpr uint32_t kv_bytes(int dhc) { return (uint32_t) dhc * 2 * kKeys; }
// q of an item and, where it fits, of the next one
__host__ __device__ constexpr uint32_t q_buffers(int dhc) { return dhc <= 128 ? 2 : 1; }
__host__ __device__ constexpr uint32_t tile_bytes(int dhc) { return q_buffers(dhc) * (uint32_t) blocks_at_once(dhc) * q_bytes(dhc) + 4 * kv_bytes(dhc); }
__host__ __device__ constexpr uint32_t smem_bytes(int dhc) { return tile_bytes(dhc) + kScaleSets * (uint32_t) sizeof(TileScales) + kBars * 8 + 32; }
static_assert(smem_bytes(64) <= 232448 && smem_bytes(128) <= 232448 && smem_bytes(256) <= 232448, "a CTA's shared memory");
static_assert(kPrefillMaxBatch * 8 <= tile_bytes(64), "the sequences' unit counts fit the tiles' memory");

// Products issued by a warp as a whole, the instruction itself by its elected lane: D[tmem] (+)= A * B[smem desc], A from
// shared memory or from TMEM (rows are lanes, two fp16 elements per column).  Code that the compiler knows to be the same
// in all lanes keeps descriptors in uniform registers; in a branch of one lane each product took 96 cycles to issue
// whatever its size, here 48 (64 columns of B) and 64 (128 columns), the tensor core's own pace.
__device__ __forceinline__ uint32_t elect_lane() {
    uint32_t lead;
    asm volatile("{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(lead));
    return lead;
}
__device__ __forceinline__ void umma_f16_ss(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate, uint32_t lead) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "setp.ne.b32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate), "r"(lead)
        : "memory");
}
__device__ __forceinline__ void umma_f16_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate, uint32_t lead) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "setp.ne.b32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
        ::"r"(tmem_d), "r"(tmem_a), "l"(desc_b), "r"(idesc), "r"(accumulate), "r"(lead)
        : "memory");
}
__device__ __forceinline__ void umma_commit_by(uint64_t *bar, uint32_t lead) {
    asm volatile(
        "{\n\t.reg .pred q;\n\t"
        "setp.ne.b32 q, %1, 0;\n\t"
        "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}"
        ::"r"(smem_u32(bar)), "r"(lead)
        : "memory");
}
// a poll that never suspends the thread
__device__ __forceinline__ bool mbar_test_wait(uint64_t *bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    return ok != 0;
}
// A warp waits as one: lanes leave a wait at different times, what follows (TMEM accesses, votes) is the whole warp's, and a
// wait that runs out ends the loop for all of its lanes.
__device__ __forceinline__ bool warp_wait(uint64_t *bar, uint32_t parity, volatile int *abort_flag, bool one_poll) {
    bool done = one_poll ? mbar_test_wait(bar, parity) : mbar_try_wait(bar, parity);
    if (!done) {
        const long long t0 = clock64();
        while (one_poll || !(done = mbar_try_wait_hint(bar, parity, kSuspendNs))) {
            if (*abort_flag) break;
            if (one_poll || clock64() - t0 > kWaitBudget) {
                *abort_flag = 1;
                atomicAdd(&g_tc_gemm_timeouts, 1ull);
                break;
            }
        }
    }
    return __all_sync(0xffffffffu, done);
}

// 32 columns of this warp's 32 lanes
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t *r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {"
        "%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, "
        "%22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};\n\t"
        "tcgen05.wait::st.sync.aligned;"
        ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
          "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]),
          "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]),
          "r"(r[30]), "r"(r[31])
        : "memory");
}
// 32 columns without the wait, and the wait
__device__ __forceinline__ void tmem_st32_start(uint32_t taddr, const float *r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {"
        "%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, "
        "%22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
        ::"r"(taddr), "f"(r[0]), "f"(r[1]), "f"(r[2]), "f"(r[3]), "f"(r[4]), "f"(r[5]), "f"(r[6]), "f"(r[7]), "f"(r[8]), "f"(r[9]),
          "f"(r[10]), "f"(r[11]), "f"(r[12]), "f"(r[13]), "f"(r[14]), "f"(r[15]), "f"(r[16]), "f"(r[17]), "f"(r[18]), "f"(r[19]),
          "f"(r[20]), "f"(r[21]), "f"(r[22]), "f"(r[23]), "f"(r[24]), "f"(r[25]), "f"(r[26]), "f"(r[27]), "f"(r[28]), "f"(r[29]),
          "f"(r[30]), "f"(r[31])
        : "memory");
}
__device__ __forceinline__ void tmem_st_finish() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// 64 columns of this warp's 32 lanes; the load and its wait are one statement
__device__ __forceinline__ void tmem_ld64(uint32_t taddr, float *v) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x64.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32, %33, %34, %35, %36, %37, %38, %39, %40, %41, %42, %43, %44, %45, %46, %47, %48, %49, %50, %51, %52, %53, %54, %55, %56, %57, %58, %59, %60, %61, %62, %63}, [%64];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]), "=f"(v[16]), "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]), "=f"(v[24]), "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31]), "=f"(v[32]), "=f"(v[33]), "=f"(v[34]), "=f"(v[35]), "=f"(v[36]), "=f"(v[37]), "=f"(v[38]), "=f"(v[39]), "=f"(v[40]), "=f"(v[41]), "=f"(v[42]), "=f"(v[43]), "=f"(v[44]), "=f"(v[45]), "=f"(v[46]), "=f"(v[47]), "=f"(v[48]), "=f"(v[49]), "=f"(v[50]), "=f"(v[51]), "=f"(v[52]), "=f"(v[53]), "=f"(v[54]), "=f"(v[55]), "=f"(v[56]), "=f"(v[57]), "=f"(v[58]), "=f"(v[59]), "=f"(v[60]), "=f"(v[61]), "=f"(v[62]), "=f"(v[63])
        : "r"(taddr)
        : "memory");
}
// 32 columns without the wait, and the wait that hands them over
__device__ __forceinline__ void tmem_ld32_start(uint32_t taddr, float *v) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
                 : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]), "=f"(v[16]), "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]), "=f"(v[24]), "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31])
                 : "r"(taddr)
                 : "memory");
}
__device__ __forceinline__ void tmem_ld32_finish(float *v) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]), "+f"(v[8]), "+f"(v[9]), "+f"(v[10]), "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]), "+f"(v[15]), "+f"(v[16]), "+f"(v[17]), "+f"(v[18]), "+f"(v[19]), "+f"(v[20]), "+f"(v[21]), "+f"(v[22]), "+f"(v[23]), "+f"(v[24]), "+f"(v[25]), "+f"(v[26]), "+f"(v[27]), "+f"(v[28]), "+f"(v[29]), "+f"(v[30]), "+f"(v[31]) :: "memory");
}
// two fp32 operations per instruction
__device__ __forceinline__ uint64_t pack2f(float lo, float hi) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ float2 unpack2f(uint64_t v) {
    float2 f;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(v));
    return f;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

// Items of a sequence and kv head, and the tiles of one: up to the last key that its last row sees, one at least (rows
// without keys get zeros).
template<int ROWS>
__device__ __forceinline__ int32_t items_of(const AttendParams &p, const Seq &s) {
    return (int32_t) (((uint32_t) s.n * (uint32_t) p.group + ROWS - 1) / ROWS);
}
template<int ROWS>
__device__ __forceinline__ int32_t tiles_of(const AttendParams &p, const Seq &s, int32_t rb) {
    const uint32_t rows = (uint32_t) s.n * (uint32_t) p.group, end = ((uint32_t) rb + 1) * ROWS;
    const int32_t tok = (int32_t) p.group_div.div((end < rows ? end : rows) - 1);
    const int32_t limit = min(s.len - s.n + tok + 1, held(s.len, p.t.cap));
    return limit > 0 ? (limit - 1) / kKeys + 1 : 1;
}

// A stretch of units, item by item.  Every role keeps its own.  The first kItemUnits units of an item hold no tile.
struct Segment {
    Seq s;
    int32_t b, kvh, rb, t0, t1, tiles;
    int64_t last_unit;// of the item
};
template<int ROWS>
struct Walker {
    const AttendParams &p;
    Seq s;
    int32_t b, kvh, rb, at, blocks;// `at`: unit of the item
    int64_t u, end;
    __device__ __forceinline__ bool next(Segment &g) {
        while (u < end) {
            if (blocks < 0) s = seq_of(p.lens, p.offs, p.rows, b), blocks = items_of<ROWS>(p, s);
            while (blocks == 0) s = seq_of(p.lens, p.offs, p.rows, ++b), blocks = items_of<ROWS>(p, s);// (units are left: there is one)
            const int32_t tiles = tiles_of<ROWS>(p, s, rb), size = tiles + kItemUnits;
            const int32_t n = end - u < size - at ? (int32_t) (end - u) : size - at;
            g.s = s, g.b = b, g.kvh = kvh, g.rb = rb, g.tiles = tiles;
            g.t0 = max(0, at - kItemUnits), g.t1 = max(0, at + n - kItemUnits);
            g.last_unit = u - at + size - 1;
            u += n;
            const bool ends = at + n == size;
            at = 0;
            if (ends && ++rb == blocks) {
                rb = 0;
                if (++kvh == p.c.heads) kvh = 0, ++b, blocks = -1;
            }
            if (g.t1 > g.t0) return true;
        }
        return false;
    }
};

template<int N>
__device__ __forceinline__ float largest(const float *v) {
    float t4[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
    for (int i = 4; i < N; i += 4) {
#pragma unroll
        for (int j = 0; j < 4; ++j) t4[j] = fmaxf(t4[j], v[i + j]);
    }
    return fmaxf(fmaxf(t4[0], t4[1]), fmaxf(t4[2], t4[3]));
}

// GROUPS of a tile's keys that each lie in one page: 1 (page sizes that are multiples of 64), 4 (of 16), 0 (any other, and
// codes whose rows are no aligned vectors: a page, a scale and a mask bit per key).  512 new tokens over 16384 cached ones, 32
// heads on 8 of 128 elements: 152 us with pages of 64 tokens (1), 165 us with 16 and 163 us with 48 (4), 436 us with 20 (0).
template<int DHC, int GROUPS>
__global__ void __launch_bounds__(threads_of(blocks_at_once(DHC)), 1) prefill_kernel(const SplitParams sp) {
    constexpr int kNB = blocks_at_once(DHC), kItemRows = kNB * kRows, kThreads = threads_of(kNB), kWarps = kThreads / 32;
    constexpr uint32_t kQ = q_bytes(DHC), kKV = kv_bytes(DHC);
    constexpr int kGroupsOr1 = GROUPS > 0 ? GROUPS : 1;
    extern __shared__ __align__(1024) unsigned char smem[];
    __shared__ int64_t slot[kWarps], found_base;
    __shared__ int32_t found_b, found_rb, found_t;
    const AttendParams &p = sp.a;
    // the swizzled tiles need 1024-byte alignment
    if ((smem_u32(smem) & 1023u) != 0) {
        if (threadIdx.x == 0) atomicAdd(&g_tc_gemm_timeouts, 1ull), sp.meta[blockIdx.x] = CtaMeta{-1, 0, 0, 0};
        return;
    }
    constexpr uint32_t kQBufs = q_buffers(DHC);
    const uint32_t sq = smem_u32(smem), sk = sq + kQBufs * kNB * kQ, sv = sk + 2 * kKV;
    TileScales *scales = reinterpret_cast<TileScales *>(smem + tile_bytes(DHC));
    uint64_t *bars = reinterpret_cast<uint64_t *>(scales + kScaleSets);
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + kBars);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
    const uint32_t warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;

    // ---- this CTA's stretch.  Units of a kv head of each sequence: a warp per sequence, a lane per item.
    int64_t *sums = reinterpret_cast<int64_t *>(smem);
    for (int32_t b = (int32_t) warp; b < p.t.batch; b += kWarps) {
        const Seq s = seq_of(p.lens, p.offs, p.rows, b);
        const int32_t blocks = items_of<kItemRows>(p, s);
        int64_t n = 0;
        for (int32_t rb = (int32_t) lane; rb < blocks; rb += 32) n += tiles_of<kItemRows>(p, s, rb) + kItemUnits;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
        if (lane == 0) sums[b] = n;
    }
    __syncthreads();
    int64_t mine = 0, total;
    for (int32_t b = (int32_t) threadIdx.x; b < p.t.batch; b += kThreads) mine += sums[b] * p.c.heads;
    cta_exclusive_sum64<kWarps>(mine, slot, total);
    const int64_t each = stretch_of(total, kMinUnits), u0 = each * blockIdx.x, u1 = u0 + each < total ? u0 + each : total;
    if (u0 >= u1) {
        if (threadIdx.x == 0) sp.meta[blockIdx.x] = CtaMeta{-1, 0, 0, 0};
        return;
    }
    {
        int64_t base = 0;
        for (int32_t b0 = 0; b0 < p.t.batch && base <= u0; b0 += kThreads) {
            const int32_t b = b0 + (int32_t) threadIdx.x;
            const int64_t n = b < p.t.batch ? sums[b] * p.c.heads : 0;
            int64_t sum;
            const int64_t before = base + cta_exclusive_sum64<kWarps>(n, slot, sum);
            if (u0 >= before && u0 - before < n) found_b = b, found_base = before;
            base += sum;
        }
        __syncthreads();
    }
    const int32_t b_first = found_b;
    const int64_t per_head = sums[b_first];
    const int32_t kvh_first = (int32_t) divide(u0 - found_base, per_head);
    if (warp == 0) {
        // the item where the stretch begins, and the unit in it
        const Seq s = seq_of(p.lens, p.offs, p.rows, b_first);
        const int32_t blocks = items_of<kItemRows>(p, s);
        const int64_t x = u0 - found_base - kvh_first * per_head;
        int64_t base = 0;
        for (int32_t rb0 = 0; rb0 < blocks && base <= x; rb0 += 32) {
            const int32_t rb = rb0 + (int32_t) lane;
            const int64_t n = rb < blocks ? tiles_of<kItemRows>(p, s, rb) + kItemUnits : 0;
            int64_t incl = n;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int64_t v = __shfl_up_sync(0xffffffffu, incl, o);
                if ((int) lane >= o) incl += v;
            }
            const int64_t before = base + incl - n;
            if (x >= before && x - before < n) found_rb = rb, found_t = (int32_t) (x - before);
            base += __shfl_sync(0xffffffffu, incl, 31);
        }
    }
    if (threadIdx.x == 32) {
        for (int i = 0; i < kBars; ++i) {
            const int own = i >= kBlock ? (i - kBlock) % kBlockBars : -1;
            const bool rows = own == kQFull || own == kWFull || own == kWFull1;
            const bool codes = i == kKFull || i == kKFull1 || i == kVFull || i == kVFull1, keys = i >= kScFull && i < kBlock;
            mbar_init(&bars[i], rows ? 128u : codes || keys ? 64u : 1u);
        }
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kWarps - 1) {
        tmem_alloc(tmem_slot, kTmemCols);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();// (the sums are read, the tiles' memory is free)
    tc_fence_after();
    if (p.c.dh < DHC) {
        // codes of head elements beyond dh: zeros that nothing overwrites
        for (uint32_t i = threadIdx.x * 16; i < 4 * kKV; i += kThreads * 16) {
            asm volatile("st.shared.v4.u32 [%0], {%1,%1,%1,%1};" ::"r"(sk + i), "r"(0) : "memory");
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncthreads();
    }
    const uint32_t tmem = *tmem_slot;
    Walker<kItemRows> walk{p, Seq{}, b_first, kvh_first, found_rb, found_t, -1, u0, u1};
    Segment g;
    // the second block of an item has rows
    auto second = [&](const Segment &x) { return kNB == 2 && (uint32_t) x.s.n * (uint32_t) p.group > (uint32_t) x.rb * kItemRows + kRows; };

    if (warp >= kWarps - 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(issue_regs(kNB)));
        if (warp == kWarps - 1) {
        // ------------------------------------------------------------ products
        // (the shuffles and votes tell the compiler what is the same in all lanes)
        const uint32_t steps = (uint32_t) (p.c.dh + 15) / 16;// of 16 head elements
        const uint32_t idesc_s = make_idesc(kRows, kKeys, 0, 0), idesc_o = make_idesc(kRows, steps * 16, 0, 1);
        const uint64_t dq = make_smem_desc(sq, 16, 1024), dk = make_smem_desc(sk, 16, 1024), dv = make_smem_desc(sv, kKeys * 128u, 1024);
        const uint32_t lead = elect_lane(), tm = __shfl_sync(0xffffffffu, tmem, 0);
        uint32_t n = 0, bn[2] = {0, 0}, bseg[2] = {0, 0};// tiles of the stretch; tiles and items of each block
        auto wait = [&](uint64_t *bar, uint32_t parity) -> bool {
            const bool done = warp_wait(bar, parity, abort_flag, sp.one_poll);
            tc_fence_after();
            return done;
        };
        // S of the n-th tile for the active blocks
        auto issue_s = [&](uint32_t i, uint32_t ahead, int nb) -> bool {
            const uint32_t b = i & 1u;
            if (!wait(&bars[kKFull + b], (i >> 1) & 1u)) return false;
#pragma unroll
            for (int x = 0; x < kNB; ++x) {
                if (x >= nb) break;
                const uint32_t sb = (bn[x] + ahead) & 1u;
#pragma unroll 1
                for (uint32_t box = 0; box * 4 < steps; ++box) {// 64 elements (four products) at a time
                    const uint64_t dqb = dq + ((((kQBufs == 2 ? (bseg[x] - 1) & 1u : 0u) * kNB + x) * kQ + box * (kRows * 128u)) >> 4), dkb = dk + ((b * kKV + box * (kKeys * 128u)) >> 4);
#pragma unroll
                    for (uint32_t k = 0; k < 4; ++k) {
                        if (box * 4 + k < steps) umma_f16_ss(tm + x * 256u + sb * kKeys, dqb + 2 * k, dkb + 2 * k, idesc_s, (box | k) > 0 ? 1u : 0u, lead);
                    }
                }
                if (x + 1 == nb) umma_commit_by(&bars[kKEmpty + b], lead);
                umma_commit_by(&bars[kBlock + x * kBlockBars + kSFull + sb], lead);
            }
            return true;
        };
        bool ok = true;
        while (ok && __any_sync(0xffffffffu, walk.next(g))) {
            const uint32_t tiles = __shfl_sync(0xffffffffu, (uint32_t) (g.t1 - g.t0), 0);
            const int nb = __any_sync(0xffffffffu, second(g)) ? 2 : 1;
            for (int x = 0; ok && x < nb; ++x) ok = wait(&bars[kBlock + x * kBlockBars + kQFull], bseg[x]++ & 1u);
            if (!ok || !(ok = issue_s(n, 0, nb))) break;
            for (uint32_t j = 0; ok && j < tiles; ++j, ++n) {
                const uint32_t b = n & 1u;
                if (j + 1 < tiles && !(ok = issue_s(n + 1, 1, nb))) break;
                if (!(ok = wait(&bars[kVFull + b], (n >> 1) & 1u))) break;
#pragma unroll
                for (int x = 0; x < kNB; ++x) {
                    if (x >= nb) break;
                    uint64_t *own = bars + kBlock + x * kBlockBars;
                    const uint32_t sb = bn[x] & 1u;
                    if (!(ok = wait(&own[kWFull + sb], (bn[x] >> 1) & 1u))) break;
#pragma unroll
                    for (uint32_t k = 0; k < kKeys / 16; ++k) {
                        umma_f16_ts(tm + x * 256u + 2 * kKeys, tm + x * 256u + sb * kKeys + k * 8u, dv + ((b * kKV + k * 2048u) >> 4), idesc_o,
                                    (j > 0 || k > 0) ? 1u : 0u, lead);
                    }
                    if (x + 1 == nb) umma_commit_by(&bars[kVEmpty + b], lead);
                    umma_commit_by(&own[kPvDone + sb], lead);
                    ++bn[x];
                }
            }
        }
        __syncwarp();
        }
    } else if (warp >= 4 * kNB) {
        // ------------------------------------------------------------ codes to fp16: two warps for K and the scales, two for V
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(convert_regs(kNB)));
        constexpr int kGroups = DHC / 64;// 4 lanes take 64 bytes of a row; 8 rows per warp and load
        constexpr int kLoads = 4;// rows per thread, 16 apart
        const bool is_v = warp >= 4 * kNB + 2;
        const uint32_t c = (threadIdx.x - 128 * kNB) & 63u, cw = c >> 5, c4 = lane & 3u, r0 = cw * 8 + (lane >> 2);
        uint64_t *full = bars + (is_v ? kVFull : kKFull), *empty = bars + (is_v ? kVEmpty : kKEmpty);
        const PoolStrides st = is_v ? p.c.v : p.c.k;
        const uint8_t *pool = (is_v ? p.vp : p.kp) + c4 * 16;
        // rows as TMA with 128-byte swizzle would lay them: 16-byte chunk j of row r at j ^ (r & 7); this thread's rows are
        // r0, r0 + 16, .., its chunks 2 c4 and 2 c4 + 1 of every box of 64 elements
        const uint32_t row_at = (is_v ? sv : sk) + r0 * 128u, chunk0 = ((2 * c4) ^ (r0 & 7u)) << 4, chunk1 = ((2 * c4 + 1) ^ (r0 & 7u)) << 4;
        uint4 data[kLoads][kGroups];
        auto store_tile = [&](uint32_t b) {
            const uint32_t at = row_at + b * kKV;
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
#pragma unroll
                for (int q = 0; q < kGroups; ++q) {
                    if ((q * 4 + (int32_t) c4) * 16 >= p.c.dh) continue;
                    const uint4 w = data[i][q];
                    uint32_t h[8];
                    e4m3x4_to_f16x4(w.x, h[0], h[1]), e4m3x4_to_f16x4(w.y, h[2], h[3]);
                    e4m3x4_to_f16x4(w.z, h[4], h[5]), e4m3x4_to_f16x4(w.w, h[6], h[7]);
                    const uint32_t row = at + (uint32_t) (q * (kKeys * 128) + i * (16 * 128));
                    asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(row + chunk0), "r"(h[0]), "r"(h[1]), "r"(h[2]), "r"(h[3]) : "memory");
                    asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(row + chunk1), "r"(h[4]), "r"(h[5]), "r"(h[6]), "r"(h[7]) : "memory");
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");// the products read through the async proxy
        };
        bool ok = true;
        uint32_t n = 0;
        while (ok && walk.next(g)) {
            // The codes of a tile are loaded while the tile before is converted.
            const int32_t keys = held(g.s.len, p.t.cap), t1 = g.t1;
            const int32_t *ids = p.table + (int64_t) g.b * p.t.stride;
            const uint8_t *head = pool + (int64_t) g.kvh * st.sh;
            if constexpr (GROUPS > 0) {
                // Lane j holds where the codes of the j-th of 32 groups begin (-1: no page), so that pages are read once in
                // kChunk tiles; the next 32 are requested long before they are looked at.
                constexpr int kChunk = 32 / kGroupsOr1, kTokens = kKeys / kGroupsOr1;
                auto page_at = [&](int32_t group) -> int32_t {
                    return group >= t1 * kGroupsOr1 || group * kTokens >= keys ? -1 : ids[p.page_div.div((uint32_t) (group * kTokens))];
                };
                auto base_of = [&](int32_t group, int32_t page) -> int64_t {
                    if (page < 0 || page >= p.c.pages) return -1;
                    const int32_t tok = group * kTokens;
                    return (int64_t) page * st.sn + (int64_t) (tok - (int32_t) p.page_div.div((uint32_t) tok) * p.c.page) * st.sp;
                };
                int32_t first = g.t0, id_next = -1;// `first`: the tile of lane 0
                int64_t base = base_of(first * kGroupsOr1 + (int32_t) lane, page_at(first * kGroupsOr1 + (int32_t) lane));
                const uint8_t *mine = head + (int64_t) r0 * st.sp;
                const int64_t step = 16 * st.sp;
                auto load = [&](int32_t tile) {
                    const int32_t left = keys - tile * kKeys;
                    int64_t from = __shfl_sync(0xffffffffu, base, (tile - first) * kGroupsOr1);
#pragma unroll
                    for (int i = 0; i < kLoads; ++i) {// (16 rows apart: the i-th group's where there are four)
                        if (GROUPS == 4 && i > 0) from = __shfl_sync(0xffffffffu, base, (tile - first) * kGroupsOr1 + i);
                        const uint8_t *at = mine + from + (GROUPS == 4 ? 0 : i * step);
#pragma unroll
                        for (int q = 0; q < kGroups; ++q) {
                            data[i][q] = make_uint4(0u, 0u, 0u, 0u);
                            if (from >= 0 && (int32_t) r0 + 16 * i < left && (q * 4 + (int32_t) c4) * 16 < p.c.dh) data[i][q] = *reinterpret_cast<const uint4 *>(at + q * 64);
                        }
                    }
                };
                load(g.t0);
#pragma unroll 1
                for (int32_t tile = g.t0; tile < t1; ++tile, ++n) {
                    const uint32_t b = n & 1u;
                    const int32_t j = tile - first;
                    if (j == kChunk / 2) id_next = page_at((first + kChunk) * kGroupsOr1 + (int32_t) lane);
                    if (!(ok = warp_wait(&empty[b], ((n >> 1) & 1u) ^ 1u, abort_flag, sp.one_poll))) break;
                    store_tile(b);
                    mbar_arrive(&full[b]);
                    if (j == kChunk - 1) first += kChunk, base = base_of(first * kGroupsOr1 + (int32_t) lane, id_next);
                    if (tile + 1 < t1) load(tile + 1);
                }
            } else {
                // pages that end inside a tile: a page per row and per key
                auto page_of = [&](int32_t tok) -> int32_t {
                    if (tok >= keys) return -1;
                    const int32_t x = ids[p.page_div.div((uint32_t) tok)];
                    return x >= 0 && x < p.c.pages ? x : -1;
                };
                float ks = 0.f, vs = 0.f;
                bool key_ok = false;
                auto load = [&](int32_t tile) {
#pragma unroll
                    for (int i = 0; i < kLoads; ++i) {
                        const int32_t tok = tile * kKeys + (int32_t) r0 + 16 * i, page = page_of(tok);
                        const int32_t in_page = tok - (int32_t) p.page_div.div((uint32_t) tok) * p.c.page;
                        const uint8_t *at = head + (int64_t) max(page, 0) * st.sn + (int64_t) in_page * st.sp;
#pragma unroll
                        for (int q = 0; q < kGroups; ++q) {
                            const int32_t d0 = (q * 4 + (int32_t) c4) * 16;
                            data[i][q] = make_uint4(0u, 0u, 0u, 0u);
                            if (page < 0 || d0 >= p.c.dh) continue;
                            if (p.vec) {
                                data[i][q] = *reinterpret_cast<const uint4 *>(at + q * 64);
                            } else {// rows that are no whole aligned vectors: code by code
                                uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
                                for (int x = 0; x < 4; ++x) {
#pragma unroll 1
                                    for (int y = 0; y < 4; ++y) {
                                        if (d0 + 4 * x + y < p.c.dh) w[x] |= (uint32_t) at[q * 64 + 4 * x + y] << (8 * y);
                                    }
                                }
                                data[i][q] = make_uint4(w[0], w[1], w[2], w[3]);
                            }
                        }
                    }
                    if (!is_v) {
                        const int32_t page = page_of(tile * kKeys + (int32_t) c);
                        key_ok = page >= 0;
                        ks = key_ok ? p.ks[(int64_t) page * p.c.k.cn + (int64_t) g.kvh * p.c.k.ch] : 0.f;
                        vs = key_ok ? p.vs[(int64_t) page * p.c.v.cn + (int64_t) g.kvh * p.c.v.ch] : 0.f;
                    }
                };
                load(g.t0);
                for (int32_t tile = g.t0; tile < t1; ++tile, ++n) {
                    const uint32_t b = n & 1u;
                    if (!(ok = warp_wait(&empty[b], ((n >> 1) & 1u) ^ 1u, abort_flag, sp.one_poll))) break;
                    if (!is_v) {
                        TileScales &sc = scales[n % kScaleSets];
                        const uint32_t mask = __ballot_sync(0xffffffffu, key_ok);
                        sc.ks[c] = ks, sc.lv[c] = log2_of(vs);
                        if (lane == 0) sc.mask[cw] = mask;
                        mbar_arrive(&bars[kScFull + n % kScaleSets]);
                    }
                    store_tile(b);
                    mbar_arrive(&full[b]);
                    if (tile + 1 < t1) load(tile + 1);
                }
            }
        }
    } else {
        // ------------------------------------------------------------ softmax and epilogue: a thread per row
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(softmax_regs(kNB)));
        const uint32_t blk = warp >> 2, quarter = warp & 3u, r = quarter * 32u + lane;// row of the block
        const uint32_t t_lane = tmem + blk * 256u + ((quarter * 32u) << 16);
        uint64_t *own = bars + kBlock + blk * kBlockBars;
        CtaMeta meta{-1, 0, 0, 0};
        bool ok = true;
        uint32_t n_all = 0, n = 0;// tiles of the stretch, and of them this block's
        // the next item with rows in this block; tiles of those without
        auto next_item = [&](Segment &x, uint32_t &skipped) -> bool {
            skipped = 0;
            while (walk.next(x)) {
                if (blk == 0 || second(x)) return true;
                skipped += (uint32_t) (x.t1 - x.t0);
            }
            return false;
        };
        // q of a row: its first row in the block, the row's token, whether it exists, where it is
        struct Place {
            uint32_t rr0, rows;
            int32_t tok, head;
            bool have;
        };
        auto place_of = [&](const Segment &x) -> Place {
            Place y;
            y.rows = (uint32_t) x.s.n * (uint32_t) p.group, y.rr0 = (uint32_t) x.rb * kItemRows + blk * kRows;
            y.have = y.rr0 + r < y.rows;
            y.tok = y.have ? (int32_t) p.group_div.div(y.rr0 + r) : 0;
            y.head = x.kvh * p.group + (y.have ? (int32_t) (y.rr0 + r) - y.tok * p.group : 0);
            return y;
        };
        // q: a warp requests its 32 rows, a row's 16-byte pieces side by side in the lanes, into swizzled shared memory, zeros
        // for rows that there are not and head elements beyond dh.
        auto request_q = [&](const Segment &x, uint32_t to) {
            constexpr int kPer = DHC / 8, kAtOnce = 32 / kPer;// lanes per row, rows at once
            const Place y = place_of(x);
            const int32_t d = (int32_t) (lane % kPer) * 8;
            const bool vec = p.q_vec && p.c.dh % 8 == 0;
            const int64_t mine = (int64_t) (x.s.first + y.tok) * p.q_st + (int64_t) y.head * p.q_sh;
#pragma unroll 4
            for (int i = 0; i < 32 / kAtOnce; ++i) {
                const uint32_t row = (uint32_t) i * kAtOnce + lane / kPer, br = quarter * 32u + row;
                const uint16_t *from = p.q + __shfl_sync(0xffffffffu, mine, (int) row);
                const bool valid = y.rr0 + br < y.rows && d < p.c.dh;
                const uint32_t at = to + ((uint32_t) d >> 6) * (kRows * 128u) + br * 128u + (((((uint32_t) d >> 3) & 7u) ^ (br & 7u)) << 4);
                if (vec) {
                    cp_async16(at, valid ? from + d : p.q, valid);
                } else {
                    uint32_t e[4] = {0u, 0u, 0u, 0u};
                    if (valid) {
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            if (d + 2 * k < p.c.dh) e[k] = (uint32_t) from[d + 2 * k];
                            if (d + 2 * k + 1 < p.c.dh) e[k] |= (uint32_t) from[d + 2 * k + 1] << 16;
                        }
                    }
                    asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(e[0]), "r"(e[1]), "r"(e[2]), "r"(e[3]) : "memory");
                }
            }
            cp_async_commit();
        };
        // q has come: fp16 rows stay as they are; bf16 rows are multiplied by a power of two after their largest magnitude, a
        // thread per row.  The sign of the scale goes with q, so that the factor of the scores (returned) is not negative.
        auto finish_q = [&](uint32_t at0) -> float {
            float f = fabsf(p.scale_log2);
            cp_async_wait<0>();
            __syncwarp();
            const uint32_t flip = p.scale_log2 < 0.f ? 0x80008000u : 0u;
            if (p.bf16 || flip != 0u) {
                const uint32_t row = at0 + r * 128u;
                float up = 1.f;
                if (p.bf16) {
                    uint32_t top = 0u;
#pragma unroll
                    for (uint32_t i = 0; i < DHC / 8; ++i) {
                        const uint4 x = lds128(row + (i >> 3) * (kRows * 128u) + (((i & 7u) ^ (r & 7u)) << 4));
                        top = __vmaxu2(__vmaxu2(__vmaxu2(top, x.x & 0x7FFF7FFFu), __vmaxu2(x.y & 0x7FFF7FFFu, x.z & 0x7FFF7FFFu)), x.w & 0x7FFF7FFFu);
                    }
                    const int32_t shift = query_shift(true, max(top & 0xFFFFu, top >> 16));
                    up = __uint_as_float(pow2_bits(shift)), f *= __uint_as_float(pow2_bits(-shift));
                }
#pragma unroll 4
                for (uint32_t i = 0; i < DHC / 8; ++i) {
                    const uint32_t at = row + (i >> 3) * (kRows * 128u) + (((i & 7u) ^ (r & 7u)) << 4);
                    const uint4 v = lds128(at);
                    uint32_t x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        if (p.bf16) {
                            const float2 y = unpack2_t<kBF16>(x[k]);
                            x[k] = round16x2(false, y.x * up, y.y * up);
                        }
                        x[k] ^= flip;
                    }
                    asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3]) : "memory");
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            mbar_arrive(&own[kQFull]);
            return f;
        };
        // The pages and scales of 32 groups in the lanes, as in the converting warps.  (The upper bound is looked at later, so
        // that nothing waits for the load.)
        constexpr int kChunk = 32 / kGroupsOr1, kTokens = kKeys / kGroupsOr1;
        auto page_at = [&](const Segment &x, int32_t tile) -> int32_t {
            const int32_t group = tile * kGroupsOr1 + (int32_t) lane;
            if (group >= x.t1 * kGroupsOr1 || group * kTokens >= held(x.s.len, p.t.cap)) return -1;
            return p.table[(int64_t) x.b * p.t.stride + (int64_t) p.page_div.div((uint32_t) (group * kTokens))];
        };
        auto scales_of = [&](const Segment &x, int32_t page, float &k, float &v) {
            k = page >= 0 ? p.ks[(int64_t) page * p.c.k.cn + (int64_t) x.kvh * p.c.k.ch] : 0.f;
            v = page >= 0 ? p.vs[(int64_t) page * p.c.v.cn + (int64_t) x.kvh * p.c.v.ch] : 0.f;
        };
        // What the next item needs is requested while this one is worked on, and its q is made ready before this one's output
        // leaves, so that its first scores are computed meanwhile.
        Segment gn;
        uint32_t skipped, buf = 0;
        int32_t id = -1;
        float rf_next = 0.f, ks = 0.f, vs = 0.f;
        bool more = next_item(gn, skipped);
        if (more) {
            request_q(gn, sq + blk * kQ);
            if (GROUPS > 0) id = page_at(gn, gn.t0);
            rf_next = finish_q(sq + blk * kQ);
            if (id >= p.c.pages) id = -1;
            if (GROUPS > 0) scales_of(gn, id, ks, vs);
        }
        while (ok && more) {
            g = gn, n_all += skipped;
            const float rf = rf_next;
            const uint32_t myq = sq + (buf * kNB + blk) * kQ, other = kQBufs == 2 ? sq + ((buf ^ 1u) * kNB + blk) * kQ : myq;
            const Seq s = g.s;
            const Place at_q = place_of(g);
            const uint32_t rows = at_q.rows, rr0 = at_q.rr0;
            const bool have = at_q.have;
            const int32_t tok = at_q.tok;
            const int32_t limit = have ? max(0, min(s.len - s.n + tok + 1, held(s.len, p.t.cap))) : 0;// keys this row sees
            more = next_item(gn, skipped);
            if (kQBufs == 2 && more) request_q(gn, other);
            int32_t first = g.t0, id_next = -1;
            float ks_next = 0.f, vs_next = 0.f;
            float m = -INFINITY, wm = -INFINITY, l = 0.f;
            // O so far is multiplied by a factor per row.  Every product into it must have completed.
            auto scale_o = [&](float by) -> bool {
                if (!warp_wait(&own[kPvDone + ((n & 1u) ^ 1u)], ((n - 1) >> 1) & 1u, abort_flag, sp.one_poll)) return false;
                tc_fence_after();
                for (int32_t c0 = 0; c0 < p.c.dh; c0 += 64) {
                    float o[64];
                    tmem_ld64(t_lane + 2 * kKeys + c0, o);
#pragma unroll
                    for (int i = 0; i < 64; ++i) o[i] *= by;
                    tmem_st32_start(t_lane + 2 * kKeys + c0, o);
                    tmem_st32_start(t_lane + 2 * kKeys + c0 + 32, o + 32);
                }
                tmem_st_finish();
                return true;
            };
            // The references of the rows that ask for it rise to this tile's largest: O so far and the sum follow.  (A score
            // may be the largest so far and its weight a small one, by its values' scale, and the other way round.)
            auto move_references = [&](bool up, float top, float wtop, int32_t tile) -> bool {
                float shrink = 1.f;
                if (up) {
                    const float m_new = fmaxf(m, top), wm_new = fmaxf(wm, wtop);
                    if (wm_new > wm) shrink = fast_exp2(wm - wm_new);// (from -inf: 0)
                    l *= fast_exp2(m - m_new);
                    m = m_new, wm = wm_new;
                }
                return tile == g.t0 || !__any_sync(0xffffffffu, up) || scale_o(shrink);
            };
            if constexpr (GROUPS > 0) {
                float lv_lane = log2_of(vs);
                // per group: exponent from p to w, 2^-e, e - m, and the scale (log2) they are for
                float e[GROUPS], e_back[GROUPS], shift[GROUPS], lv_of_e[GROUPS];
#pragma unroll
                for (int i = 0; i < GROUPS; ++i) lv_of_e[i] = NAN;
                auto forget = [&]() {
#pragma unroll
                    for (int i = 0; i < GROUPS; ++i) lv_of_e[i] = NAN;
                };
                // the groups' factors and scales, those without a page, and how many of the tile's keys this row sees; formed
                // while the tile before is worked on
                float factor[GROUPS], lv[GROUPS];
                int32_t left;
                uint32_t gone;
                bool hidden;
                auto look_at = [&](int32_t tile) {
                    const int32_t j = (tile - first) * GROUPS;
                    gone = __ballot_sync(0xffffffffu, id < 0) >> j & ((1u << GROUPS) - 1u);
#pragma unroll
                    for (int i = 0; i < GROUPS; ++i) factor[i] = __shfl_sync(0xffffffffu, ks, j + i) * rf, lv[i] = __shfl_sync(0xffffffffu, lv_lane, j + i);
                    left = limit - tile * kKeys;
                    if (GROUPS == 1 && gone != 0u) left = 0, gone = 0u;
                    hidden = __any_sync(0xffffffffu, have && (left < kKeys || gone != 0u));
                };
                look_at(g.t0);
#pragma unroll 1
                for (int32_t tile = g.t0; tile < g.t1; ++tile, ++n) {
                    const uint32_t b = n & 1u, gone_now = gone;
                    const int32_t j = tile - first, left_now = left;
                    float factor_now[GROUPS], lv_now[GROUPS];
#pragma unroll
                    for (int i = 0; i < GROUPS; ++i) factor_now[i] = factor[i], lv_now[i] = lv[i];
                    const bool hidden_now = hidden;
                    // a row without a reference (its first keys are in this tile) looks through the tile for its largest score
                    bool move = m == -INFINITY && left > 0;
                    const bool some = __any_sync(0xffffffffu, move);
                    auto next = [&]() {
                        // pages and scales of the next 32 groups: requested and looked at some tiles apart
                        if (j == kChunk / 2) id_next = page_at(g, first + kChunk);
                        if (j == kChunk * 3 / 4 - 2 + GROUPS / 2) {
                            if (id_next >= p.c.pages) id_next = -1;
                            scales_of(g, id_next, ks_next, vs_next);
                        }
                        if (j == kChunk - 1) first += kChunk, id = id_next, ks = ks_next, lv_lane = log2_of(vs_next);
                        if (tile + 1 < g.t1) look_at(tile + 1);
                    };
                    if (!(ok = warp_wait(&own[kSFull + b], (n >> 1) & 1u, abort_flag, sp.one_poll))) break;
                    tc_fence_after();
                    uint32_t w[kKeys / 2];
                    float gain = 0.f, most = 0.f;// what the tile adds to l; the largest sum of 16 (or 8) weights
                    auto exponents = [&]() {
#pragma unroll
                        for (int i = 0; i < GROUPS; ++i) {
                            if (!(lv_now[i] == lv_of_e[i])) {// (the references or the scale have changed)
                                e[i] = wm == -INFINITY ? 0.f : fmaxf(m - wm + kLift + lv_now[i], kLeast);
                                e_back[i] = fast_exp2(-e[i]);
                                shift[i] = e[i] - (m == -INFINITY ? 0.f : m);
                                lv_of_e[i] = lv_now[i];
                            }
                        }
                    };
                    // Weights of half a tile (the `half`-th), and what they add up to: four sums of 16 keys of the tile, or two
                    // of 8 keys of each group.
                    uint64_t part[GROUPS == 4 ? 4 : 2];
                    auto weigh = [&](float *x, uint32_t *to, const float *f, int half) {
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            const int gr = GROUPS == 4 ? 2 * half + (i >> 3) : 0, at = GROUPS == 4 ? gr : i & 1;
                            const float2 a = unpack2f(fma2(pack2f(x[2 * i], x[2 * i + 1]), pack2f(f[gr], f[gr]), pack2f(shift[gr], shift[gr])));
                            x[2 * i] = fast_exp2(a.x), x[2 * i + 1] = fast_exp2(a.y);
                            part[at] = add2(part[at], pack2f(x[2 * i], x[2 * i + 1]));
                            to[i] = round16x2(false, x[2 * i], x[2 * i + 1]);
                        }
                    };
                    auto add_up = [&]() {
                        gain = most = 0.f;
                        if (GROUPS == 4) {
#pragma unroll
                            for (int i = 0; i < GROUPS; ++i) {
                                const float2 y = unpack2f(part[i]);
                                gain = fmaf(y.x + y.y, e_back[i], gain), most = fmaxf(most, fmaxf(y.x, y.y));
                            }
                        } else {
                            const float2 s0 = unpack2f(part[0]), s1 = unpack2f(part[1]);
                            gain = __fmul_rn((s0.x + s0.y) + (s1.x + s1.y), e_back[0]);
                            most = fmaxf(fmaxf(s0.x, s0.y), fmaxf(s1.x, s1.y));
                        }
                    };
                    // (the sum of p may go far where the weights tell nothing, where the values' scale is small)
                    auto far = [&]() -> bool { return most > kFarWeight || gain > kFarGain; };
                    auto clear = [&]() {
#pragma unroll
                        for (int i = 0; i < (GROUPS == 4 ? 4 : 2); ++i) part[i] = 0ull;
                    };
                    // Most tiles hide nothing and move no reference: their weights are formed at once, and the sums tell
                    // whether one may have grown beyond what fp16 holds.  A row that finds so lets the weights' reference
                    // follow by a power of two, which its weights (still in fp32) and O are divided by, exactly.
                    //
                    // What a row does, and so its bits, depends on its own scores alone, whichever way its warp goes: a row
                    // without references takes its tile's largest; one whose weights or sum went far moves them there; one
                    // whose weights outgrew fp16 follows.  A tile taken a second time for the sake of one row gives the
                    // others the weights that they had: the same references, the same arithmetic (products and sums that
                    // the compiler may not contract).
                    float x[kKeys];
                    bool again = hidden_now || some;
                    if (!again) {
                        tmem_ld32(t_lane + b * kKeys, x);
                        tmem_ld32_start(t_lane + b * kKeys + 32, x + 32);
                        exponents();
                        clear();
                        weigh(x, w, factor_now, 0);
                        next();
                        tmem_ld32_finish(x + 32);
                        weigh(x + 32, w + 16, factor_now, 1);
                        add_up();
                        move = far();
                        again = __any_sync(0xffffffffu, move);
                    } else {
                        next();
                    }
                    if (again) {
#pragma unroll 1
                        for (int pass = 0; pass < 3; ++pass) {// (a row that has moved has weights of 2^lift at most: it ends here)
                            // (a factor of zero, which would make NaN of -inf, becomes scores of zero)
                            float f[GROUPS];
                            tmem_ld64(t_lane + b * kKeys, x);
#pragma unroll
                            for (int i = 0; i < GROUPS; ++i) f[i] = factor_now[i] > 0.f ? factor_now[i] : 1.f;
#pragma unroll
                            for (int i = 0; i < kKeys; ++i) {
                                const int gr = i / kTokens;
                                if (!(factor_now[gr] > 0.f)) x[i] *= factor_now[gr];
                                if (i >= left_now || (GROUPS > 1 && (gone_now >> gr & 1u))) x[i] = -INFINITY;
                            }
                            if (__any_sync(0xffffffffu, move)) {
                                float top = -INFINITY, wtop = -INFINITY;
#pragma unroll
                                for (int i = 0; i < GROUPS; ++i) {
                                    const float y = GROUPS == 4 ? largest<16>(x + i * kTokens) : fmaxf(largest<32>(x), largest<32>(x + 32));
                                    if (y > -INFINITY) top = fmaxf(top, __fmul_rn(y, f[i])), wtop = fmaxf(wtop, __fadd_rn(__fmul_rn(y, f[i]), lv_now[i]));
                                }
                                if (!(ok = move_references(move && top > -INFINITY, top, wtop, tile))) break;
                                forget();
                            }
                            exponents();
                            clear();
                            weigh(x, w, f, 0);
                            weigh(x + 32, w + 16, f, 1);
                            add_up();
                            move = far();
                            if (!__any_sync(0xffffffffu, move)) break;
                        }
                        if (!ok) break;
                    }
                    if (__any_sync(0xffffffffu, most > kMostWeight)) {
                        const float top = fmaxf(largest<32>(x), largest<32>(x + 32));
                        const int32_t up = most > kMostWeight ? (int32_t) (__float_as_uint(top) >> 23) - (127 + (int32_t) kLift) : 0;
                        const float by = __uint_as_float(pow2_bits(-up));
#pragma unroll
                        for (int i = 0; i < kKeys / 2; ++i) w[i] = round16x2(false, x[2 * i] * by, x[2 * i + 1] * by);
                        wm += (float) up, forget();
                        if (tile > g.t0 && !(ok = scale_o(by))) break;
                    }
                    l += gain;
                    __syncwarp();
                    tmem_st32(t_lane + b * kKeys, w);
                    tc_fence_before();
                    mbar_arrive(&own[kWFull + b]);
                }
            } else {
                // pages that end inside a tile: a factor, a scale and a mask bit per key, from shared memory
#pragma unroll 1
                for (int32_t tile = g.t0; tile < g.t1; ++tile, ++n, ++n_all) {
                    const uint32_t b = n & 1u;
                    const TileScales &sc = scales[n_all % kScaleSets];
                    if (!(ok = warp_wait(&own[kSFull + b], (n >> 1) & 1u, abort_flag, sp.one_poll))) break;
                    // (after S: a block that sat out items may be ahead by more than a parity can tell)
                    if (!(ok = warp_wait(&bars[kScFull + n_all % kScaleSets], (n_all / kScaleSets) & 1u, abort_flag, sp.one_poll))) break;
                    tc_fence_after();
                    float x[kKeys];
                    tmem_ld64(t_lane + b * kKeys, x);
                    const uint32_t m0 = sc.mask[0], m1 = sc.mask[1];
                    const int32_t left = limit - tile * kKeys;
                    const bool hidden = __any_sync(0xffffffffu, (m0 & m1) != 0xFFFFFFFFu || (have && left < kKeys));
#pragma unroll
                    for (int i = 0; i < kKeys; ++i) x[i] *= sc.ks[i] * rf;
                    if (hidden) {
#pragma unroll
                        for (int i = 0; i < kKeys; ++i) {
                            if (!(((i < 32 ? m0 : m1) >> (i & 31)) & 1u) || i >= left) x[i] = -INFINITY;
                        }
                    }
                    const float top = fmaxf(largest<32>(x), largest<32>(x + 32));
                    float wtop = -INFINITY;
#pragma unroll
                    for (int i = 0; i < kKeys; ++i) wtop = fmaxf(wtop, x[i] == -INFINITY ? -INFINITY : x[i] + sc.lv[i]);
                    // (the sum's own reference: it may exceed the weights' by what the scales differ)
                    const bool far = top > m + 64.f && m != -INFINITY;
                    if (far) l *= fast_exp2(m - top), m = top;
                    const bool up = wtop > wm + kSlack || (wm == -INFINITY && wtop > wm);
                    if (__any_sync(0xffffffffu, up) && !(ok = move_references(up, top, wtop, tile))) break;
                    const float mm = m == -INFINITY ? 0.f : m, e = wm == -INFINITY ? 0.f : mm - wm + kLift;
                    uint32_t w[kKeys / 2];
                    float sum = 0.f;
#pragma unroll
                    for (int i = 0; i < kKeys / 2; ++i) {
                        const float a0 = x[2 * i] - mm, a1 = x[2 * i + 1] - mm;
                        sum += fast_exp2(a0) + fast_exp2(a1);
                        w[i] = round16x2(false, a0 == -INFINITY ? 0.f : fast_exp2(a0 + (e + sc.lv[2 * i])),
                                         a1 == -INFINITY ? 0.f : fast_exp2(a1 + (e + sc.lv[2 * i + 1])));
                    }
                    l += sum;
                    __syncwarp();
                    tmem_st32(t_lane + b * kKeys, w);
                    tc_fence_before();
                    mbar_arrive(&own[kWFull + b]);
                }
            }
            if (!ok) break;
            if (more) {
                if (GROUPS > 0) id = page_at(gn, gn.t0);
                if (kQBufs == 2) rf_next = finish_q(other);
            }
            // ---- the item's output, or its part
            if (!(ok = warp_wait(&own[kPvDone + ((n - 1) & 1u)], ((n - 1) >> 1) & 1u, abort_flag, sp.one_poll))) break;
            tc_fence_after();
            if (more && GROUPS > 0) {
                if (id >= p.c.pages) id = -1;
                scales_of(gn, id, ks, vs);
            }
            const bool whole = g.t0 == 0 && g.t1 == g.tiles;
            const int part = g.t0 > 0 ? 0 : 1;
            const int64_t at0 = ((int64_t) blockIdx.x * 2 + part) * kItemRows + blk * kRows + quarter * 32u;// this warp's first row
            const bool none = wm == -INFINITY;// (O holds products with weights of zero)
            const int64_t out_at = (int64_t) (s.first + tok) * p.o_st + (int64_t) at_q.head * p.o_sh;
            // Through this warp's part of q's memory (rows of 128 bytes, their 16-byte pieces rotated by the row), so that a
            // row's pieces leave side by side: finished outputs 64 columns at a time, parts 32 columns in fp32.
            const uint32_t stage = myq + quarter * 32u * 128u, piece = lane & 7u, sub = lane >> 3;
            auto put = [&](uint32_t i, uint32_t a, uint32_t c, uint32_t d, uint32_t f) {
                asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(stage + lane * 128u + ((i ^ (lane & 7u)) << 4)), "r"(a), "r"(c), "r"(d), "r"(f) : "memory");
            };
            auto take = [&](uint32_t wr) -> uint4 {
                uint4 y;
                asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(y.x), "=r"(y.y), "=r"(y.z), "=r"(y.w) : "r"(stage + wr * 128u + ((piece ^ (wr & 7u)) << 4)) : "memory");
                return y;
            };
            if (whole) {
                const float2 fac = out_factors(p, g.b, limit, l, wm - kLift - m);
                for (int32_t c0 = 0; c0 < p.c.dh; c0 += 64) {
                    float o[64];
                    __syncwarp();
                    tmem_ld64(t_lane + 2 * kKeys + c0, o);
#pragma unroll
                    for (uint32_t i = 0; i < 8; ++i) {
                        uint32_t h[4];
#pragma unroll
                        for (uint32_t j = 0; j < 4; ++j) {
                            const float y0 = o[8 * i + 2 * j], y1 = o[8 * i + 2 * j + 1];
                            h[j] = fac.x == 0.f ? 0u : round16x2(p.bf16, y0 * fac.x * fac.y, y1 * fac.x * fac.y);
                        }
                        put(i, h[0], h[1], h[2], h[3]);
                    }
                    __syncwarp();
                    const int32_t d = c0 + (int32_t) piece * 8;
#pragma unroll
                    for (uint32_t i = 0; i < 8; ++i) {
                        const uint32_t wr = i * 4u + sub, row = rr0 + quarter * 32u + wr;
                        const uint4 y = take(wr);
                        uint16_t *out = p.out + __shfl_sync(0xffffffffu, out_at, (int) wr) + d;
                        if (row < rows && d < p.c.dh) {
                            if (p.o_vec8) {
                                *reinterpret_cast<uint4 *>(out) = y;
                            } else {
                                const uint32_t h[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
                                for (int j = 0; j < 8; ++j) {
                                    if (d + j < p.c.dh) out[j] = (uint16_t) (h[j >> 1] >> (16 * (j & 1)));
                                }
                            }
                        }
                    }
                }
            } else {
                float *parts = sp.parts + at0 * DHC;
                for (int32_t c0 = 0; c0 < p.c.dh; c0 += 32) {
                    float o[32];
                    __syncwarp();
                    tmem_ld32(t_lane + 2 * kKeys + c0, o);
#pragma unroll
                    for (uint32_t i = 0; i < 8; ++i) {
                        if (none) o[4 * i] = o[4 * i + 1] = o[4 * i + 2] = o[4 * i + 3] = 0.f;
                        put(i, __float_as_uint(o[4 * i]), __float_as_uint(o[4 * i + 1]), __float_as_uint(o[4 * i + 2]), __float_as_uint(o[4 * i + 3]));
                    }
                    __syncwarp();
#pragma unroll
                    for (uint32_t i = 0; i < 8; ++i) {
                        const uint32_t wr = i * 4u + sub;
                        const uint4 y = take(wr);
                        if (rr0 + quarter * 32u + wr < rows) *reinterpret_cast<uint4 *>(parts + wr * DHC + c0 + piece * 4u) = y;
                    }
                }
            }
            __syncwarp();
            if (!whole && have) sp.heads[at0 + lane] = PartHead{m, l, wm - kLift, 0};
            if (!whole && part == 1) meta = CtaMeta{g.b, g.kvh, g.rb, (int32_t) divide(g.last_unit, each)};
            tc_fence_before();
            if (kQBufs == 2) {
                buf ^= 1u;
            } else if (more) {
                request_q(gn, myq);
                rf_next = finish_q(myq);
            }
        }
        if (threadIdx.x == 0) sp.meta[blockIdx.x] = meta;
    }

    tc_fence_before();
    __syncthreads();
    asm volatile("griddepcontrol.launch_dependents;");
    if (*abort_flag) {
        // Waits ran out: q may still be on its way, and products that nobody has waited for may be reading tiles and writing
        // TMEM.  Shared memory is the CTA's until its last warp has left, the one that issued them.
        cp_async_wait<0>();
        if (warp == kWarps - 1) {
            umma_commit_by(&bars[kDrained], elect_lane());
            const long long t0 = clock64();
            while (!mbar_try_wait(&bars[kDrained], 0) && clock64() - t0 < kDrainTicks) {}
            __syncwarp();
        }
    }
    if (warp == kWarps - 1) {
        tc_fence_after();
        tmem_dealloc(tmem, kTmemCols);
    }
}

std::atomic<uint32_t> g_wait_polls[64];// per device: 0, or a limit that a test has set

template<int DHC, int GROUPS>
cudaError_t launch_as(const SplitParams &sp, uint32_t ctas, int device_id, cudaStream_t st) {
    static std::atomic<uint64_t> ready{0};// devices on which the shared memory has been asked for
    const uint64_t bit = device_id < 64 ? 1ull << device_id : 0;
    cudaError_t e = cudaSuccess;
    if ((ready.load(std::memory_order_relaxed) & bit) == 0) {
        e = cudaFuncSetAttribute(prefill_kernel<DHC, GROUPS>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int) smem_bytes(DHC));
        if (e != cudaSuccess) return e;
        ready.fetch_or(bit, std::memory_order_relaxed);
    }
    prefill_kernel<DHC, GROUPS><<<ctas, threads_of(blocks_at_once(DHC)), smem_bytes(DHC), st>>>(sp);
    e = cudaGetLastError();
    if (e != cudaSuccess || ctas == 1) return e;
    return launch_join<DHC, blocks_at_once(DHC) * kRows>(sp, ctas, st);
}
template<int DHC>
cudaError_t launch(const AttendParams &a, void *workspace, uint32_t ctas, int device_id, cudaStream_t st) {
    SplitParams sp = split_params(a, workspace, ctas, (uint64_t) prefill_rows(DHC), DHC);
    sp.one_poll = g_wait_polls[device_id & 63].load(std::memory_order_relaxed) != 0;
    if (a.vec && a.c.page % kKeys == 0) return launch_as<DHC, 1>(sp, ctas, device_id, st);
    return a.vec && a.c.page % 16 == 0 ? launch_as<DHC, 4>(sp, ctas, device_id, st) : launch_as<DHC, 0>(sp, ctas, device_id, st);
}

}// namespace

cudaError_t launch_prefill(const AttendParams &a, void *workspace, int dhc, uint32_t ctas, int device_id, cudaStream_t st) {
    return dhc == 64 ? launch<64>(a, workspace, ctas, device_id, st) : dhc == 128 ? launch<128>(a, workspace, ctas, device_id, st)
                                                                                  : launch<256>(a, workspace, ctas, device_id, st);
}

}// namespace paged

void paged_prefill_set_wait_polls(int device_id, unsigned int polls) { paged::g_wait_polls[device_id & 63].store(polls, std::memory_order_relaxed); }

unsigned long long paged_prefill_timeouts_read() {
    unsigned long long v = 0;
    if (cudaMemcpyFromSymbol(&v, tc::g_tc_gemm_timeouts, sizeof(v)) != cudaSuccess) {
        cudaGetLastError();
        return ~0ull;
    }
    return v;
}

}// namespace b200
