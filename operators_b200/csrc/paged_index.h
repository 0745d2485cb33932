// Index arithmetic of the paged KV cache that host and device code share: which rows of the new tokens belong to a
// sequence, which pages they touch, and the power of two that scales a block of codes.  Everything read from a
// device array (lengths, offsets, page ids) is clamped or checked here, so that no value of theirs leads out of a
// tensor.  Plain C++: the CPU tests compile it with g++.
#pragma once

#include <stdint.h>

#ifdef __CUDACC__
#define B200_HD __host__ __device__ __forceinline__
#else
#define B200_HD inline
#endif

namespace b200 {
namespace paged {

// One sequence of a call.  Its new tokens are rows first .. first + n of k, v, q and out; token i of them stands at
// position len - n + i of the sequence (negative: the token exists but has no place in the cache and sees nothing).
struct Seq {
    int32_t first, n, len;
};

// `offs` == nullptr: one new token per sequence.  `rows` = new tokens of the call (rows of q / k).
B200_HD Seq seq_of(const int32_t *lens, const int32_t *offs, int32_t rows, int32_t b) {
    Seq s;
    int32_t lo = b, hi = b + 1;
    if (offs != nullptr) {
        lo = offs[b], hi = offs[b + 1];
        lo = lo < 0 ? 0 : lo > rows ? rows : lo;
        hi = hi < 0 ? 0 : hi > rows ? rows : hi;
    }
    s.first = lo;
    s.n = hi > lo ? hi - lo : 0;
    s.len = lens[b] > 0 ? lens[b] : 0;
    return s;
}

// Cached tokens that the block table can hold of a sequence: `cap` = table columns x page size.
B200_HD int32_t held(int32_t len, int32_t cap) { return len < cap ? len : cap; }

// The positions of a sequence that an append writes, [lo, hi): the new tokens that have a place in the table.
B200_HD void written(const Seq &s, int32_t cap, int32_t &lo, int32_t &hi) {
    lo = s.len > s.n ? s.len - s.n : 0;
    hi = held(s.len, cap);
}
// Pages that [lo, hi) touches; page_of(token) is a token's column of the table.
template<class PageOf>
B200_HD int32_t pages_touched(int32_t lo, int32_t hi, const PageOf &page_of) {
    return hi > lo ? page_of(hi - 1) - page_of(lo) + 1 : 0;
}
// More pages than all appends of a call can touch: m tokens touch at most m pages, and at most m / page + 2.
B200_HD int64_t pages_bound(int64_t rows, int64_t batch, int64_t page) {
    const int64_t b = rows / page + 2 * batch;
    return b < rows ? b : rows;
}

// Exponent of the scale of a block whose largest finite magnitude is 1.m x 2^e (fp32 bits of it): the smallest x
// with amax <= 448 x 2^x = 1.75 x 2^(x + 8), not below kMinExp (blocks of zeros; what is below 2^(kMinExp - 10) is
// stored as zero).  fp32 subnormals lie far below and need no care.
constexpr int32_t kMinExp = -40;
B200_HD int32_t scale_exponent(uint32_t amax_bits) {
    const int32_t e = (int32_t) (amax_bits >> 23) - 127, x = (amax_bits & 0x7FFFFFu) <= 0x600000u ? e - 8 : e - 7;
    return x < kMinExp ? kMinExp : x;
}
// 2^x, -126 <= x <= 127, as fp32 bits
B200_HD uint32_t pow2_bits(int32_t x) { return (uint32_t) (x + 127) << 23; }

}// namespace paged
}// namespace b200
