// paged_index.hpp -- which page, slot and row something is in: the index
// arithmetic of the ops over a paged cache, for the kernels and, without a
// GPU, for the host.
#pragma once

#include <stdint.h>

#if defined(__HIPCC__)
#define VVLI_HD __host__ __device__ inline
#else
#define VVLI_HD inline
#endif

namespace vvli {

// n / d for n < 2^31 by a product: with s = ceil(log2 d) and
// m = floor(2^(31+s) / d) + 1, m d - 2^(31+s) lies in 1..2^s, which makes
// floor(n m / 2^(31+s)) exact for every n below 2^31. (m < 2^32 + 1: the
// quotient is below 2^32 unless d is a power of two, where it is 2^31.)
struct PageDiv {
    uint32_t d, m, shift;
};
VVLI_HD PageDiv page_div(uint32_t d) {
    uint32_t s = 0;
    while ((uint64_t{1} << s) < d) ++s;
    return PageDiv{d, static_cast<uint32_t>((uint64_t{1} << (31 + s)) / d + 1), 31 + s};
}
VVLI_HD uint32_t page_of(const PageDiv& p, uint32_t n) {
    return static_cast<uint32_t>((static_cast<uint64_t>(n) * p.m) >> p.shift);
}
VVLI_HD uint32_t pages_for(const PageDiv& p, uint32_t tokens) { return tokens ? page_of(p, tokens - 1) + 1 : 0; }

// Slot of position `pos` through a request's row of the table; -1 behind the
// row's end or where it names no page of the cache.
VVLI_HD int32_t page_slot(const int32_t* row, uint32_t stride, uint32_t pages, const PageDiv& p, uint32_t pos) {
    const uint32_t i = page_of(p, pos);
    if (i >= stride) return -1;
    const uint32_t page = static_cast<uint32_t>(row[i]);
    return page < pages ? static_cast<int32_t>(page * p.d + (pos - i * p.d)) : -1;
}

// Rows first .. first + count - 1 of request r, whatever row_start holds.
struct RowSpan {
    uint32_t first, count;
};
VVLI_HD RowSpan row_span(int32_t begin, int32_t end, uint32_t rows) {
    const int64_t n = rows, b = begin < 0 ? 0 : begin > n ? n : begin, e = end < b ? b : end > n ? n : end;
    return RowSpan{static_cast<uint32_t>(b), static_cast<uint32_t>(e - b)};
}

// Keys that a row at position pos sees: lo .. hi - 1 (empty: lo = hi = 0);
// `room` = positions that the table has.
struct KeySpan {
    uint32_t lo, hi;
};
VVLI_HD KeySpan key_span(int64_t pos, uint32_t window, uint32_t room) {
    if (pos < 0) return KeySpan{0, 0};
    const int64_t hi = pos + 1 < room ? pos + 1 : room;
    const int64_t lo = window && pos + 1 > window ? pos + 1 - window : 0;
    return lo < hi ? KeySpan{static_cast<uint32_t>(lo), static_cast<uint32_t>(hi)} : KeySpan{0, 0};
}

}  // namespace vvli
