// paged_runs.hpp -- which keys of which item a block of attention over a paged
// cache has: the items' units, the runs that they are cut into and the parts
// that a cut leaves, for the kernels and, without a GPU, for the host.
#pragma once

#include <type_traits>

#include "paged_index.hpp"

namespace vvli {

struct Request {
    uint32_t first, vecs;  // first row, vectors of one kv head
    int64_t start;
};

// How a kernel cuts its items: M vectors, steps of WK positions, units of one
// step (FIXED) or of as many as the block's waves take side by side; and in
// units what an item costs beside its keys (its q, the first loads, its end),
// what a cut costs (a part left and taken up again), the fewest of a run, and
// the most of an item that is never cut, since its parts would cost more than
// they save.
template <int M_, int WK_, bool FIXED_, uint32_t ITEM, uint32_t CUT, uint32_t FEWEST, uint32_t WHOLE>
struct Cuts {
    static constexpr int M = M_, WK = WK_;
    static constexpr bool FIXED = FIXED_;
    static constexpr uint32_t kItem = ITEM, kCut = CUT, kFewest = FEWEST, kWhole = WHOLE;
    static_assert(ITEM + (FEWEST / 4 < CUT ? FEWEST / 4 : CUT) < FEWEST, "near_lo + near_hi < per");
};
// Few rows, steps of 16 U keys. (An item at 1 and not 3 units: 24 x 5 rows of heads of 64 40.9 us and not 37.0. Runs from
// 10 units on and not 5: 45.7, and 1 x 1 row behind 2000 positions 26.9 and not 21.0. Items whole up to 24 units and not
// 12: 40 x 1 row behind 8000 102 and not 84; up to none: 1 x 1 row behind 500 15.1 and not 14.3.)
template <int U>
using FewCuts = Cuts<64, 16 * U, false, 3, 4, 5, 12>;
// Chunks. (A step takes two to four times as long in f32, so that the rest costs fewer of them: 100 rows behind 200, heads of
// 128, 55 us at 16 bits' numbers and 35 at these, 3 x 333 rows of heads of 64 42 and 37. What a cut costs, without a
// bound at a quarter of a run: 2 x 2000 rows bf16 317 us, with 4 units 269.)
template <bool F32>
using ChunkCuts = std::conditional_t<F32, Cuts<128, 32, true, 2, 2, 3, 0>, Cuts<128, 32, true, 3, 4, 5, 0>>;

// An item's vectors stand in groups of GV = M / 4, one to a wave: 1, 2 or 4
// waves side by side (the log of that in `wide`) take different vectors, and
// the 4 >> wide such sets take steps of WK positions in turn, (4 WK) >> wide a
// unit. The keys lo .. hi - 1 that some vector of the item sees (hi = 0: none),
// and the units that they touch, behind S::kItem for the item itself.
struct Units {
    uint32_t lo, hi, first, count, wide;
};
// (FIXED: units of WK positions whatever the item. `a` has the call's group, room and window.)
template <class S, class A>
VVLI_HD Units units_of(const A& a, const Request& q, uint32_t m0) {
    const uint32_t left = q.vecs - m0, vecs = left < static_cast<uint32_t>(S::M) ? left : static_cast<uint32_t>(S::M);
    const uint32_t wide = vecs <= S::M / 4 ? 0 : vecs <= S::M / 2 ? 1 : 2;
    const int64_t p0 = q.start + page_of(a.group, m0);
    const int64_t p1 = q.start + page_of(a.group, m0 + vecs - 1);
    const int64_t hi = p1 + 1 < static_cast<int64_t>(a.room) ? p1 + 1 : static_cast<int64_t>(a.room);
    const int64_t lo = a.window && p0 + 1 > a.window ? p0 + 1 - a.window : 0;
    if (hi <= lo) return Units{0, 0, 0, S::kItem, wide};
    const uint32_t unit = S::FIXED ? S::WK : (4 * S::WK) >> wide;
    Units u{static_cast<uint32_t>(lo), static_cast<uint32_t>(hi), static_cast<uint32_t>(lo) / unit, 0, wide};
    u.count = (u.hi + unit - 1) / unit - u.first + S::kItem;
    return u;
}

// (64-bit division is some 150 instructions; sums of units are mostly below 2^32.)
VVLI_HD uint64_t quotient(uint64_t n, uint64_t d) {
    return ((n | d) >> 32) == 0 ? static_cast<uint32_t>(n) / static_cast<uint32_t>(d) : n / d;
}

// Run b holds the units from per * b on to per * (b + 1), but that a border
// within near_lo units of an item's start (anywhere in one of few units) or
// near_hi of its end moves there (near_lo + near_hi < per, so that borders keep
// their order): fewer items are cut, and none before its first keys.
struct Borders {
    uint64_t per;
    uint32_t near_lo, near_hi, runs;
};
template <class S>
VVLI_HD Borders borders_of(uint64_t total, uint32_t blocks) {
    Borders b{};
    const uint64_t even = quotient(total + blocks - 1, blocks);
    b.per = even > S::kFewest ? even : S::kFewest;
    b.near_hi = static_cast<uint32_t>(b.per / 4 < S::kCut ? b.per / 4 : S::kCut);
    b.near_lo = b.near_hi > S::kItem ? b.near_hi : S::kItem;
    b.runs = static_cast<uint32_t>(quotient(total + b.per - 1, b.per));
    return b;
}

// Blocks go to the eight XCDs in turn. Each XCD takes as many runs, side by side: neighbours share keys and table
// rows in its L2, and fewer runs than blocks still have all of the GPU. (A number from `runs` on: no run.)
VVLI_HD uint32_t run_of_block(uint32_t block, uint32_t blocks, uint32_t runs) {
    if (blocks % 8 != 0) return block;
    const uint32_t each = (runs + 7) / 8;
    return block / 8 < each ? block % 8 * each + block / 8 : runs;
}

// What the run that ends at unit `to` has of the item that starts at unit
// `start`, units t0 .. t1 - 1; `begun` if the run starts at unit `unit` inside it
// (taken back where the border has moved to the item's start).
struct Part {
    uint32_t t0, t1;
    bool cut;  // the run ends inside the item
};
enum class Share { kEnd, kNone, kPart };  // the item is the next run's, what is left of it is the last run's, this one has a part
template <class S>
VVLI_HD __attribute__((always_inline)) Share part_of(const Borders& b, const Units& un, uint64_t start, uint64_t to, uint32_t unit,
                                                     bool& begun, Part& p) {
    const uint32_t lo = un.count <= S::kWhole ? un.count - 1 : b.near_lo;
    begun = begun && unit > lo;  // (a border near an item's start is its start)
    if (begun && un.count - unit <= b.near_hi) return Share::kNone;
    if (!begun && to <= start + (lo < un.count - 1 ? lo : un.count - 1)) return Share::kEnd;
    p.t0 = begun ? unit : 0;
    p.cut = to < start + un.count && start + un.count - to > b.near_hi;
    p.t1 = p.cut ? static_cast<uint32_t>(to - start) : un.count;
    return Share::kPart;
}

// Borders inside a cut item, from near_lo behind its start to near_hi before its end: run first_border() - 1 has its
// first part (in its second slot), the runs from first_border() on the others (in their first).
VVLI_HD uint64_t first_border(const Borders& b, uint64_t start) { return quotient(start + b.near_lo, b.per) + 1; }
VVLI_HD uint32_t parts_of(const Borders& b, uint64_t start, uint32_t count) {
    return static_cast<uint32_t>(quotient(start + count - b.near_hi - 1, b.per) - first_border(b, start)) + 2;
}

}  // namespace vvli
