// row_bytes.hpp -- whether rows of two arguments share memory: host arithmetic
// behind the refusals of the ops around 8-bit products.
#pragma once

#include <stdint.h>

namespace vvli {

// Bytes that `rows` rows touch: `width` bytes at every `ld`-th.
struct RowBytes {
    const void* p;
    uint64_t ld, width, rows;
};

// Whether two sets of rows share a byte. Rows of the same stride may lie beside each other (the halves of one
// product's rows): then they share one exactly if their distance, modulo the stride, puts one row's bytes into
// another's. Rows of different strides are taken to share bytes where their ranges meet.
inline bool rows_meet(const RowBytes& a, const RowBytes& b) {
    if (!a.p || !b.p || !a.rows || !b.rows || !a.width || !b.width) return false;
    const uint64_t pa = reinterpret_cast<uintptr_t>(a.p), pb = reinterpret_cast<uintptr_t>(b.p);
    const uint64_t ea = pa + (a.rows - 1) * a.ld + a.width, eb = pb + (b.rows - 1) * b.ld + b.width;
    if (pa >= eb || pb >= ea) return false;
    if (a.ld != b.ld) return true;
    const bool up = pb >= pa;  // the later start, relative to the rows of the earlier
    const uint64_t at = (up ? pb - pa : pa - pb) % a.ld, first = up ? a.width : b.width, second = up ? b.width : a.width;
    return at < first || at + second > a.ld;
}

}  // namespace vvli
