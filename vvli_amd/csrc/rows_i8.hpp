// rows_i8.hpp -- argument checks shared by the ops around 8-bit products.
#pragma once

#include "paged.hpp"
#include "row_bytes.hpp"

namespace vvli {

constexpr uint32_t kCodesPerUnit = 16;  // rows of codes start at, and are padded to, multiples of this

// Rows of `width` elements of `bytes` each, `ld` elements apart, read and written in 16-byte units.
inline int check_row_units(const void* p, uint64_t ld, uint64_t width, uint32_t bytes, const char* what, const char* who) {
    if (!p) return set_error(VVLI_NULL_ARG, "%s: NULL %s", who, what);
    if (ld < width || ld >= kPagedMost || ld * bytes % 16 != 0 || !aligned16(p))
        return set_error(VVLI_INVALID_CONFIG, "%s: rows of %s (stride %llu) are not whole 16-byte units", who, what,
                         static_cast<unsigned long long>(ld));
    return VVLI_OK;
}

}  // namespace vvli
