// paged.hpp -- argument checks shared by the ops over a paged cache.
#pragma once

#include <hip/hip_runtime.h>

#include <cmath>

#include "internal.hpp"
#include "kernels.hpp"
#include "paged_index.hpp"

namespace vvli {

#define PAGED_TRY(expr)                                                                                \
    do {                                                                                               \
        const hipError_t e_ = (expr);                                                                  \
        if (e_ != hipSuccess) return set_error(VVLI_HIP_ERROR, "%s: %s", #expr, hipGetErrorString(e_)); \
    } while (0)

constexpr uint64_t kPagedMost = uint64_t{1} << 31;  // slots, positions and table entries are below this

inline bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

inline int check_cache(const vvli_gpu_paged_cache* c, const char* who) {
    if (!c || !c->k || !c->v) return set_error(VVLI_NULL_ARG, "%s: NULL cache", who);
    if (c->kind > VVLI_CACHE_F16) return set_error(VVLI_INVALID_CONFIG, "%s: unknown cache kind %u", who, c->kind);
    const uint32_t e = c->kind == VVLI_CACHE_F32 ? 4 : 2;
    if (c->head_dim != 32 && c->head_dim != 64 && c->head_dim != 128)
        return set_error(VVLI_INVALID_CONFIG, "%s: head_dim %u is not 32, 64 or 128", who, c->head_dim);
    if (c->kv_heads == 0 || c->kv_heads > 65535 || c->page_size == 0 || c->pages == 0 ||
        static_cast<uint64_t>(c->page_size) * c->pages >= kPagedMost)
        return set_error(VVLI_INVALID_CONFIG, "%s: bad cache of %u pages of %u slots, %u heads", who, c->pages,
                         c->page_size, c->kv_heads);
    if (c->slot_stride < static_cast<uint64_t>(c->kv_heads) * c->head_dim || c->slot_stride >= kPagedMost ||
        c->slot_stride * e % 16 != 0 || !aligned16(c->k) || !aligned16(c->v))
        return set_error(VVLI_INVALID_CONFIG, "%s: the cache's slots are not whole 16-byte units (stride %llu)", who,
                         static_cast<unsigned long long>(c->slot_stride));
    return VVLI_OK;
}

// f32 rows of `width` values, `ld` apart, read and written in 16-byte units.
inline int check_rows(const void* p, uint64_t ld, uint64_t width, const char* what, const char* who) {
    if (!p) return set_error(VVLI_NULL_ARG, "%s: NULL %s", who, what);
    if (ld < width || ld >= kPagedMost || ld % 4 != 0 || !aligned16(p))
        return set_error(VVLI_INVALID_CONFIG, "%s: rows of %s (stride %llu) are not whole 16-byte units", who, what,
                         static_cast<unsigned long long>(ld));
    return VVLI_OK;
}

}  // namespace vvli
