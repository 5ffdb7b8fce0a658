// norm_rope.hip -- RMS norm of every q and k head, rotation by the row's
// position and the append of k and v to the paged cache, in one pass over a
// projection's rows (vvli_gpu_norm_rope_append).
//
// y = x * (mean(x^2) + eps)^(-1/2) * w, then each pair (a, b) of a head turns
// by pos * inv_freq[i]: (a cos - b sin, b cos + a sin). Nothing is reused
// between rows, so memory bounds it.
#include <hip/hip_fp16.h>

#include "device_common.hpp"
#include "paged.hpp"

using namespace vvli;

namespace {

struct NormRopeArgs {
    const float *q, *k, *v, *inv_freq;
    float* q_out;
    const int32_t* pos;
    const int64_t* slots;
    const void *q_norm, *k_norm;
    void *kc, *vc;
    uint64_t ldq, ldk, ldv, ldo, slot_stride, n_slots;
    uint32_t rows, heads, kv_heads;
    bool split, weight_bf16;
    float eps;
};

__device__ inline float norm_weight(const void* w, bool bf16, uint32_t i) {
    return bf16 ? __uint_as_float(static_cast<uint32_t>(static_cast<const uint16_t*>(w)[i]) << 16) : static_cast<const float*>(w)[i];
}

template <typename T> __device__ inline T cache_value(float x) { return static_cast<T>(x); }

// One wave per head: lane l holds the pair l of it (head_dim / 2 lanes).
template <int HD, typename T>
__global__ __launch_bounds__(64) void norm_rope_kernel(NormRopeArgs a) {
    constexpr int P = HD / 2;
    const uint32_t row = blockIdx.x, h = blockIdx.y, lane = threadIdx.x;
    if (lane >= P) return;
    const bool is_q = h < a.heads, is_k = !is_q && h < a.heads + a.kv_heads;
    const uint32_t kvh = is_q ? 0 : is_k ? h - a.heads : h - a.heads - a.kv_heads;
    const float* x = is_q ? a.q + row * a.ldq + static_cast<size_t>(h) * HD
                          : (is_k ? a.k + row * a.ldk : a.v + row * a.ldv) + static_cast<size_t>(kvh) * HD;
    const uint32_t i0 = a.split ? lane : 2 * lane, i1 = a.split ? lane + P : 2 * lane + 1;
    float x0 = x[i0], x1 = x[i1];
    if (is_q || is_k) {
        const void* w = is_q ? a.q_norm : a.k_norm;
        if (w) {
            float ss = x0 * x0 + x1 * x1;
            for (int o = P / 2; o; o >>= 1) ss += __shfl_xor(ss, o, 64);
            const float inv = 1.0f / sqrtf(ss / HD + a.eps);
            x0 = x0 * inv * norm_weight(w, a.weight_bf16, i0);
            x1 = x1 * inv * norm_weight(w, a.weight_bf16, i1);
        }
        double s, c;
        sincos(static_cast<double>(a.pos[row]) * static_cast<double>(a.inv_freq[lane]), &s, &c);
        const float cf = static_cast<float>(c), sf = static_cast<float>(s);
        const float y0 = x0 * cf - x1 * sf, y1 = x1 * cf + x0 * sf;
        x0 = y0, x1 = y1;
    }
    if (is_q) {
        float* o = a.q_out + row * a.ldo + static_cast<size_t>(h) * HD;
        o[i0] = x0, o[i1] = x1;
        return;
    }
    const int64_t slot = a.slots[row];
    if (slot < 0 || static_cast<uint64_t>(slot) >= a.n_slots) return;
    T* o = static_cast<T*>(is_k ? a.kc : a.vc) + static_cast<uint64_t>(slot) * a.slot_stride + static_cast<size_t>(kvh) * HD;
    o[i0] = cache_value<T>(x0), o[i1] = cache_value<T>(x1);
}

template <int HD>
hipError_t launch(const NormRopeArgs& a, uint32_t kind, hipStream_t s) {
    const dim3 grid(a.rows, a.heads + 2 * a.kv_heads), block(64);
    if (kind == VVLI_CACHE_F32) return vlaunch(norm_rope_kernel<HD, float>, grid, block, 0, s, a);
    if (kind == VVLI_CACHE_BF16) return vlaunch(norm_rope_kernel<HD, __bf16>, grid, block, 0, s, a);
    return vlaunch(norm_rope_kernel<HD, _Float16>, grid, block, 0, s, a);
}

}  // namespace

extern "C" int vvli_gpu_norm_rope_append(const vvli_gpu_paged_cache* cache, const float* q, uint64_t ldq, const float* k,
                                         uint64_t ldk, const float* v, uint64_t ldv, uint32_t rows, uint32_t heads,
                                         float* q_out, uint64_t ldo, const float* inv_freq, const int32_t* pos,
                                         const int64_t* slots, uint32_t rope_layout, const void* q_norm,
                                         const void* k_norm, uint32_t weight_kind, float eps, void* stream) {
    const char* who = "vvli_gpu_norm_rope_append";
    int rc = check_cache(cache, who);
    if (rc) return rc;
    if (!inv_freq || !pos || !slots) return set_error(VVLI_NULL_ARG, "NULL argument to %s", who);
    const uint64_t hd = cache->head_dim, wq = heads * hd, wk = cache->kv_heads * hd;
    if (heads == 0 || heads + 2ull * cache->kv_heads > 65535 || rows >= kPagedMost || rope_layout > VVLI_ROPE_SPLIT_HALF ||
        weight_kind > VVLI_WEIGHT_BF16)
        return set_error(VVLI_INVALID_CONFIG, "%s: bad sizes (%u rows, %u heads, layout %u, weight kind %u)", who, rows, heads,
                         rope_layout, weight_kind);
    if ((q_norm || k_norm) && !(eps >= 0.f && std::isfinite(eps)))
        return set_error(VVLI_INVALID_CONFIG, "%s: eps %g", who, static_cast<double>(eps));
    if ((rc = check_rows(q, ldq, wq, "q", who)) || (rc = check_rows(k, ldk, wk, "k", who)) ||
        (rc = check_rows(v, ldv, wk, "v", who)) || (rc = check_rows(q_out, ldo, wq, "q_out", who)))
        return rc;
    if (q_out == q && ldo != ldq) return set_error(VVLI_INVALID_CONFIG, "%s: q_out is q with another stride", who);
    if (rows == 0) return VVLI_OK;
    NormRopeArgs a{q,    k,        v,     inv_freq, q_out,           pos,
                   slots, q_norm,  k_norm, cache->k, cache->v,        ldq,
                   ldk,  ldv,      ldo,   cache->slot_stride, static_cast<uint64_t>(cache->pages) * cache->page_size, rows,
                   heads, cache->kv_heads, rope_layout == VVLI_ROPE_SPLIT_HALF, weight_kind == VVLI_WEIGHT_BF16, eps};
    const hipStream_t s = static_cast<hipStream_t>(stream);
    PAGED_TRY(cache->head_dim == 128 ? launch<128>(a, cache->kind, s)
              : cache->head_dim == 64 ? launch<64>(a, cache->kind, s)
                                      : launch<32>(a, cache->kind, s));
    return VVLI_OK;
}
