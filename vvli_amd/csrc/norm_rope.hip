// norm_rope.hip -- RMS norm of every q and k head, rotation by the row's
// position and the append of k and v to the paged cache, in one pass over a
// projection's rows (vvli_gpu_norm_rope_append).
//
// y = x * (mean(x^2) + eps)^(-1/2) * w, then each pair (a, b) of a head turns
// by pos * inv_freq[i]: (a cos - b sin, b cos + a sin). Nothing is reused
// between rows, so memory bounds it: 6000 rows of 28 + 8 heads of 128 into an
// f16 cache 47.7 us, 4.4 TB/s, 20000 rows 140 us, 5.0 TB/s (a copy reaches 4.8
// to 5.4); 75 rows 5.5 us and 1 row 5.4 us are a launch and its chain of loads.
//
// A wave takes heads of one row: HD / 4 lanes a head, 4 values a lane, as many
// heads side by side as fit. A lane's values are two pairs, the same ones in
// every head, so that it forms their sine and cosine once for all heads of its
// row.
#include <hip/hip_fp16.h>

#include <algorithm>

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
    uint32_t rows, heads, kv_heads, chunks;
    bool split, weight_bf16;
    float eps;
};

__device__ inline float norm_weight(const void* w, bool bf16, uint32_t i) {
    return bf16 ? __uint_as_float(static_cast<uint32_t>(static_cast<const uint16_t*>(w)[i]) << 16) : static_cast<const float*>(w)[i];
}

// Sine and cosine of pos * f: the angle in 64 bits, turns taken off there
// (2 pi in two doubles: 106 bits, so that what is left is exact to f32 for any
// 31-bit position), then f32 (rows of an f32 cache are off by 5.9e-8 in the
// 2-norm, where sine and cosine in 64 bits would leave 4.2e-8).
__device__ inline void turn(int32_t pos, float f, float& c, float& s) {
    constexpr double kHi = 6.283185307179586, kLo = 2.4492935982947064e-16, kInv = 0.15915494309189535;
    const double t = static_cast<double>(pos) * static_cast<double>(f), n = rint(t * kInv);
    sincosf(static_cast<float>(fma(-n, kLo, fma(-n, kHi, t))), &s, &c);
}

template <typename T>
__device__ inline void put2(T* p, float x, float y) {
    typedef T T2 __attribute__((ext_vector_type(2)));
    *reinterpret_cast<T2*>(p) = T2{static_cast<T>(x), static_cast<T>(y)};
}
template <typename T>
__device__ inline void put4(T* p, const float (&x)[4]) {
    typedef T T4 __attribute__((ext_vector_type(4)));
    *reinterpret_cast<T4*>(p) = T4{static_cast<T>(x[0]), static_cast<T>(x[1]), static_cast<T>(x[2]), static_cast<T>(x[3])};
}

constexpr int kThreads = 256;
constexpr uint32_t kRowsMost = 1u << 26;  // a wave a row: a launch takes fewer than 2^32 threads

// Wave w of the grid: row w / chunks, turns w % chunks, + chunks, ... of the row's heads.
template <int HD, typename T, bool SPLIT>
__global__ __launch_bounds__(kThreads) void norm_rope_kernel(NormRopeArgs a) {
    constexpr int L = HD / 4, SIDE = 64 / L, N = 4;  // lanes of a head, heads side by side, turns in flight
    const uint64_t w = static_cast<uint64_t>(blockIdx.x) * (kThreads / 64) + threadIdx.x / 64;
    const uint32_t row = static_cast<uint32_t>(w / a.chunks), chunk = static_cast<uint32_t>(w % a.chunks);
    if (row >= a.rows) return;
    const uint32_t lane = threadIdx.x & 63, i = lane % L, side = lane / L;
    const uint32_t at0 = SPLIT ? 2 * i : 4 * i, at1 = SPLIT ? HD / 2 + 2 * i : 4 * i + 2;  // values at0, at0 + 1, at1, at1 + 1
    const uint32_t heads = a.heads + 2 * a.kv_heads, turned = a.heads + a.kv_heads;
    const int64_t slot = a.slots[row];
    const bool append = slot >= 0 && static_cast<uint64_t>(slot) < a.n_slots;
    const uint64_t cache_at = append ? static_cast<uint64_t>(slot) * a.slot_stride : 0;
    const float *qr = a.q + row * a.ldq, *kr = a.k + row * a.ldk, *vr = a.v + row * a.ldv;
    float c0 = 1, s0 = 0, c1 = 1, s1 = 0;
    const int32_t pos = a.pos[row];
    turn(pos, a.inv_freq[2 * i], c0, s0);
    turn(pos, a.inv_freq[2 * i + 1], c1, s1);
    float qw[4], kw[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const uint32_t at = e < 2 ? at0 + e : at1 + e - 2;
        qw[e] = a.q_norm ? norm_weight(a.q_norm, a.weight_bf16, at) : 1.f;
        kw[e] = a.k_norm ? norm_weight(a.k_norm, a.weight_bf16, at) : 1.f;
    }
    const uint32_t step = a.chunks * SIDE;
    for (uint32_t h0 = chunk * SIDE + side; h0 - side < heads; h0 += N * step) {
        float x[N][4];
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const uint32_t h = h0 + n * step;
            const float* p = h < a.heads ? qr + static_cast<size_t>(h) * HD
                             : h < turned ? kr + static_cast<size_t>(h - a.heads) * HD
                                          : vr + static_cast<size_t>(h - turned) * HD;
            if (h < heads) {
                if constexpr (SPLIT) {
                    const uint2 u = load_u32x2(p + at0), v = load_u32x2(p + at1);
                    x[n][0] = __uint_as_float(u.x), x[n][1] = __uint_as_float(u.y);
                    x[n][2] = __uint_as_float(v.x), x[n][3] = __uint_as_float(v.y);
                } else {
                    const float4 u = load_f32x4(p + at0);
                    x[n][0] = u.x, x[n][1] = u.y, x[n][2] = u.z, x[n][3] = u.w;
                }
            } else {
                x[n][0] = x[n][1] = x[n][2] = x[n][3] = 0.f;
            }
        }
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const uint32_t h = h0 + n * step;
            const bool is_q = h < a.heads, is_v = h >= turned;
            float ss = x[n][0] * x[n][0] + x[n][1] * x[n][1] + (x[n][2] * x[n][2] + x[n][3] * x[n][3]);
#pragma unroll
            for (int o = 1; o < L; o <<= 1) ss += __shfl_xor(ss, o, 64);  // (every lane of the wave is here)
            if (h >= heads) continue;
            if (!is_v) {
                if (is_q ? a.q_norm != nullptr : a.k_norm != nullptr) {
                    const float inv = 1.0f / sqrtf(ss / HD + a.eps);
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[n][e] = x[n][e] * inv * (is_q ? qw[e] : kw[e]);
                }
                // Pairs: split (x0, x2) and (x1, x3), interleaved (x0, x1) and (x2, x3), pair 2 i and 2 i + 1.
                float &a0 = x[n][0], &b0 = x[n][SPLIT ? 2 : 1], &a1 = x[n][SPLIT ? 1 : 2], &b1 = x[n][3];
                const float y0 = a0 * c0 - b0 * s0, z0 = b0 * c0 + a0 * s0, y1 = a1 * c1 - b1 * s1, z1 = b1 * c1 + a1 * s1;
                a0 = y0, b0 = z0, a1 = y1, b1 = z1;
            }
            if (is_q) {
                float* o = a.q_out + row * a.ldo + static_cast<size_t>(h) * HD;
                if constexpr (SPLIT) put2(o + at0, x[n][0], x[n][1]), put2(o + at1, x[n][2], x[n][3]);
                else put4(o + at0, x[n]);
            } else if (append) {
                T* o = static_cast<T*>(is_v ? a.vc : a.kc) + cache_at + static_cast<size_t>(is_v ? h - turned : h - a.heads) * HD;
                if constexpr (SPLIT) put2(o + at0, x[n][0], x[n][1]), put2(o + at1, x[n][2], x[n][3]);
                else put4(o + at0, x[n]);
            }
        }
    }
}

template <int HD, typename T>
hipError_t launch(NormRopeArgs& a, hipStream_t s) {
    // Waves of a row: one where the rows alone fill the GPU (a wave's angles then serve all heads of the row),
    // more down to a wave for each turn where they do not. (Waves for 16 a CU: 1000 rows 11.5 us, 2000 15.7; for
    // 64 a CU 15.5 and 18.2. 300 and 6000 rows take the same with either.)
    constexpr uint32_t SIDE = 256 / HD;
    const uint32_t turns = (a.heads + 2 * a.kv_heads + SIDE - 1) / SIDE;
    const uint32_t fill = gemm_cus() * 16;
    a.chunks = std::min(turns, std::max(1u, fill / a.rows));
    const uint64_t blocks = (static_cast<uint64_t>(a.rows) * a.chunks + kThreads / 64 - 1) / (kThreads / 64);
    const dim3 grid(static_cast<uint32_t>(blocks)), block(kThreads);
    return a.split ? vlaunch(norm_rope_kernel<HD, T, true>, grid, block, 0, s, a)
                   : vlaunch(norm_rope_kernel<HD, T, false>, grid, block, 0, s, a);
}

template <int HD>
hipError_t launch(NormRopeArgs& a, uint32_t kind, hipStream_t s) {
    return kind == VVLI_CACHE_F32 ? launch<HD, float>(a, s)
           : kind == VVLI_CACHE_BF16 ? launch<HD, __bf16>(a, s)
                                     : launch<HD, _Float16>(a, s);
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
    if (heads == 0 || heads + 2ull * cache->kv_heads > 65535 || rows >= kRowsMost || rope_layout > VVLI_ROPE_SPLIT_HALF ||
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
    NormRopeArgs a{};
    a.q = q, a.k = k, a.v = v, a.inv_freq = inv_freq, a.q_out = q_out, a.pos = pos, a.slots = slots, a.q_norm = q_norm, a.k_norm = k_norm;
    a.kc = cache->k, a.vc = cache->v, a.ldq = ldq, a.ldk = ldk, a.ldv = ldv, a.ldo = ldo, a.slot_stride = cache->slot_stride;
    a.n_slots = static_cast<uint64_t>(cache->pages) * cache->page_size, a.rows = rows, a.heads = heads, a.kv_heads = cache->kv_heads;
    a.split = rope_layout == VVLI_ROPE_SPLIT_HALF, a.weight_bf16 = weight_kind == VVLI_WEIGHT_BF16, a.eps = eps;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    PAGED_TRY(cache->head_dim == 128 ? launch<128>(a, cache->kind, s)
              : cache->head_dim == 64 ? launch<64>(a, cache->kind, s)
                                      : launch<32>(a, cache->kind, s));
    return VVLI_OK;
}
