// linear_i8.hip -- the product of rows of 8-bit codes, a scale for each row of
// both sides (vvli_gpu_linear_i8):
//   Y[m,n] = f32(sum_k W[n,k] X[m,k]) * x_scales[m] * w_scales[n] + bias[n].
//
// The sums are exact in 32 bits, so no split or order of them changes a result.
#include <algorithm>

#include "device_common.hpp"
#include "rows_i8.hpp"

using namespace vvli;

namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));

struct LinearI8Args {
    const int8_t *W, *X;
    const float *w_scales, *x_scales;
    const uint16_t* bias;
    float* Y;
    uint64_t ldw, ldx, ldy;
    uint32_t M, N, K;
};

constexpr uint32_t kMostK = 131056;  // 131056 * 128 * 128 < 2^31

__device__ __forceinline__ float finish(int sum, float x_scale, float w_scale, float bias) {
#pragma clang fp contract(off)
    return static_cast<float>(sum) * x_scale * w_scale + bias;  // each rounded: no multiply-add
}

// A wave 16 rows of W times 16 of X, operands straight from memory: lane l
// holds row l % 16, codes 16 (l / 16) .. + 15 of a step of 64, of both; output
// column (row of X) l % 16, rows 4 (l / 16) .. + 3.
__global__ __launch_bounds__(256) void linear_i8_kernel(LinearI8Args a) {
    const uint32_t lane = threadIdx.x & 63, tn = (a.N + 15) / 16, tm = (a.M + 15) / 16;
    const uint64_t tiles = static_cast<uint64_t>(tn) * tm;
    for (uint64_t t = blockIdx.x * 4ull + threadIdx.x / 64; t < tiles; t += gridDim.x * 4ull) {
    const uint32_t n0 = static_cast<uint32_t>(t % tn) * 16, m0 = static_cast<uint32_t>(t / tn) * 16;
    const uint32_t n = min(n0 + lane % 16, a.N - 1), m = min(m0 + lane % 16, a.M - 1);
    const int8_t *w = a.W + n * a.ldw, *x = a.X + m * a.ldx;
    i32x4 sum = {0, 0, 0, 0};
    for (uint32_t k = lane / 16 * 16; k - lane / 16 * 16 < a.K; k += 64) {
        const i32x4 zero = {0, 0, 0, 0};
        const i32x4 p = k < a.K ? *reinterpret_cast<const i32x4*>(w + k) : zero, q = k < a.K ? *reinterpret_cast<const i32x4*>(x + k) : zero;
        sum = __builtin_amdgcn_mfma_i32_16x16x64_i8(p, q, sum, 0, 0, 0);
    }
    if (m0 + lane % 16 >= a.M) continue;
#pragma unroll
    for (uint32_t j = 0; j < 4; ++j) {
        const uint32_t row = n0 + lane / 16 * 4 + j;
        if (row < a.N)
            a.Y[m * a.ldy + row] = finish(sum[j], a.x_scales[m], a.w_scales[row],
                                          a.bias ? __uint_as_float(static_cast<uint32_t>(a.bias[row]) << 16) : 0.f);
    }
    }
}

bool sizes_ok(uint32_t M, uint32_t N, uint32_t K) {
    return M < kPagedMost && N > 0 && N < kPagedMost && K > 0 && K <= kMostK && K % kCodesPerUnit == 0;
}

}  // namespace

extern "C" {

size_t vvli_gpu_linear_i8_workspace(uint32_t M, uint32_t N, uint32_t K) { return sizes_ok(M, N, K) ? 16 : 0; }

int vvli_gpu_linear_i8(const int8_t* W, uint64_t ldw, const float* w_scales, const int8_t* X, uint64_t ldx,
                       const float* x_scales, const uint16_t* bias, float* Y, uint64_t ldy, uint32_t M, uint32_t N,
                       uint32_t K, void* workspace, size_t workspace_bytes, void* stream) {
    const char* who = "vvli_gpu_linear_i8";
    if (!W || !w_scales || !X || !x_scales || !Y || !workspace) return set_error(VVLI_NULL_ARG, "NULL argument to %s", who);
    if (!sizes_ok(M, N, K))
        return set_error(VVLI_INVALID_CONFIG, "%s: bad sizes M=%u N=%u K=%u (K: whole 16s up to %u)", who, M, N, K, kMostK);
    int rc;
    if ((rc = check_row_units(W, ldw, K, 1, "W", who)) || (rc = check_row_units(X, ldx, K, 1, "X", who))) return rc;
    if (ldy < N || ldy >= kPagedMost)
        return set_error(VVLI_INVALID_CONFIG, "%s: rows of Y of %u (stride %llu)", who, N, static_cast<unsigned long long>(ldy));
    if (!aligned16(workspace) || workspace_bytes < vvli_gpu_linear_i8_workspace(M, N, K))
        return set_error(VVLI_INVALID_CONFIG, "%s: workspace of %zu bytes", who, workspace_bytes);
    const RowBytes y{Y, ldy * 4, uint64_t{N} * 4, M};
    if (rows_meet(y, RowBytes{W, ldw, K, N}) || rows_meet(y, RowBytes{X, ldx, K, M}) || rows_meet(y, RowBytes{w_scales, 4, 4, N}) ||
        rows_meet(y, RowBytes{x_scales, 4, 4, M}) || rows_meet(y, RowBytes{bias, 2, 2, N}) ||
        rows_meet(y, RowBytes{workspace, workspace_bytes, workspace_bytes, 1}))
        return set_error(VVLI_INVALID_CONFIG, "%s: Y overlaps another argument", who);
    if (M == 0) return VVLI_OK;
    LinearI8Args a{};
    a.W = W, a.X = X, a.w_scales = w_scales, a.x_scales = x_scales, a.bias = bias, a.Y = Y;
    a.ldw = ldw, a.ldx = ldx, a.ldy = ldy, a.M = M, a.N = N, a.K = K;
    const uint64_t tiles = (uint64_t{N} + 15) / 16 * ((uint64_t{M} + 15) / 16);
    PAGED_TRY(vlaunch(linear_i8_kernel, dim3(static_cast<uint32_t>(std::min<uint64_t>((tiles + 3) / 4, 1u << 20))), dim3(256), 0, static_cast<hipStream_t>(stream), a));
    return VVLI_OK;
}

}  // extern "C"
