// rows_i8.hip -- rows in 8 bits with a scale each: of given rows
// (vvli_gpu_quantize_rows), of a residual's sum behind its RMS norm
// (vvli_gpu_add_norm) and of a gated activation (vvli_gpu_silu_mul).
//
// scale = f32(max |v| / 127), code = rint(v / scale). Which code a value near
// a border between two gets follows its 64-bit value, so that codes do not
// change with the order of a row's sums.
#include <algorithm>

#include "device_common.hpp"
#include "rows_i8.hpp"

using namespace vvli;

namespace {

enum { kRowsF32 = 0, kRowsBf16 = 1, kRowsNorm = 2, kRowsGate = 3 };

struct RowsArgs {
    const void *x, *weight;  // x: rows, or gate
    const float* b;          // delta or up (NULL: none)
    float *sum, *y, *scales;
    int8_t* codes;
    uint64_t ldx, ldb, lds, ldy, ldc;  // elements
    uint32_t rows, width;
    bool weight_bf16;
    float eps;
};

__device__ __forceinline__ float bf16_at(const void* p, size_t i) {
    return __uint_as_float(static_cast<uint32_t>(static_cast<const uint16_t*>(p)[i]) << 16);
}

constexpr int kThreads = 1024, kWaves = kThreads / 64;

// The sum of a block's values, in an order that does not change.
__device__ __forceinline__ double block_sum(double v, double (&part)[kWaves]) {
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o, 64);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0;
    for (int i = 0; i < kWaves; ++i) v += part[i];
    return v;
}
// The largest; NaN if a value is NaN.
__device__ __forceinline__ double larger(double a, double b) { return a >= b || a != a ? a : b; }
__device__ __forceinline__ double block_max(double v, double (&part)[kWaves]) {
    for (int o = 32; o; o >>= 1) v = larger(v, __shfl_xor(v, o, 64));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    v = part[0];
    for (int i = 1; i < kWaves; ++i) v = larger(v, part[i]);
    return v;
}

// A block a row, two passes over it.
template <int OP>
__global__ __launch_bounds__(kThreads) void rows_i8_kernel(RowsArgs a) {
    __shared__ double part[kWaves];
    for (uint32_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const float* x = static_cast<const float*>(a.x) + row * a.ldx;
        const float* b = a.b ? a.b + row * a.ldb : nullptr;
        auto weight = [&](uint32_t e) { return a.weight_bf16 ? bf16_at(a.weight, e) : static_cast<const float*>(a.weight)[e]; };
        auto hidden = [&](uint32_t e) { return b ? x[e] + b[e] : x[e]; };
        auto value = [&](uint32_t e) -> double {  // norm: without the factor of its row
            if constexpr (OP == kRowsF32) return x[e];
            if constexpr (OP == kRowsBf16) return bf16_at(a.x, row * a.ldx + e);
            if constexpr (OP == kRowsNorm) return static_cast<double>(hidden(e)) * static_cast<double>(weight(e));
            const double g = x[e];
            return g / (1.0 + exp(-g)) * static_cast<double>(b[e]);
        };
        double top = 0, square = 0;
        for (uint32_t e = threadIdx.x; e < a.width; e += kThreads) {
            top = larger(top, fabs(value(e)));
            if constexpr (OP == kRowsNorm) {
                const double h = hidden(e);
                square = fma(h, h, square);
            }
        }
        top = block_max(top, part);
        double factor = 1;
        if constexpr (OP == kRowsNorm) {
            factor = 1.0 / sqrt(block_sum(square, part) / a.width + static_cast<double>(a.eps));
            top *= factor;
        }
        float scale = static_cast<float>(top / 127.0);
        if (!(scale < INFINITY)) scale = NAN;
        for (uint32_t e = threadIdx.x; e < a.width; e += kThreads) {
            double v = value(e);
            if constexpr (OP == kRowsNorm) {
                const float h = hidden(e);
                v *= factor;
                if (a.sum) a.sum[row * a.lds + e] = h;
                if (a.y) a.y[row * a.ldy + e] = static_cast<float>(v);
            }
            if (a.codes) {
                const double t = rint(v / static_cast<double>(scale));
                a.codes[row * a.ldc + e] = scale > 0 ? static_cast<int8_t>(fmin(fmax(t, -127.0), 127.0)) : 0;
            }
        }
        if (a.codes) {
            const uint32_t end = (a.width + kCodesPerUnit - 1) / kCodesPerUnit * kCodesPerUnit;
            for (uint32_t e = a.width + threadIdx.x; e < end; e += kThreads) a.codes[row * a.ldc + e] = 0;
            if (threadIdx.x == 0) a.scales[row] = scale;
        }
    }
}

template <int OP>
int launch(RowsArgs& a, hipStream_t s) {
    const uint32_t blocks = std::min(a.rows, 1u << 20);
    PAGED_TRY(vlaunch(rows_i8_kernel<OP>, dim3(blocks), dim3(kThreads), 0, s, a));
    return VVLI_OK;
}

uint64_t padded(uint32_t width) { return (uint64_t{width} + kCodesPerUnit - 1) / kCodesPerUnit * kCodesPerUnit; }

int check_codes(const int8_t* codes, uint64_t ldc, const float* scales, uint32_t width, const char* who) {
    const int rc = check_row_units(codes, ldc, padded(width), 1, "codes", who);
    if (rc) return rc;
    if (!scales) return set_error(VVLI_NULL_ARG, "%s: NULL scales", who);
    return VVLI_OK;
}

int check_sizes(uint32_t rows, uint32_t width, const char* who) {
    if (rows >= kPagedMost || width == 0 || width >= kPagedMost - kCodesPerUnit)
        return set_error(VVLI_INVALID_CONFIG, "%s: bad sizes (%u rows of %u)", who, rows, width);
    return VVLI_OK;
}

struct Outputs {  // what a call writes, and whether an input meets it
    RowBytes at[4];
    const char* name[4];
    int n = 0;
    void add(const void* p, uint64_t ld, uint64_t width, uint64_t rows, const char* what) {
        if (p) at[n] = RowBytes{p, ld, width, rows}, name[n++] = what;
    }
    int each_other(const char* who) const {
        for (int i = 0; i < n; ++i)
            for (int j = 0; j < i; ++j)
                if (rows_meet(at[i], at[j])) return set_error(VVLI_INVALID_CONFIG, "%s: %s overlaps %s", who, name[i], name[j]);
        return VVLI_OK;
    }
    // same: an output that is the input itself, with its stride, is fine (each value is read before its place is written)
    int input(const RowBytes& in, bool same, const char* what, const char* who) const {
        for (int i = 0; i < n; ++i)
            if (rows_meet(at[i], in) && !(same && at[i].p == in.p && at[i].ld == in.ld))
                return set_error(VVLI_INVALID_CONFIG, "%s: %s overlaps %s", who, name[i], what);
        return VVLI_OK;
    }
};

}  // namespace

extern "C" {

int vvli_gpu_quantize_rows(const void* x, uint32_t kind, uint64_t ldx, uint32_t rows, uint32_t width, int8_t* codes,
                           uint64_t ldc, float* scales, void* stream) {
    const char* who = "vvli_gpu_quantize_rows";
    if (kind > VVLI_WEIGHT_BF16) return set_error(VVLI_INVALID_CONFIG, "%s: unknown kind %u", who, kind);
    const uint32_t e = kind == VVLI_WEIGHT_BF16 ? 2 : 4;
    int rc;
    if ((rc = check_sizes(rows, width, who)) || (rc = check_row_units(x, ldx, width, e, "x", who)) ||
        (rc = check_codes(codes, ldc, scales, width, who)))
        return rc;
    Outputs out;
    out.add(codes, ldc, padded(width), rows, "codes"), out.add(scales, 4, 4, rows, "scales");
    if ((rc = out.each_other(who)) || (rc = out.input(RowBytes{x, ldx * e, uint64_t{width} * e, rows}, false, "x", who))) return rc;
    if (rows == 0) return VVLI_OK;
    RowsArgs a{};
    a.x = x, a.scales = scales, a.codes = codes, a.ldx = ldx, a.ldc = ldc, a.rows = rows, a.width = width;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    return kind == VVLI_WEIGHT_BF16 ? launch<kRowsBf16>(a, s) : launch<kRowsF32>(a, s);
}

int vvli_gpu_add_norm(const float* x, uint64_t ldx, const float* delta, uint64_t ldd, uint32_t rows, uint32_t width,
                      const void* weight, uint32_t weight_kind, float eps, float* sum, uint64_t lds, float* y, uint64_t ldy,
                      int8_t* codes, uint64_t ldc, float* scales, void* stream) {
    const char* who = "vvli_gpu_add_norm";
    int rc;
    if ((rc = check_sizes(rows, width, who)) || (rc = check_row_units(x, ldx, width, 4, "x", who)) ||
        (delta && (rc = check_row_units(delta, ldd, width, 4, "delta", who))) ||
        (sum && (rc = check_row_units(sum, lds, width, 4, "sum", who))) ||
        (y && (rc = check_row_units(y, ldy, width, 4, "y", who))))
        return rc;
    if (!weight) return set_error(VVLI_NULL_ARG, "%s: NULL weight", who);
    if (weight_kind > VVLI_WEIGHT_BF16 || !aligned16(weight))
        return set_error(VVLI_INVALID_CONFIG, "%s: weight of kind %u, or not at a 16-byte address", who, weight_kind);
    if (!(eps >= 0.f && std::isfinite(eps))) return set_error(VVLI_INVALID_CONFIG, "%s: eps %g", who, static_cast<double>(eps));
    if (sum && !delta) return set_error(VVLI_INVALID_CONFIG, "%s: a sum of x alone", who);
    if (codes || scales || !y) {
        if ((rc = check_codes(codes, ldc, scales, width, who))) return rc;
    }
    const uint64_t w = uint64_t{width} * 4;
    Outputs out;
    out.add(sum, lds * 4, w, rows, "sum"), out.add(y, ldy * 4, w, rows, "y");
    out.add(codes, ldc, padded(width), rows, "codes"), out.add(scales, 4, 4, rows, "scales");
    const uint64_t wb = uint64_t{width} * (weight_kind == VVLI_WEIGHT_BF16 ? 2 : 4);
    if ((rc = out.each_other(who)) || (rc = out.input(RowBytes{x, ldx * 4, w, rows}, true, "x", who)) ||
        (rc = out.input(RowBytes{delta, ldd * 4, w, rows}, true, "delta", who)) ||
        (rc = out.input(RowBytes{weight, wb, wb, 1}, false, "weight", who)))
        return rc;
    if (rows == 0) return VVLI_OK;
    RowsArgs a{};
    a.x = x, a.weight = weight, a.b = delta, a.sum = sum, a.y = y, a.scales = scales, a.codes = codes;
    a.ldx = ldx, a.ldb = ldd, a.lds = lds, a.ldy = ldy, a.ldc = ldc, a.rows = rows, a.width = width;
    a.weight_bf16 = weight_kind == VVLI_WEIGHT_BF16, a.eps = eps;
    return launch<kRowsNorm>(a, static_cast<hipStream_t>(stream));
}

int vvli_gpu_silu_mul(const float* gate, uint64_t ldg, const float* up, uint64_t ldu, uint32_t rows, uint32_t width,
                      int8_t* codes, uint64_t ldc, float* scales, void* stream) {
    const char* who = "vvli_gpu_silu_mul";
    int rc;
    if ((rc = check_sizes(rows, width, who)) || (rc = check_row_units(gate, ldg, width, 4, "gate", who)) ||
        (rc = check_row_units(up, ldu, width, 4, "up", who)) || (rc = check_codes(codes, ldc, scales, width, who)))
        return rc;
    const uint64_t w = uint64_t{width} * 4;
    Outputs out;
    out.add(codes, ldc, padded(width), rows, "codes"), out.add(scales, 4, 4, rows, "scales");
    if ((rc = out.each_other(who)) || (rc = out.input(RowBytes{gate, ldg * 4, w, rows}, false, "gate", who)) ||
        (rc = out.input(RowBytes{up, ldu * 4, w, rows}, false, "up", who)))
        return rc;
    if (rows == 0) return VVLI_OK;
    RowsArgs a{};
    a.x = gate, a.b = up, a.scales = scales, a.codes = codes, a.ldx = ldg, a.ldb = ldu, a.ldc = ldc, a.rows = rows, a.width = width;
    return launch<kRowsGate>(a, static_cast<hipStream_t>(stream));
}

}  // extern "C"
