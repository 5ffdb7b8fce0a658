// rows_i8.hip -- rows in 8 bits with a scale each: of given rows
// (vvli_gpu_quantize_rows), of a residual's sum behind its RMS norm
// (vvli_gpu_add_norm) and of a gated activation (vvli_gpu_silu_mul).
//
// scale = f32(max |v| / 127), code = rint(v / scale), of v as it is in exact
// arithmetic, so that codes do not change with the order of a row's sums.
// Memory bounds all three, and 64-bit arithmetic on every value would be longer
// than the memory's time (a block a row, all in f64: gate 2500 x 18944 385 us,
// norm 6001 x 3584 314): values are formed in f32, whose error is known, and 64
// bits settle what f32 cannot, which is
//   * the largest value of a gated row: those whose f32 value is within that
//     error of the largest one (mostly one of a row) are formed in f64 (a
//     norm's are all: a product each);
//   * a code whose f32 quotient is within the error of a border between two
//     codes. Its unit of 16 bytes is read again, at once, and f64 forms the values
//     that are in doubt alone (of a wave's 64 units one in 30 holds one, gated one
//     in 8; of bf16, whose few bits make ties, nine of ten waves do. Read and
//     formed one after the other, weights took 59 us, gate 10 more).
// Where f32's error is not the usual one (values that left its normal range) a
// row is formed in f64 as a whole. Measured (calls that follow one another over
// inputs that no cache holds; a copy of 1 GB moves 5.06 TB/s): weights 18944 x 3584
// bf16 41.6 us (4.9 TB/s), f32 rows 6001 x 3584 19.4 (5.5), their norm with the sum
// 55.2 (5.1), gate 2500 x 18944 80.1 (5.3). Behind a fill of 300 MB, whose lines the
// caches have yet to write: weights 55.7, norm 56.0, gate 101.8.
// One row of 2048: 4.2, 4.5 and 4.4 us, of which 3.8 is a launch.
#include <algorithm>
#include <type_traits>

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
    bool once;  // gate and up pass the caches
    float eps;
};

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ float bf16_bits(uint32_t u) { return __uint_as_float(u << 16); }
__device__ __forceinline__ float bf16_at(const void* p, size_t i) { return bf16_bits(static_cast<const uint16_t*>(p)[i]); }

// ---- reductions: within a wave by DPP, between waves through LDS -----------
// (quad_perm, row_half_mirror and row_mirror leave every lane of 16 with their total; four totals by readlane)
template <int CTRL>
__device__ __forceinline__ uint32_t dpp(uint32_t v) {
    return __builtin_amdgcn_update_dpp(0, v, CTRL, 0xF, 0xF, false);
}
template <int CTRL>
__device__ __forceinline__ double dpp(double v) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    return __builtin_bit_cast(double, static_cast<uint64_t>(dpp<CTRL>(static_cast<uint32_t>(u >> 32))) << 32 |
                                          dpp<CTRL>(static_cast<uint32_t>(u)));
}
template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
    return __uint_as_float(dpp<CTRL>(__float_as_uint(v)));
}
__device__ __forceinline__ uint32_t lane_of(uint32_t v, int lane) { return __builtin_amdgcn_readlane(v, lane); }
__device__ __forceinline__ double lane_of(double v, int lane) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    return __builtin_bit_cast(double, static_cast<uint64_t>(lane_of(static_cast<uint32_t>(u >> 32), lane)) << 32 |
                                          lane_of(static_cast<uint32_t>(u), lane));
}
__device__ __forceinline__ float lane_of(float v, int lane) { return __uint_as_float(lane_of(__float_as_uint(v), lane)); }
struct Add {
    template <typename T>
    __device__ __forceinline__ T operator()(T a, T b) const { return a + b; }
};
struct Max {  // (of doubles: NaN if one is NaN)
    __device__ __forceinline__ float operator()(float a, float b) const { return fmaxf(a, b); }
    __device__ __forceinline__ double operator()(double a, double b) const { return a >= b || a != a ? a : b; }
};
template <typename T, typename F>
__device__ __forceinline__ T reduce_wave(T v, F f) {
    v = f(v, dpp<0xB1>(v)), v = f(v, dpp<0x4E>(v)), v = f(v, dpp<0x141>(v)), v = f(v, dpp<0x140>(v));
    return f(f(lane_of(v, 0), lane_of(v, 16)), f(lane_of(v, 32), lane_of(v, 48)));
}
// Two values of a row's WAVES waves at once; part: 2 WAVES values.
template <int WAVES, typename T, typename F, typename H>
__device__ __forceinline__ void reduce(T& v, F f, T& w, H h, T* part) {
    v = reduce_wave(v, f), w = reduce_wave(w, h);
    if constexpr (WAVES > 1) {
        __syncthreads();
        if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v, part[WAVES + (threadIdx.x >> 6)] = w;
        __syncthreads();
        v = part[0], w = part[WAVES];
#pragma unroll
        for (int i = 1; i < WAVES; ++i) v = f(v, part[i]), w = h(w, part[WAVES + i]);
    }
}
template <int WAVES, typename T, typename F>
__device__ __forceinline__ T reduce(T v, F f, T* part) {
    v = reduce_wave(v, f);
    if constexpr (WAVES > 1) {
        __syncthreads();
        if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
        __syncthreads();
        v = part[0];
#pragma unroll
        for (int i = 1; i < WAVES; ++i) v = f(v, part[i]);
    }
    return v;
}

// f32's silu(g) u, for g >= -16 off by less than 1.3e-6 < 2^-19.5 of the value: the exponent's product with log2 e is off by
// 2^-20 and 2.3e-7 where it is largest (of a value between 16 and 32), v_exp_f32 and v_rcp_f32 by one last bit, the rest
// by half of one each. Below -16 it is off by 2^-16 of a value that is under 1.9e-6 |u|: rows where that could be a
// larger part of the row's largest value than 2^-9 are not usual ones.
__device__ __forceinline__ float gated32(float g, float u) {
    const float p = __builtin_amdgcn_exp2f(g * -1.44269502f);
    return g * u * __builtin_amdgcn_rcpf(1.f + p);
}

// The weights of unit u, whole.
__device__ __forceinline__ f32x4 weights4(const RowsArgs& a, uint32_t u) {
    if (!a.weight_bf16) return *as_global(static_cast<const f32x4*>(a.weight) + u);
    const uint2 t = load_u32x2(static_cast<const uint2*>(a.weight) + u);
    return f32x4{bf16_bits(t.x), __uint_as_float(t.x & 0xffff0000u), bf16_bits(t.y), __uint_as_float(t.y & 0xffff0000u)};
}

// ---- a row's values ---------------------------------------------------------
// Rows that are mostly not read again pass the caches, which leaves them to what is stored (norm, us: 6001 x 3584 58.0, so
// 55.2; 2500 x 18944 128, 114; f32 rows 6001 x 3584 21.3, 19.4). Units in doubt are read again. Of bf16 rows they are many
// (18944 x 3584 41.6, so 43.6), and of gated ones, which pass the caches only where they are too long for them to hold
// (300 x 4864 8.5, so 9.8; 3000 x 4864 31.7, 34.3; 4096 x 8192 58.2, 53.1; 2500 x 18944 86.7, 80.1). Codes stay in the
// caches for whoever reads them next.
constexpr uint64_t kOnceBytes = uint64_t{128} << 20;
template <bool ONCE>
__device__ __forceinline__ f32x4 read16(const void* p, uint32_t u) {
    const auto at = as_global(static_cast<const f32x4*>(p) + u);
    return ONCE ? __builtin_nontemporal_load(at) : *at;
}

// A value is made of one or two others: of a row's, a hidden value and its weight, or gate and up.
template <int OP>
struct Row {
    static constexpr int E = OP == kRowsBf16 ? 8 : 4;  // values of 16 bytes
    const RowsArgs& a;
    const float *x, *b;
    uint32_t row;
    const float* h;  // where the sum is stored (in x's or delta's place, it may be): read there from then on
    __device__ __forceinline__ Row(const RowsArgs& a_, uint32_t r)
        : a(a_), x(static_cast<const float*>(a_.x) + r * a_.ldx), b(a_.b ? a_.b + r * a_.ldb : nullptr), row(r),
          h(a_.sum ? a_.sum + r * a_.lds : nullptr) {}
    __device__ __forceinline__ float weight(uint32_t e) const {
        return a.weight_bf16 ? bf16_at(a.weight, e) : static_cast<const float*>(a.weight)[e];
    }
    __device__ __forceinline__ float first(uint32_t e) const {
        if constexpr (OP == kRowsBf16) return bf16_at(a.x, row * a.ldx + e);
        if constexpr (OP == kRowsNorm) return h ? h[e] : b ? x[e] + b[e] : x[e];
        return x[e];
    }
    __device__ __forceinline__ float second(uint32_t e) const {
        return OP == kRowsNorm ? weight(e) : OP == kRowsGate ? b[e] : 0.f;
    }
    typedef float Unit __attribute__((ext_vector_type(E)));
    // The E values of unit u, 0 behind the width (whole: none is).
    __device__ __forceinline__ void unit(uint32_t u, bool whole, Unit& p, Unit& q) const {
        if (!whole) {
#pragma unroll
            for (uint32_t e = 0; e < E; ++e) {
                const bool in = u * E + e < a.width;
                p[e] = in ? first(u * E + e) : 0.f, q[e] = in ? second(u * E + e) : 0.f;
            }
            return;
        }
        const void* at = OP == kRowsBf16 ? static_cast<const void*>(static_cast<const uint16_t*>(a.x) + row * a.ldx) : OP == kRowsNorm && h ? h : x;
        f32x4 v = *as_global(static_cast<const f32x4*>(at) + u), w = {0, 0, 0, 0};
        if constexpr (OP == kRowsNorm) {
            w = weights4(a, u);
            if (!h && b) v += *as_global(reinterpret_cast<const f32x4*>(b) + u);
        }
        if constexpr (OP == kRowsGate) w = *as_global(reinterpret_cast<const f32x4*>(b) + u);
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const uint32_t two = __float_as_uint(v[e * 4 / E]);
            p[e] = OP != kRowsBf16 ? v[e * 4 / E] : e % 2 ? __uint_as_float(two & 0xffff0000u) : bf16_bits(two), q[e] = w[e * 4 / E];
        }
    }
    // As the definition has it (norm: without the factor of its row), and as f32 has it.
    static __device__ __forceinline__ double f64(float p, float q) {
        if constexpr (OP == kRowsNorm) return static_cast<double>(p) * static_cast<double>(q);
        const double g = p;
        if constexpr (OP == kRowsGate) return g / (1.0 + exp(-g)) * static_cast<double>(q);
        return g;
    }
    static __device__ __forceinline__ float f32(float p, float q) { return OP == kRowsNorm ? p * q : OP == kRowsGate ? gated32(p, q) : p; }
    __device__ __forceinline__ double operator()(uint32_t e) const { return f64(first(e), second(e)); }
};
template <typename U>
__device__ __forceinline__ float pick(U v, uint32_t i) {
    float r = v[0];
#pragma unroll
    for (uint32_t e = 1; e < sizeof(U) / 4; ++e) r = i == e ? v[e] : r;
    return r;
}

__device__ __forceinline__ float scale_of(double top) {
    const float s = static_cast<float>(top / 127.0);
    return s < INFINITY ? s : NAN;
}
__device__ __forceinline__ int code_of(double v, float scale) {
    return scale > 0 ? static_cast<int>(fmin(fmax(rint(v / static_cast<double>(scale)), -127.0), 127.0)) : 0;
}

// ---- any width: a block a row, two passes over it, all in f64 ----------------
constexpr int kAnyThreads = 1024, kAnyWaves = kAnyThreads / 64;

template <int OP>
__global__ __launch_bounds__(kAnyThreads) void rows_any_kernel(RowsArgs a) {
    __shared__ double part[kAnyWaves];
    for (uint32_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const Row<OP> value(a, row);
        double top = 0, square = 0;
        for (uint32_t e = threadIdx.x; e < a.width; e += kAnyThreads) {
            if constexpr (OP == kRowsNorm) {
                if (a.sum) a.sum[row * a.lds + e] = value.x[e] + value.b[e];
            }
            top = Max()(top, fabs(value(e)));
            if constexpr (OP == kRowsNorm) {
                const double h = value.first(e);
                square = fma(h, h, square);
            }
        }
        top = reduce<kAnyWaves>(top, Max(), part);
        double factor = 1;
        if constexpr (OP == kRowsNorm) {
            factor = 1.0 / sqrt(reduce<kAnyWaves>(square, Add(), part) / a.width + static_cast<double>(a.eps));
            top *= factor;
        }
        const float scale = scale_of(top);
        for (uint32_t e = threadIdx.x; e < a.width; e += kAnyThreads) {
            double v = value(e);
            if constexpr (OP == kRowsNorm) {
                v *= factor;
                if (a.y) a.y[row * a.ldy + e] = static_cast<float>(v);
            }
            if (a.codes) a.codes[row * a.ldc + e] = static_cast<int8_t>(code_of(v, scale));
        }
        if (a.codes) {
            const uint32_t end = (a.width + kCodesPerUnit - 1) / kCodesPerUnit * kCodesPerUnit;
            for (uint32_t e = a.width + threadIdx.x; e < end; e += kAnyThreads) a.codes[row * a.ldc + e] = 0;
            if (threadIdx.x == 0) a.scales[row] = scale;
        }
    }
}

// ---- rows that registers hold: WAVES waves a row, one pass -------------------
// A lane holds units of E values (4 of f32, 8 of bf16: 16 bytes), unit lane + 64
// WAVES j of the row for j < V, so that a load of a wave is 1 KiB in a row; what
// it keeps are the f32 values that the codes are made of (of bf16 the units as
// they come). What f64 settles is read again.

constexpr float kMostUp = 0x1p10f;  // of a usual row: max |u| over the largest value
// How far |t - rint(t)| may be from 1/2 for f32 to tell the code of t = value / scale, |t| <= 127: off by 127 halves of a
// last bit of f32 for the product and for the quotient each (2^-16), and of a norm's value (2^-17); a gated value by
// 127 * 1.3e-6 more (1.7e-4).
template <int OP>
constexpr float band() { return OP == kRowsGate ? 0x1p-12f : 0x1p-14f; }
// Last bits of f32 by which two gated values may be off (2 * 1.3e-6 * 2^24 = 44).
constexpr uint32_t kTopBits = 48;

// Keeps the compiler from reading ahead over all of a row's units, and from keeping each unit's address and bound from
// one use to the next: either takes more registers than there are.
__device__ __forceinline__ void in_turn(uint32_t& id) { asm volatile("" : "+v"(id)::"memory"); }

template <int OP, int WAVES, int V>
__global__ __launch_bounds__(WAVES == 1 ? 256 : WAVES * 64, 4) void rows_i8_kernel(RowsArgs a) {
    constexpr int G = WAVES * 64, E = Row<OP>::E, ROWS = WAVES == 1 ? 4 : 1;  // rows of a block
    constexpr int N = V % 4 == 0 ? 4 : V % 3 == 0 ? 3 : 2;  // units in flight
    static_assert(V % N == 0, "whole turns");
    __shared__ double part_d[2 * WAVES];
    __shared__ float part_f[2 * WAVES];
    uint32_t id = WAVES == 1 ? threadIdx.x & 63 : threadIdx.x;
    // Whole units, and those behind them up to the padded width: the first may hold the row's last values, lane i has
    // the i-th of them as its unit V.
    const uint32_t full = a.width / E, units = (a.width + kCodesPerUnit - 1) / kCodesPerUnit * (kCodesPerUnit / E);
    const bool tail = units > full;  // (the same for all, as a width is: whole units mostly)
    const uint32_t first = blockIdx.x * ROWS + (WAVES == 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x / 64) : 0);
    for (uint32_t row = first; row < a.rows; row += gridDim.x * ROWS) {
        const Row<OP> value(a, row);
        f32x4 v[V + 1];
        float top = 0, most_u = 0, odd32 = 0;
        double square = 0, exact = 0, odd = 0;  // odd: NaN if a value is not finite
        auto norm_value = [&](float h, float w) {
            const double x = h, y = x * static_cast<double>(w);
            square = fma(x, x, square), exact = fmax(exact, fabs(y)), odd = fma(y, 0.0, odd);
            return h * w;
        };
#pragma unroll
        for (int j0 = 0; j0 < V; j0 += N) {
            in_turn(id);
#pragma unroll
            for (int j = j0; j < j0 + N; ++j) v[j] = f32x4{0, 0, 0, 0};
            if (static_cast<uint32_t>(j0) * G >= full) continue;  // (the same for all)
            f32x4 p[N], q[N];
            auto load = [&](auto once) {
#pragma unroll
                for (int j = 0; j < N; ++j) {
                    const uint32_t u = min(id + (j0 + j) * G, full - 1);
                    if constexpr (OP == kRowsBf16) p[j] = read16<once>(static_cast<const uint16_t*>(a.x) + row * a.ldx, u);
                    else p[j] = read16<once>(value.x, u);
                    if constexpr (OP == kRowsGate || OP == kRowsNorm) q[j] = value.b ? read16<once>(value.b, u) : f32x4{0, 0, 0, 0};
                }
            };
            if constexpr (OP != kRowsGate) {
                load(std::bool_constant<OP != kRowsBf16>{});
            } else if (a.once) {
                load(std::true_type{});
                in_turn(id);  // (else the compiler makes both branches one)
            } else {
                load(std::false_type{});
            }
#pragma unroll
            for (int j = j0; j < j0 + N; ++j) {
                const uint32_t at = id + j * G;
                v[j] = p[j - j0];
                if constexpr (OP == kRowsGate) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[j][e] = gated32(v[j][e], q[j - j0][e]), most_u = fmaxf(most_u, fabsf(q[j - j0][e]));
                }
                if constexpr (OP == kRowsNorm) {
                    const bool in = at < full;
                    const f32x4 w = weights4(a, min(at, full - 1));
                    if (value.b) v[j] += q[j - j0];
                    if (a.sum && in) *as_global(reinterpret_cast<f32x4*>(a.sum + row * a.lds) + at) = v[j];
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[j][e] = norm_value(in ? v[j][e] : 0.f, in ? w[e] : 0.f);
                }
            }
        }
        v[V] = f32x4{0, 0, 0, 0};
        if (tail && id == 0) {
#pragma unroll
            for (uint32_t e = 0; e < E; ++e) {
                const uint32_t at = full * E + e;
                if (at >= a.width) continue;
                if constexpr (OP == kRowsBf16) {
                    const uint32_t w = static_cast<const uint16_t*>(a.x)[row * a.ldx + at];
                    v[V][e / 2] = __uint_as_float(__float_as_uint(v[V][e / 2]) | w << (e % 2 * 16));
                } else if constexpr (OP == kRowsGate) {
                    v[V][e] = gated32(value.x[at], value.b[at]), most_u = fmaxf(most_u, fabsf(value.b[at]));
                } else if constexpr (OP == kRowsNorm) {
                    const float h = value.b ? value.x[at] + value.b[at] : value.x[at];
                    if (a.sum) a.sum[row * a.lds + at] = h;
                    v[V][e] = norm_value(h, value.weight(at));
                } else {
                    v[V][e] = value.x[at];
                }
            }
        }
        in_turn(id);
        double factor = 1;
        bool usual = true;  // (of the whole row)
        auto unit_of = [&](int j) { return j < V ? id + j * G : full + id; };
        if constexpr (OP == kRowsNorm) {
            if (!(odd == 0)) exact = odd;
            reduce<WAVES>(exact, Max(), square, Add(), part_d);
            factor = 1.0 / sqrt(square / a.width + static_cast<double>(a.eps));
            usual = exact >= 0x1p-100 && exact <= 0x1p100;
            exact *= factor;
        } else {
            if constexpr (OP == kRowsBf16) {  // (two values at a time: without their signs, bits are ordered as values are)
                u16x2 most = {0, 0};
#pragma unroll
                for (int j = 0; j <= V; ++j) {
                    if (j == V && !tail) continue;
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        most = __builtin_elementwise_max(most, __builtin_bit_cast(u16x2, __float_as_uint(v[j][e]) & 0x7fff7fffu));
                }
                const uint32_t m = max(most[0], most[1]);
                top = bf16_bits(m), odd32 = m < 0x7f80u ? 0.f : NAN;
            } else {
#pragma unroll
                for (int j = 0; j <= V; ++j) {
                    if (j == V && !tail) continue;
#pragma unroll
                    for (int e = 0; e < 4; ++e) top = fmaxf(top, fabsf(v[j][e])), odd32 = fmaf(v[j][e], 0.f, odd32);
                }
            }
            float largest = odd32 == 0 ? top : INFINITY;  // (of the thread's)
            if constexpr (OP == kRowsGate) reduce<WAVES>(largest, Max(), most_u, Max(), part_f);
            else largest = reduce<WAVES>(largest, Max(), part_f);
            exact = top = largest;
        }
        if constexpr (OP == kRowsGate) {
            usual = top >= 0x1p-40f && top <= 0x1p100f && most_u <= kMostUp * top;
            const uint32_t least = __float_as_uint(top) - kTopBits;
            uint32_t near = 0;  // units that may hold the largest
#pragma unroll
            for (int j = 0; j <= V; ++j) {
                if (j == V && !tail) continue;
                const float most = fmaxf(fmaxf(fabsf(v[j][0]), fabsf(v[j][1])), fmaxf(fabsf(v[j][2]), fabsf(v[j][3])));
                if (most >= __uint_as_float(least)) near |= 1u << j;
            }
            if (!usual) near = (2u << V) - 1;  // (unit V too: there are no values in it where there is no tail)
            exact = 0;
            for (; near; near &= near - 1) {
                const uint32_t u = unit_of(__builtin_ctz(near));
                typename Row<OP>::Unit p, q;
                value.unit(u, u < full, p, q);
                uint32_t some = 0;
#pragma unroll
                for (uint32_t e = 0; e < E; ++e)
                    if (u * E + e < a.width && (!usual || fabsf(gated32(p[e], q[e])) >= __uint_as_float(least - 1))) some |= 1u << e;
                for (; some; some &= some - 1) exact = Max()(exact, fabs(value.f64(pick(p, __builtin_ctz(some)), pick(q, __builtin_ctz(some)))));
            }
            exact = reduce<WAVES>(exact, Max(), part_d);
        }
        // (0 beside a scale of 0 or NaN: the zeros behind the width are stored as they come, and a norm's NaN would bring
        // its bits into them.)
        const float scale = scale_of(exact), quotient = scale > 0 ? static_cast<float>(factor / static_cast<double>(scale)) : 0.f;
        // (Rows of zeros, padding mostly, have no codes to settle: f32's values are finite there, a norm's below 2^-15.)
        usual = scale == 0 ? OP == kRowsNorm || top < INFINITY : usual && scale >= 0x1p-126f;
        int8_t* const codes = a.codes ? a.codes + row * a.ldc : nullptr;
        if (codes) {
            if (id == 0) a.scales[row] = scale;
            uint32_t doubt = 0;
#pragma unroll
            for (int j = 0; j <= V; ++j) {
                if (j % N == 0) in_turn(id);
                if (j == V && !tail) continue;
                const uint32_t u = unit_of(j);
                uint32_t word[E / 4];
                float far = 0;
#pragma unroll
                for (int q = 0; q < E / 4; ++q) {
                    uint32_t bits[4];
                    float off[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        float x = v[j][e];
                        if constexpr (OP == kRowsBf16) {
                            const uint32_t two = __float_as_uint(v[j][q * 2 + e / 2]);
                            x = e % 2 ? __uint_as_float(two & 0xffff0000u) : bf16_bits(two);
                        }
                        const float near = fmaf(x, quotient, 0x1.8p23f);  // rint of the product in the last bits
                        off[e] = fmaf(x, quotient, 0x1.8p23f - near), bits[e] = __float_as_uint(near);
                    }
                    far = fmaxf(fmaxf(far, fmaxf(fabsf(off[0]), fabsf(off[1]))), fmaxf(fabsf(off[2]), fabsf(off[3])));
                    // (v_perm_b32: bytes 0-3 of the second operand, 4-7 of the first)
                    word[q] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(bits[3], bits[2], 0x0c0c0400),
                                                    __builtin_amdgcn_perm(bits[1], bits[0], 0x0c0c0400), 0x05040100);
                }
                if (u < (j < V ? full : units)) {
                    if (!usual || far > 0.5f - band<OP>()) doubt |= 1u << j;
                    if constexpr (E == 8) *as_global(reinterpret_cast<vvli_u32x2*>(codes) + u) = vvli_u32x2{word[0], word[1]};
                    else *as_global(reinterpret_cast<uint32_t*>(codes) + u) = word[0];
                }
            }
            // (Of a unit in doubt, only the values that are, mostly one. The bound is a little wider than the one above.)
            for (; doubt; doubt &= doubt - 1) {
                const uint32_t u = unit_of(__builtin_ctz(doubt));
                typename Row<OP>::Unit p, q;
                value.unit(u, u < full, p, q);
                uint32_t some = 0;
#pragma unroll
                for (uint32_t e = 0; e < E; ++e) {
                    const float x = value.f32(p[e], q[e]), near = fmaf(x, quotient, 0x1.8p23f), off = fmaf(x, quotient, 0x1.8p23f - near);
                    if (u * E + e < a.width && (!usual || fabsf(off) > 0.5f - 1.0625f * band<OP>())) some |= 1u << e;
                }
                for (; some; some &= some - 1) {
                    const uint32_t e = __builtin_ctz(some);
                    codes[u * E + e] = static_cast<int8_t>(code_of(value.f64(pick(p, e), pick(q, e)) * factor, scale));
                }
            }
        }
        if constexpr (OP == kRowsNorm) {
            if (a.y) {  // (may be x or delta: behind all that reads them)
                float* y = a.y + row * a.ldy;
#pragma unroll
                for (int j0 = 0; j0 < V; j0 += N) {
                    in_turn(id);
                    if (static_cast<uint32_t>(j0) * G >= full) continue;
                    typename Row<OP>::Unit p[N], q[N];
#pragma unroll
                    for (int j = 0; j < N; ++j) value.unit(min(id + (j0 + j) * G, full - 1), true, p[j], q[j]);
#pragma unroll
                    for (int j = 0; j < N; ++j) {
                        const uint32_t u = id + (j0 + j) * G;
                        f32x4 o;
#pragma unroll
                        for (int e = 0; e < 4; ++e) o[e] = static_cast<float>(value.f64(p[j][e], q[j][e]) * factor);
                        if (u < full) *as_global(reinterpret_cast<f32x4*>(y) + u) = o;
                    }
                }
                if (const uint32_t e = full * 4 + id; e < a.width) y[e] = static_cast<float>(value(e) * factor);
            }
        }
    }
}

template <int OP, int WAVES, int V>
hipError_t launch_rows(const RowsArgs& a, hipStream_t s) {
    constexpr uint32_t ROWS = WAVES == 1 ? 4 : 1, THREADS = WAVES == 1 ? 256 : WAVES * 64;
    const uint32_t blocks = std::min((a.rows - 1) / ROWS + 1, 1u << 20);
    return vlaunch(rows_i8_kernel<OP, WAVES, OP == kRowsBf16 ? V / 2 : V>, dim3(blocks), dim3(THREADS), 0, s, a);
}

template <int OP>
int launch(RowsArgs a, hipStream_t s) {
    a.once = uint64_t{a.rows} * a.width * 8 > kOnceBytes;
    // By the width alone: the fewest waves that hold a row in 4 to 12 units a lane, so that several rows' blocks share a
    // CU and one's loads run beside another's codes. Norm, us, of waves x units (6001 x 3584: 4 x 4 55, 2 x 8 58, 8 x 4
    // 70; 2500 x 8192: 4 x 8 51, 8 x 4 52, 16 x 4 81; 300 x 8192: 12.7, 12.1, 17.1; 2500 x 18944: 8 x 12 114, 16 x 8 146;
    // 75 x 3584: 4 x 4 5.6, 2 x 8 6.8, 8 x 4 6.1; 1 x 2048: 4.8 from 2 waves on, 1 x 8 5.8).
    const uint32_t w = a.width;
    hipError_t e;
    if (w <= 1024) e = launch_rows<OP, 1, 4>(a, s);
    else if (w <= 2048) e = launch_rows<OP, 2, 4>(a, s);
    else if (w <= 4096) e = launch_rows<OP, 4, 4>(a, s);
    else if (w <= 8192) e = launch_rows<OP, 4, 8>(a, s);
    else if (w <= 16384) e = launch_rows<OP, 8, 8>(a, s);
    else if (w <= 24576) e = launch_rows<OP, 8, 12>(a, s);
    else if (w <= 32768) e = launch_rows<OP, 16, 8>(a, s);
    else e = vlaunch(rows_any_kernel<OP>, dim3(std::min(a.rows, 1u << 20)), dim3(kAnyThreads), 0, s, a);
    PAGED_TRY(e);
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
    bool in_place[4];
    int n = 0;
    // may: the output may be an input itself, with its stride (each value is read before its place is written)
    void add(const void* p, uint64_t ld, uint64_t width, uint64_t rows, const char* what, bool may = false) {
        if (p) at[n] = RowBytes{p, ld, width, rows}, in_place[n] = may, name[n++] = what;
    }
    int each_other(const char* who) const {
        for (int i = 0; i < n; ++i)
            for (int j = 0; j < i; ++j)
                if (rows_meet(at[i], at[j])) return set_error(VVLI_INVALID_CONFIG, "%s: %s overlaps %s", who, name[i], name[j]);
        return VVLI_OK;
    }
    int input(const RowBytes& in, const char* what, const char* who) const {
        for (int i = 0; i < n; ++i)
            if (rows_meet(at[i], in) && !(in_place[i] && at[i].p == in.p && at[i].ld == in.ld))
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
    if ((rc = out.each_other(who)) || (rc = out.input(RowBytes{x, ldx * e, uint64_t{width} * e, rows}, "x", who))) return rc;
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
    out.add(sum, lds * 4, w, rows, "sum", true), out.add(y, ldy * 4, w, rows, "y", true);
    out.add(codes, ldc, padded(width), rows, "codes"), out.add(scales, 4, 4, rows, "scales");
    const uint64_t wb = uint64_t{width} * (weight_kind == VVLI_WEIGHT_BF16 ? 2 : 4);
    if ((rc = out.each_other(who)) || (rc = out.input(RowBytes{x, ldx * 4, w, rows}, "x", who)) ||
        (rc = out.input(RowBytes{delta, ldd * 4, w, rows}, "delta", who)) ||
        (rc = out.input(RowBytes{weight, wb, wb, 1}, "weight", who)))
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
    if ((rc = out.each_other(who)) || (rc = out.input(RowBytes{gate, ldg * 4, w, rows}, "gate", who)) ||
        (rc = out.input(RowBytes{up, ldu * 4, w, rows}, "up", who)))
        return rc;
    if (rows == 0) return VVLI_OK;
    RowsArgs a{};
    a.x = gate, a.b = up, a.scales = scales, a.codes = codes, a.ldx = ldg, a.ldb = ldu, a.ldc = ldc, a.rows = rows, a.width = width;
    return launch<kRowsGate>(a, static_cast<hipStream_t>(stream));
}

}  // extern "C"
