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
typedef float f32x4 __attribute__((ext_vector_type(4)));

struct LinearI8Args {
    const int8_t *W, *X;
    const float *w_scales, *x_scales;
    const uint16_t* bias;
    float* Y;
    uint64_t ldw, ldx, ldy;
    uint32_t M, N, K;
    bool vector;  // Y's rows and w_scales at 16-byte addresses
};

constexpr int kOnce = 2;  // cache policy of copies of what is read once: nontemporal
constexpr uint32_t kMostK = 131056;  // 131056 * 128 * 128 < 2^31

__device__ __forceinline__ float finish(int sum, float x_scale, float w_scale, float bias) {
#pragma clang fp contract(off)
    return static_cast<float>(sum) * x_scale * w_scale + bias;  // each rounded: no multiply-add
}

__device__ __forceinline__ float bias_at(const uint16_t* bias, uint32_t n) {
    return bias ? __uint_as_float(static_cast<uint32_t>(bias[n]) << 16) : 0.f;
}
// Four results of one row of Y, n .. n + 3.
__device__ __forceinline__ void store4(const LinearI8Args& a, uint32_t m, uint32_t n, i32x4 sum) {
    if (m >= a.M) return;
    const float x_scale = a.x_scales[m];
    float* y = a.Y + m * a.ldy + n;
    if (a.vector && n + 3 < a.N) {
        const f32x4 w = *reinterpret_cast<const f32x4*>(a.w_scales + n);
        f32x4 v;
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = finish(sum[j], x_scale, w[j], bias_at(a.bias, n + j));
        *reinterpret_cast<f32x4*>(y) = v;
        return;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (n + j < a.N) y[j] = finish(sum[j], x_scale, a.w_scales[n + j], bias_at(a.bias, n + j));
}

typedef __attribute__((address_space(3))) void lds_void;
__device__ __forceinline__ uint32_t lds_address(const void* p) { return (uint32_t)(uintptr_t)(lds_void*)p; }
__device__ __align__(16) int8_t no_codes[16];  // what lanes behind K copy

// 1 KiB into LDS, 16 bytes a lane. POLICY: of the caches.
template <int POLICY>
__device__ __forceinline__ void copy16(const void* from, char* to) {
    __builtin_amdgcn_global_load_lds(from, (lds_void*)to, 16, 0, POLICY);
}
// At most n of the wave's copies in flight.
template <int N>
__device__ __forceinline__ void wait_copies() {
    static_assert(N >= 0 && N < 64, "vmcnt is 6 bits");
    __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | (7 << 4) | (15 << 8));
}

// A step's fragments out of LDS: 16 rows of 128 bytes are 2048 bytes behind one another. The wait stands in the same
// block: nothing can come between the reads and it.
template <int R, int MT>
__device__ __forceinline__ void read_fragments(i32x4 (&w)[R], i32x4 (&x)[MT], uint32_t wa, uint32_t xa) {
    static_assert((R == 1 || R == 2 || R == 4) && (MT == 1 || MT == 2 || MT == 4), "as written");
#define LDS_W(i, at) "ds_read_b128 %" #i ", %[wa] offset:" #at "\n\t"
#define LDS_X(i, at) "ds_read_b128 %" #i ", %[xa] offset:" #at "\n\t"
#define LDS_END "s_waitcnt lgkmcnt(0)"
#define LDS_IN : [wa] "v"(wa), [xa] "v"(xa) : "memory"
    if constexpr (R == 1 && MT == 1)
        asm volatile(LDS_W(0, 0) LDS_X(1, 0) LDS_END : "=&v"(w[0]), "=&v"(x[0]) LDS_IN);
    if constexpr (R == 1 && MT == 2)
        asm volatile(LDS_W(0, 0) LDS_X(1, 0) LDS_X(2, 2048) LDS_END : "=&v"(w[0]), "=&v"(x[0]), "=&v"(x[1]) LDS_IN);
    if constexpr (R == 1 && MT == 4)
        asm volatile(LDS_W(0, 0) LDS_X(1, 0) LDS_X(2, 2048) LDS_X(3, 4096) LDS_X(4, 6144) LDS_END
                     : "=&v"(w[0]), "=&v"(x[0]), "=&v"(x[1]), "=&v"(x[2]), "=&v"(x[3]) LDS_IN);
    if constexpr (R == 2 && MT == 1)
        asm volatile(LDS_W(0, 0) LDS_W(1, 2048) LDS_X(2, 0) LDS_END : "=&v"(w[0]), "=&v"(w[1]), "=&v"(x[0]) LDS_IN);
    if constexpr (R == 2 && MT == 2)
        asm volatile(LDS_W(0, 0) LDS_W(1, 2048) LDS_X(2, 0) LDS_X(3, 2048) LDS_END
                     : "=&v"(w[0]), "=&v"(w[1]), "=&v"(x[0]), "=&v"(x[1]) LDS_IN);
    if constexpr (R == 2 && MT == 4)
        asm volatile(LDS_W(0, 0) LDS_W(1, 2048) LDS_X(2, 0) LDS_X(3, 2048) LDS_X(4, 4096) LDS_X(5, 6144) LDS_END
                     : "=&v"(w[0]), "=&v"(w[1]), "=&v"(x[0]), "=&v"(x[1]), "=&v"(x[2]), "=&v"(x[3]) LDS_IN);
    if constexpr (R == 4 && MT == 1)
        asm volatile(LDS_W(0, 0) LDS_W(1, 2048) LDS_W(2, 4096) LDS_W(3, 6144) LDS_X(4, 0) LDS_END
                     : "=&v"(w[0]), "=&v"(w[1]), "=&v"(w[2]), "=&v"(w[3]), "=&v"(x[0]) LDS_IN);
    if constexpr (R == 4 && MT == 2)
        asm volatile(LDS_W(0, 0) LDS_W(1, 2048) LDS_W(2, 4096) LDS_W(3, 6144) LDS_X(4, 0) LDS_X(5, 2048) LDS_END
                     : "=&v"(w[0]), "=&v"(w[1]), "=&v"(w[2]), "=&v"(w[3]), "=&v"(x[0]), "=&v"(x[1]) LDS_IN);
    if constexpr (R == 4 && MT == 4)
        asm volatile(LDS_W(0, 0) LDS_W(1, 2048) LDS_W(2, 4096) LDS_W(3, 6144) LDS_X(4, 0) LDS_X(5, 2048) LDS_X(6, 4096) LDS_X(7, 6144) LDS_END
                     : "=&v"(w[0]), "=&v"(w[1]), "=&v"(w[2]), "=&v"(w[3]), "=&v"(x[0]), "=&v"(x[1]), "=&v"(x[2]), "=&v"(x[3]) LDS_IN);
#undef LDS_W
#undef LDS_X
#undef LDS_END
#undef LDS_IN
}

// ---- few rows: every wave a stream of its own ---------------------------------
// A block has R * 16 rows of W times XG * 8 rows of X, its WV waves all of them
// over chunks of 128 codes of K: wave w the chunks w, w + WV, ... A wave copies
// its chunks into its own ST stages of LDS (copies of 1 KiB, 8 rows of 128 bytes
// each) and reads them back in the order of the products' lanes (16-byte unit c of
// row r at c ^ (r & 7): no bank conflicts), so that no wave waits for another
// before the sums of all meet at the end.
template <int R, int XG, int ST, int WV>
__global__ __launch_bounds__(WV * 64) void linear_i8_stream_kernel(LinearI8Args a) {
    constexpr int MT = (XG + 1) / 2, D = 2 * R + XG, STAGE = D * 1024;  // X tiles of 16 rows, copies and bytes of a stage
    extern __shared__ __attribute__((aligned(1024))) char stream_lds[];  // [WV][ST][W: R * 2 KiB | X: XG KiB]
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // Blocks of the same rows of W follow one another on one XCD (block b runs on b % 8).
    const uint32_t tn = (a.N + 16 * R - 1) / (16 * R), tm = (a.M + 8 * XG - 1) / (8 * XG);
    const uint32_t n_tile = blockIdx.x / (8 * tm) * 8 + blockIdx.x % 8, m_tile = blockIdx.x / 8 % tm;
    if (n_tile >= tn) return;
    const uint32_t n0 = n_tile * 16 * R, m0 = m_tile * 8 * XG;
    const uint32_t chunks = (a.K + 127) / 128, mine = wave < chunks ? (chunks - wave + WV - 1) / WV : 0;
    const uint32_t unit = (lane % 8 ^ lane / 8) * 16;  // of a row's 128 codes, what this lane copies
    const int8_t *w[2 * R], *x[XG];
#pragma unroll
    for (int g = 0; g < 2 * R; ++g) w[g] = a.W + min(n0 + g * 8 + lane / 8, a.N - 1) * a.ldw + unit;
#pragma unroll
    for (int g = 0; g < XG; ++g) x[g] = a.X + min(m0 + g * 8 + lane / 8, a.M - 1) * a.ldx + unit;
    char* const ring = stream_lds + wave * (ST * STAGE);
    auto copy = [&](uint32_t i) {  // the wave's chunk i
        const uint32_t k = (wave + i * WV) * 128;
        const bool in = k + unit < a.K;
        char* to = ring + i % ST * STAGE;
#pragma unroll
        for (int g = 0; g < 2 * R; ++g) copy16<kOnce>(in ? w[g] + k : no_codes, to + g * 1024);
#pragma unroll
        for (int g = 0; g < XG; ++g) copy16<0>(in ? x[g] + k : no_codes, to + (2 * R + g) * 1024);
    };
    i32x4 sum[R][MT];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int t = 0; t < MT; ++t) sum[r][t] = i32x4{0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < ST; ++i)
        if (static_cast<uint32_t>(i) < mine) copy(i);
    const uint32_t at = (lane / 16 ^ lane % 8) * 16, ring0 = lds_address(ring);
    const uint32_t wa = lane % 16 * 128 + at, xa = R * 2048 + (XG == 1 ? lane % 8 : lane % 16) * 128 + at;
    for (uint32_t i = 0; i < mine; ++i) {
        const uint32_t newer = min(mine - 1 - i, static_cast<uint32_t>(ST - 1));
        if (newer == ST - 1) wait_copies<(ST - 1) * D>();
        else if (ST > 2 && newer == ST - 2) wait_copies<(ST > 2 ? ST - 2 : 0) * D>();
        else if (ST > 3 && newer == ST - 3) wait_copies<(ST > 3 ? ST - 3 : 0) * D>();
        else wait_copies<0>();
        const uint32_t stage = ring0 + i % ST * STAGE;
        i32x4 fw[2][R], fx[2][MT];
        read_fragments(fw[0], fx[0], stage + wa, stage + xa);
        read_fragments(fw[1], fx[1], stage + (wa ^ 64), stage + (xa ^ 64));
        if (i + ST < mine) copy(i + ST);
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int t = 0; t < MT; ++t) sum[r][t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fw[k][r], fx[k][t], sum[r][t], 0, 0, 0);
    }
    __syncthreads();  // all stages are read
    i32x4* const sums = reinterpret_cast<i32x4*>(stream_lds);  // [WV][R * MT][64]
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int t = 0; t < MT; ++t) sums[(wave * R * MT + r * MT + t) * 64 + lane] = sum[r][t];
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < R * MT * 64; i += WV * 64) {
        i32x4 v = sums[i];
#pragma unroll
        for (int k = 1; k < WV; ++k) v += sums[k * R * MT * 64 + i];
        const uint32_t tile = i / 64, l = i % 64, m = m0 + tile % MT * 16 + l % 16;
        if (XG > 1 || l % 16 < 8) store4(a, m, n0 + tile / MT * 16 + l / 16 * 4, v);
    }
}

template <int R, int XG, int ST, int WV>
hipError_t launch_stream(const LinearI8Args& a, hipStream_t s) {
    constexpr int MT = (XG + 1) / 2, LDS = WV * ST * (2 * R + XG) * 1024;
    static_assert(LDS <= 160 * 1024 && R * MT <= ST * (2 * R + XG) && ST <= 4, "stages, sums and waits fit");
    const uint64_t tn = (uint64_t{a.N} + 16 * R - 1) / (16 * R), tm = (uint64_t{a.M} + 8 * XG - 1) / (8 * XG);
    static const hipError_t ready = hipFuncSetAttribute(reinterpret_cast<const void*>(linear_i8_stream_kernel<R, XG, ST, WV>),
                                                        hipFuncAttributeMaxDynamicSharedMemorySize, LDS);
    if (ready != hipSuccess) return ready;
    return vlaunch(linear_i8_stream_kernel<R, XG, ST, WV>, dim3(static_cast<uint32_t>((tn + 7) / 8 * 8 * tm)), dim3(WV * 64), LDS, s, a);
}

// ---- many rows: 256 x 256 ------------------------------------------------------
// A block of four waves per CU, one on each SIMD, 128 x 128 each: the fewest
// fragment bytes a product that the registers hold (256 of sums, 64 for each of
// two sets of fragments). LDS takes 64 KiB of copies and gives 128 KiB of fragments
// in a step of 128 codes, 1536 cycles of its 128 bytes a cycle, for 2048 cycles of
// products; eight waves of 128 x 64 read 192 KiB, which with the copies is all of
// them (4096 x 3584 x 18944: 271 us).
//
// A step has two halves of 64 codes. While the products of a half run, the next
// half's fragments come out of LDS, a read behind every other product. In the
// middle of a step stands its one barrier: every wave has read all of the step's
// stages, and the next step's have arrived; copies into the stages just read are
// issued behind the first products after it.
//
// LDS: three stages of W and two of X, 32 KiB each (160 KiB in all), rows of 128
// bytes with 16-byte unit c of row r at c ^ (r & 7). X's copies are for the step
// after next, W's for the third from there.
constexpr int kTile = 256, kTileStage = kTile * 128, kTileLds = 5 * kTileStage, kTileThreads = 256;
constexpr uint32_t kTileBytes = 1u << 31;  // 256 rows are below it: where copies of zeros point

typedef int i32x16 __attribute__((ext_vector_type(16)));

// (No wait: whoever uses v waits for it with fragments_done, which nothing that uses it can be moved ahead of.)
template <int OFF>
__device__ __forceinline__ void read_fragment(i32x4& v, uint32_t from) {
    asm volatile("ds_read_b128 %0, %1 offset:%2" : "=&v"(v) : "v"(from), "n"(OFF) : "memory");
}
__device__ __forceinline__ void fragments_done(i32x4 (&w)[2][4], i32x4 (&x)[2][4]) {
    asm volatile("s_waitcnt lgkmcnt(0)"
                 : "+v"(w[0][0]), "+v"(w[0][1]), "+v"(w[0][2]), "+v"(w[0][3]), "+v"(w[1][0]), "+v"(w[1][1]), "+v"(w[1][2]), "+v"(w[1][3])
                 :
                 : "memory");
    asm volatile(""
                 : "+v"(x[0][0]), "+v"(x[0][1]), "+v"(x[0][2]), "+v"(x[0][3]), "+v"(x[1][0]), "+v"(x[1][1]), "+v"(x[1][2]), "+v"(x[1][3])
                 :
                 : "memory");
}
// 1 KiB into LDS from a buffer of kTileBytes bytes: 16 bytes a lane, zeros for lanes behind its end.
__device__ __forceinline__ void copy_buffer16(__amdgpu_buffer_rsrc_t from, uint32_t at, uint32_t k, char* to) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(from, (lds_void*)to, 16, at, k, 0, 0);
}

__global__ __launch_bounds__(kTileThreads, 1) void linear_i8_tile_kernel(LinearI8Args a) {
    extern __shared__ __attribute__((aligned(1024))) char tile_lds[];  // W [3] | X [2]
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t wn = wave / 2, wm = wave % 2;
    uint32_t m0, n0;
    {  // blocks of one XCD (b % 8) take tiles that follow one another: panels of 8 tiles of W by all of X
        const uint32_t tn = (a.N + kTile - 1) / kTile, tm = (a.M + kTile - 1) / kTile, tiles = tn * tm;
        const uint32_t xcd = blockIdx.x % 8, per = tiles / 8, rem = tiles % 8;
        const uint32_t u = xcd * per + min(xcd, rem) + blockIdx.x / 8;
        const uint32_t panel = u / (tm * 8), wide = min(8u, tn - 8 * panel), within = u - panel * tm * 8;
        m0 = within / wide * kTile, n0 = (8 * panel + within % wide) * kTile;
    }
    const __amdgpu_buffer_rsrc_t W = __builtin_amdgcn_make_buffer_rsrc(const_cast<int8_t*>(a.W) + n0 * a.ldw, 0, kTileBytes, 0x20000);
    const __amdgpu_buffer_rsrc_t X = __builtin_amdgcn_make_buffer_rsrc(const_cast<int8_t*>(a.X) + m0 * a.ldx, 0, kTileBytes, 0x20000);
    const uint32_t unit = (lane % 8 ^ lane / 8) * 16;  // of a row's 128 codes, what this lane copies
    uint32_t w_at[8], x_at[8];
#pragma unroll
    for (int g = 0; g < 8; ++g) {
        const uint32_t row = wave * 64 + g * 8 + lane / 8;
        w_at[g] = min(row, a.N - 1 - n0) * static_cast<uint32_t>(a.ldw) + unit;
        x_at[g] = min(row, a.M - 1 - m0) * static_cast<uint32_t>(a.ldx) + unit;
    }
    const int steps = static_cast<int>((a.K + 127) / 128);
    auto copy_w = [&](int step, int g) {
        const uint32_t k = step * 128;
        copy_buffer16(W, k + unit < a.K ? w_at[g] : kTileBytes, k, tile_lds + step % 3 * kTileStage + wave * 8192 + g * 1024);
    };
    auto copy_x = [&](int step, int g) {
        const uint32_t k = step * 128;
        copy_buffer16(X, k + unit < a.K ? x_at[g] : kTileBytes, k, tile_lds + (3 + step % 2) * kTileStage + wave * 8192 + g * 1024);
    };
    // (Copies of steps that there are none of are zeros, and what is read of them is never used: no branch is in the way.)
#pragma unroll
    for (int t = 0; t < 2; ++t) {
#pragma unroll
        for (int g = 0; g < 8; ++g) copy_w(t, g);
#pragma unroll
        for (int g = 0; g < 8; ++g) copy_x(t, g);
    }
    i32x16 sum[4][4];
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int e = 0; e < 16; ++e) sum[r][t][e] = 0;
    // Fragments [half of 64][32 codes][tile of 32 rows]: lane l row l % 32, codes 16 (l / 32) .. + 15.
    i32x4 fw[2][2][4], fx[2][2][4];
    const uint32_t at = lane % 32 * 128 + (lane / 32 ^ lane % 8) * 16;
    const uint32_t w_lds = lds_address(tile_lds) + wn * 128 * 128 + at, x_lds = lds_address(tile_lds) + 3 * kTileStage + wm * 128 * 128 + at;
#define TILE_READ(h, i, ws, xs)                                                                        \
    do {                                                                                               \
        constexpr int kk = (i) / 8, what = (i) % 8, tile = what % 4;                                   \
        if constexpr (what < 4) read_fragment<tile * 4096>(fw[h][kk][tile], (ws) ^ ((h) * 64 + kk * 32)); \
        else read_fragment<tile * 4096>(fx[h][kk][tile], (xs) ^ ((h) * 64 + kk * 32));                 \
    } while (0)
#define TILE_PAIR(h, p)                                                                                \
    do {                                                                                               \
        constexpr int kk = (p) / 8, r = (p) % 8 / 2, c = (p) % 2 * 2;                                  \
        sum[r][c] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fx[h][kk][c], fw[h][kk][r], sum[r][c], 0, 0, 0);             \
        sum[r][c + 1] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fx[h][kk][c + 1], fw[h][kk][r], sum[r][c + 1], 0, 0, 0); \
        __builtin_amdgcn_sched_barrier(0);                                                             \
    } while (0)
#define TILE_ALL(X) X(0) X(1) X(2) X(3) X(4) X(5) X(6) X(7) X(8) X(9) X(10) X(11) X(12) X(13) X(14) X(15)
    wait_copies<16>();
    __builtin_amdgcn_s_barrier();
#define FIRST(i) TILE_READ(0, i, w_lds, x_lds);
    TILE_ALL(FIRST)
    fragments_done(fw[0], fx[0]);
    for (int t = 0; t < steps; ++t) {
        const uint32_t ws = w_lds + t % 3 * kTileStage, xs = x_lds + t % 2 * kTileStage;
#define HALF0(i)                                                          \
    TILE_PAIR(0, i);                                                      \
    TILE_READ(1, i, ws, xs);                                              \
    if ((i) % 2 == 0) copy_w(t + 2, (i) / 2);                             \
    __builtin_amdgcn_sched_barrier(0);
        TILE_ALL(HALF0)
        fragments_done(fw[1], fx[1]);
        wait_copies<8>();  // (W's for t + 2 may be in flight)
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
        const uint32_t wt = w_lds + (t + 1) % 3 * kTileStage, xt = x_lds + (t + 1) % 2 * kTileStage;
#define HALF1(i)                                                          \
    TILE_PAIR(1, i);                                                      \
    TILE_READ(0, i, wt, xt);                                              \
    if ((i) % 2 == 0) copy_x(t + 2, (i) / 2);                             \
    __builtin_amdgcn_sched_barrier(0);
        TILE_ALL(HALF1)
        fragments_done(fw[0], fx[0]);
    }
    wait_copies<0>();  // (LDS is not given back with copies on their way)
#undef FIRST
#undef HALF0
#undef HALF1
#undef TILE_ALL
#undef TILE_PAIR
#undef TILE_READ
    // A lane's results are of one row of W (l % 32) for each of r and of the rows 8 e + 4 (l / 32) .. + 3 of X for each of c
    // and e, so that half a wave stores 128 bytes in a row. (As 32 bytes of each of 32 rows, scales read between the
    // stores, a tile's end took 20 us.) All scales are read before the first store: stores count among the loads.
    const uint32_t n = n0 + wn * 128 + lane % 32, m = m0 + wm * 128 + lane / 32 * 4;
    float w_scale[4], bias[4], x_scale[4][16];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const uint32_t at = min(n + r * 32, a.N - 1);
        w_scale[r] = a.w_scales[at], bias[r] = bias_at(a.bias, at);
    }
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int e = 0; e < 16; ++e) x_scale[c][e] = a.x_scales[min(m + c * 32 + e / 4 * 8 + e % 4, a.M - 1)];
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const uint32_t row = m + c * 32 + e / 4 * 8 + e % 4;
            if (row >= a.M) continue;
            float* y = a.Y + row * a.ldy + n;
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (n + r * 32 < a.N) y[r * 32] = finish(sum[r][c][e], x_scale[c][e], w_scale[r], bias[r]);
        }
}

hipError_t launch_tile(const LinearI8Args& a, hipStream_t s) {
    const uint64_t tiles = ((uint64_t{a.N} + kTile - 1) / kTile) * ((uint64_t{a.M} + kTile - 1) / kTile);
    static const hipError_t ready = hipFuncSetAttribute(reinterpret_cast<const void*>(linear_i8_tile_kernel),
                                                        hipFuncAttributeMaxDynamicSharedMemorySize, kTileLds);
    if (ready != hipSuccess) return ready;
    return vlaunch(linear_i8_tile_kernel, dim3(static_cast<uint32_t>(tiles)), dim3(kTileThreads), kTileLds, s, a);
}

hipError_t launch_linear(const LinearI8Args& a, hipStream_t s) {
    const uint64_t stride = std::max(a.ldw, a.ldx);
    if (a.M >= 256 && stride * kTile <= kTileBytes / 2) return launch_tile(a, s);
    if (a.M <= 8) return launch_stream<1, 1, 4, 4>(a, s);
    if (a.M <= 16) return launch_stream<1, 2, 4, 4>(a, s);
    if (a.M <= 32) return launch_stream<2, 4, 3, 4>(a, s);
    return launch_stream<2, 8, 2, 4>(a, s);
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
    a.vector = aligned16(Y) && ldy % 4 == 0 && aligned16(w_scales);
    const hipStream_t st = static_cast<hipStream_t>(stream);
    PAGED_TRY(launch_linear(a, st));
    return VVLI_OK;
}

}  // extern "C"
