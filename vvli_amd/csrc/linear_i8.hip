// linear_i8.hip -- the product of rows of 8-bit codes, a scale for each row of
// both sides (vvli_gpu_linear_i8):
//   Y[m,n] = f32(sum_k W[n,k] X[m,k]) * x_scales[m] * w_scales[n] + bias[n].
//
// The sums are exact in 32 bits, so no split or order of them changes a result.
//
// Up to some 100 rows W's bytes bound it, above them the products, in between what a
// launch and a block's chain of copies, products and stores cost (3.8 us is a launch
// and a block that ends at once). Measured, us (W in no cache; a copy of 256 MB
// moves 5.4 TB/s, a library product of 8192 cubed 2466 TOP/s): 1 x 37888 x 3584 22.0
// (6.2 TB/s), 5 x 2048 x 8192 6.2, 48 x 4608 x 3584 8.4, 128 x 37888 x 3584 37 (4.2
// TB/s), 333 x 896 x 4864 9.7 to 10.1, 2048 x 4608 x 3584 41 (1640 TOP/s), 4096 x 3584 x
// 18944 230 to 238 (2340 to 2420), 4096 x 37888 x 3584 507 to 522 (2130 to 2190).
#include <algorithm>
#include <atomic>
#include <type_traits>
#include <utility>

#include "device_common.hpp"
#include "linear_i8_plan.hpp"
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
    uint32_t split_steps;  // steps of 128 codes of a part of K
    int* parts;            // [part][M][N]
    bool vector;  // Y's rows and w_scales at 16-byte addresses
    bool long_y;  // Y passes the caches
};

constexpr int kOnce = 2;  // cache policy of what passes the caches: nontemporal
// Y that they would not hold till it is read leaves them to W and X (us: 4096 x 37888 x 3584 523, so 507; 2048 x 37888 x
// 3584 270, 265; 4096 x 9728 x 896 72.6, 55.1). Shorter ones are read next out of them (a layer's five calls on 64 rows
// 67.4, so 69.7; on 4096 rows, whose Y is longer, the same either way).
constexpr uint64_t kLongY = uint64_t{128} << 20;
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
    static_assert(MT >= 1 && ((R == 1 && MT <= 3) || (R == 2 && MT <= 4)), "as written");
#define LDS_W(i, at) "ds_read_b128 %" #i ", %[wa] offset:" #at "\n\t"
#define LDS_X(i, at) "ds_read_b128 %" #i ", %[xa] offset:" #at "\n\t"
#define LDS_END "s_waitcnt lgkmcnt(0)"
#define LDS_IN : [wa] "v"(wa), [xa] "v"(xa) : "memory"
    if constexpr (R == 1 && MT == 1)
        asm volatile(LDS_W(0, 0) LDS_X(1, 0) LDS_END : "=&v"(w[0]), "=&v"(x[0]) LDS_IN);
    if constexpr (R == 1 && MT == 2)
        asm volatile(LDS_W(0, 0) LDS_X(1, 0) LDS_X(2, 2048) LDS_END : "=&v"(w[0]), "=&v"(x[0]), "=&v"(x[1]) LDS_IN);
    if constexpr (R == 2 && MT == 1)
        asm volatile(LDS_W(0, 0) LDS_W(1, 2048) LDS_X(2, 0) LDS_END : "=&v"(w[0]), "=&v"(w[1]), "=&v"(x[0]) LDS_IN);
    if constexpr (R == 2 && MT == 2)
        asm volatile(LDS_W(0, 0) LDS_W(1, 2048) LDS_X(2, 0) LDS_X(3, 2048) LDS_END
                     : "=&v"(w[0]), "=&v"(w[1]), "=&v"(x[0]), "=&v"(x[1]) LDS_IN);
    if constexpr (R == 2 && MT == 4)
        asm volatile(LDS_W(0, 0) LDS_W(1, 2048) LDS_X(2, 0) LDS_X(3, 2048) LDS_X(4, 4096) LDS_X(5, 6144) LDS_END
                     : "=&v"(w[0]), "=&v"(w[1]), "=&v"(x[0]), "=&v"(x[1]), "=&v"(x[2]), "=&v"(x[3]) LDS_IN);
    if constexpr (R == 1 && MT == 3)
        asm volatile(LDS_W(0, 0) LDS_X(1, 0) LDS_X(2, 2048) LDS_X(3, 4096) LDS_END
                     : "=&v"(w[0]), "=&v"(x[0]), "=&v"(x[1]), "=&v"(x[2]) LDS_IN);
    if constexpr (R == 2 && MT == 3)
        asm volatile(LDS_W(0, 0) LDS_W(1, 2048) LDS_X(2, 0) LDS_X(3, 2048) LDS_X(4, 4096) LDS_END
                     : "=&v"(w[0]), "=&v"(w[1]), "=&v"(x[0]), "=&v"(x[1]), "=&v"(x[2]) LDS_IN);
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
// before the sums of all meet at the end. Loads into registers instead of copies
// hold as much in flight only with registers that leave fewer waves: 1 x 37888 x
// 3584 32 us, so 22.0. W is read once and passes the caches (nontemporal), X, which
// all blocks read, stays in them.
template <int R, int XG, int ST, int WV>
__global__ __launch_bounds__(WV * 64) void linear_i8_stream_kernel(LinearI8Args a) {
    static_assert(XG == 1 || XG % 2 == 0, "X tiles of 16 rows, or one of 8 twice over");
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
        if (i + 1 < mine) wait_copies<(ST - 1) * D>();  // (the next chunk's may be in flight)
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

// Lets a kernel have `bytes` of dynamic LDS, once on each device.
hipError_t allow_lds(const void* kernel, int bytes, std::atomic<uint64_t>& done) {
    int device = 0;
    hipError_t e = hipGetDevice(&device);
    if (e != hipSuccess) return e;
    const uint64_t bit = uint64_t{1} << (device & 63);
    if (done.load(std::memory_order_relaxed) & bit) return hipSuccess;
    e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == hipSuccess) done.fetch_or(bit, std::memory_order_relaxed);
    return e;
}

template <int R, int XG, int ST, int WV>
hipError_t launch_stream(const LinearI8Args& a, hipStream_t s) {
    constexpr int MT = (XG + 1) / 2, LDS = WV * ST * (2 * R + XG) * 1024;
    static_assert(LDS <= 160 * 1024 && R * MT <= ST * (2 * R + XG) && ST <= 2, "stages, sums and waits fit");
    const uint64_t tn = (uint64_t{a.N} + 16 * R - 1) / (16 * R), tm = (uint64_t{a.M} + 8 * XG - 1) / (8 * XG);
    static std::atomic<uint64_t> ready{0};
    const hipError_t set = allow_lds(reinterpret_cast<const void*>(linear_i8_stream_kernel<R, XG, ST, WV>), LDS, ready);
    if (set != hipSuccess) return set;
    return vlaunch(linear_i8_stream_kernel<R, XG, ST, WV>, dim3(static_cast<uint32_t>((tn + 7) / 8 * 8 * tm)), dim3(WV * 64), LDS, s, a);
}

// ---- more rows: tiles ----------------------------------------------------------
// A block of four waves, 2 over rows of W x 2 over rows of X, 32 RN x 32 RM each.
//
// 4 x 4 (a tile of 256 x 256, one wave on each SIMD of a CU) moves the fewest
// fragment bytes a product that the registers hold (256 of sums, 64 for each of two
// sets of fragments): of a step of 128 codes, 2048 cycles of products, LDS takes 64
// KiB of copies and gives 128 KiB of fragments (eight waves of 128 x 64 read 192
// KiB: 4096 x 3584 x 18944 271 us, four waves 238). Others are for launches whose
// large tiles would leave CUs idle.
//
// What bounds large calls is the card's power: 4096 x 3584 x 18944 runs at 2330 to
// 2390 TOP/s and 4096 x 37888 x 3584, with 620 MB of Y behind its products, at 2190,
// the products busy 60 % of the cycles at a clock of 1.75 to 1.8 of 2.4 GHz. A loop of
// nothing but these products runs at 3400 TOP/s on random codes (4700 on zeros,
// which take no power), with its fragments read from LDS at 2700 to 3000.
//
// A step has two halves of 64 codes. While the products of a half run, the next
// half's fragments come out of LDS and copies for later steps are issued, both
// spread evenly: a wave that has its SIMD to itself must not wait to issue (all of a
// step's copies in one half took 246 us). In the middle of a step stands its one
// barrier: every wave has read all of the step's stages, and the next step's have
// arrived.
//
// LDS: ST stages of X and one more of W, rows of 128 bytes with 16-byte unit c of
// row r at c ^ (r / 2 & 7): what 16 rows hold of one unit lies at 16 places of the
// 256 bytes that a cycle gives. (At c ^ (r & 7), SQ_LDS_BANK_CONFLICT was half of
// SQ_LDS_IDX_ACTIVE, now it is 0: 256 x 3584 x 3584 10.5 us then, 9.9 now, large
// calls the same.) X's copies are issued in a step's second half, into the stage
// just read, W's in the first half of the step after it. 256 x 256 leaves room for
// two stages; smaller tiles take more, since their steps are shorter and what is on
// its way lasts as long.
//
// SPLIT: a block has a part of K and leaves its sums, 32-bit integers, for
// linear_i8_join_kernel. LONG: Y passes the caches.
constexpr int kTileThreads = 256;
constexpr uint32_t kBufferBytes = 1u << 31;  // a tile's rows are below it: copies of zeros point behind it

typedef int i32x16 __attribute__((ext_vector_type(16)));

template <typename F, int... I>
__device__ __forceinline__ void each(F f, std::integer_sequence<int, I...>) {
    (f(std::integral_constant<int, I>{}), ...);
}
template <int N, typename F>
__device__ __forceinline__ void each(F f) {
    each(f, std::make_integer_sequence<int, N>{});
}

// (No wait: whoever uses v calls fragments_done first, and nothing that uses it can be moved ahead of that.)
template <int OFF>
__device__ __forceinline__ void read_fragment(i32x4& v, uint32_t from) {
    asm volatile("ds_read_b128 %0, %1 offset:%2" : "=&v"(v) : "v"(from), "n"(OFF) : "memory");
}
template <int RN, int RM>
__device__ __forceinline__ void fragments_done(i32x4 (&w)[2][RN], i32x4 (&x)[2][RM]) {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
    for (int k = 0; k < 2; ++k) {
#pragma unroll
        for (int r = 0; r < RN; ++r) asm volatile("" : "+v"(w[k][r]));
#pragma unroll
        for (int c = 0; c < RM; ++c) asm volatile("" : "+v"(x[k][c]));
    }
}
// 1 KiB into LDS from a buffer of kBufferBytes: 16 bytes a lane, zeros for lanes behind its end.
__device__ __forceinline__ void copy_buffer16(__amdgpu_buffer_rsrc_t from, uint32_t at, uint32_t k, char* to) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(from, (lds_void*)to, 16, at, k, 0, 0);
}

template <int RN, int RM, int ST>
struct TileShape {
    static constexpr int N = 64 * RN, M = 64 * RM, WStage = N * 128, XStage = M * 128, Lds = (ST + 1) * WStage + ST * XStage;
    static_assert(Lds <= 160 * 1024, "stages fit");
};

template <int RN, int RM, int ST, bool SPLIT, bool LONG>
__global__ __launch_bounds__(kTileThreads, RN * RM >= 9 ? 1 : 2) void linear_i8_tile_kernel(LinearI8Args a) {
    using S = TileShape<RN, RM, ST>;
    constexpr int WG = 2 * RN, XG = 2 * RM;  // copies of a wave a step
    extern __shared__ __attribute__((aligned(1024))) char tile_lds[];  // W [ST + 1] | X [ST]
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t wn = wave / 2, wm = wave % 2;
    uint32_t m0, n0;
    {  // blocks of one XCD (b % 8) take tiles that follow one another: panels of 8 tiles of W by all of X
        const uint32_t tn = (a.N + S::N - 1) / S::N, tm = (a.M + S::M - 1) / S::M, tiles = tn * tm;
        const uint32_t xcd = blockIdx.x % 8, per = tiles / 8, rem = tiles % 8;
        const uint32_t u = xcd * per + min(xcd, rem) + blockIdx.x / 8;
        const uint32_t panel = u / (tm * 8), wide = min(8u, tn - 8 * panel), within = u - panel * tm * 8;
        m0 = within / wide * S::M, n0 = (8 * panel + within % wide) * S::N;
    }
    const __amdgpu_buffer_rsrc_t W = __builtin_amdgcn_make_buffer_rsrc(const_cast<int8_t*>(a.W) + n0 * a.ldw, 0, kBufferBytes, 0x20000);
    const __amdgpu_buffer_rsrc_t X = __builtin_amdgcn_make_buffer_rsrc(const_cast<int8_t*>(a.X) + m0 * a.ldx, 0, kBufferBytes, 0x20000);
    // Of a row's 128 codes, what this lane copies (g: of 8 rows, odd and even ones alternate, WG and XG being even).
    auto unit = [&](int g) { return (lane % 8 ^ lane / 16 ^ g % 2 * 4) * 16; };
    uint32_t w_at[WG], x_at[XG];
#pragma unroll
    for (int g = 0; g < WG; ++g) w_at[g] = min((wave * WG + g) * 8 + lane / 8, a.N - 1 - n0) * static_cast<uint32_t>(a.ldw) + unit(g);
#pragma unroll
    for (int g = 0; g < XG; ++g) x_at[g] = min((wave * XG + g) * 8 + lane / 8, a.M - 1 - m0) * static_cast<uint32_t>(a.ldx) + unit(g);
    const int all_steps = static_cast<int>((a.K + 127) / 128);
    const int first = SPLIT ? static_cast<int>(blockIdx.y * a.split_steps) : 0, steps = SPLIT ? min(static_cast<int>(a.split_steps), all_steps - first) : all_steps;
    const uint32_t k_first = first * 128, k_end = min(k_first + steps * 128, a.K);
    // Each XCD starts at another eighth of the steps and goes round. All blocks at the same columns of rows that are an even
    // number of 256 bytes apart would meet in few of the memory's channels (512 x 4608 x 14336: 73 us).
    const int turn = steps * static_cast<int>((blockIdx.x + blockIdx.y * gridDim.x) % 8) / 8;
    // (Copies of steps that there are none of are zeros, and what is read of them is never used: no branch is in the way.)
    auto k_of = [&](int step) { return k_first + (step + turn < steps ? step + turn : step + turn - steps) * 128; };
    auto end_of = [&](int step) { return step < steps ? k_end : 0; };
    auto copy_w = [&](int step, int g) {
        const uint32_t k = k_of(step);
        copy_buffer16(W, k + unit(g) < end_of(step) ? w_at[g] : kBufferBytes, k, tile_lds + step % (ST + 1) * S::WStage + (wave * WG + g) * 1024);
    };
    auto copy_x = [&](int step, int g) {
        const uint32_t k = k_of(step);
        copy_buffer16(X, k + unit(g) < end_of(step) ? x_at[g] : kBufferBytes, k,
                      tile_lds + (ST + 1) * S::WStage + step % ST * S::XStage + (wave * XG + g) * 1024);
    };
    for (int t = 0; t < ST; ++t) {
#pragma unroll
        for (int g = 0; g < WG; ++g) copy_w(t, g);
#pragma unroll
        for (int g = 0; g < XG; ++g) copy_x(t, g);
    }
    i32x16 sum[RN][RM];
#pragma unroll
    for (int r = 0; r < RN; ++r)
#pragma unroll
        for (int c = 0; c < RM; ++c)
#pragma unroll
            for (int e = 0; e < 16; ++e) sum[r][c][e] = 0;
    // Fragments [half of 64][32 codes][32 rows]: lane l row l % 32, codes 16 (l / 32) .. + 15.
    i32x4 fw[2][2][RN], fx[2][2][RM];
    const uint32_t at = lane % 32 * 128 + (lane / 32 ^ lane / 2 % 8) * 16;
    const uint32_t w_lds = lds_address(tile_lds) + wn * (RN * 4096) + at;
    const uint32_t x_lds = lds_address(tile_lds) + (ST + 1) * S::WStage + wm * (RM * 4096) + at;
    constexpr int P = 2 * RN * RM, R = 2 * (RN + RM);  // products and reads of a half
    auto read = [&](auto half, auto i, uint32_t ws, uint32_t xs) {
        constexpr int h = half, k = i / (RN + RM), what = i % (RN + RM);
        if constexpr (what < RN) read_fragment<what * 4096>(fw[h][k][what], ws ^ (h * 64 + k * 32));
        else read_fragment<(what - RN) * 4096>(fx[h][k][what - RN], xs ^ (h * 64 + k * 32));
    };
    // The products of half h with reads and copies spread among them.
    auto half = [&](auto h, uint32_t ws, uint32_t xs, int step) {
        constexpr int C = h ? XG : WG;
        each<P>([&](auto p) {
            constexpr int k = p / (RN * RM), r = p / RM % RN, c = p % RM;
            sum[r][c] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fx[h][k][c], fw[h][k][r], sum[r][c], 0, 0, 0);
            __builtin_amdgcn_sched_barrier(0);
            constexpr int r0 = p * R / P, r1 = (p + 1) * R / P, c0 = p * C / P, c1 = (p + 1) * C / P;
            each<r1 - r0>([&](auto i) { read(std::integral_constant<int, 1 - h>{}, std::integral_constant<int, r0 + i>{}, ws, xs); });
            each<c1 - c0>([&](auto i) {
                if constexpr (h) copy_x(step, c0 + i);
                else copy_w(step, c0 + i);
            });
            __builtin_amdgcn_sched_barrier(0);
        });
        fragments_done(fw[1 - h], fx[1 - h]);
    };
    using Zero = std::integral_constant<int, 0>;
    using One = std::integral_constant<int, 1>;
    wait_copies<(ST - 1) * (WG + XG)>();
    __builtin_amdgcn_s_barrier();
    each<R>([&](auto i) { read(Zero{}, i, w_lds, x_lds); });
    fragments_done(fw[0], fx[0]);
    for (int t = 0; t < steps; ++t) {
        half(Zero{}, w_lds + t % (ST + 1) * S::WStage, x_lds + t % ST * S::XStage, t + ST);
        wait_copies<(ST - 1) * WG + (ST - 2) * XG>();  // (those for t + 2 and later may be in flight)
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
        half(One{}, w_lds + (t + 1) % (ST + 1) * S::WStage, x_lds + (t + 1) % ST * S::XStage, t + ST);
    }
    wait_copies<0>();  // (LDS is not given back with copies on their way)
    // A lane's results are of one row of W (l % 32) for each of r and of the rows 8 e + 4 (l / 32) .. + 3 of X for each of c
    // and e, so that half a wave stores 128 bytes in a row. (As 32 bytes of each of 32 rows, scales read between the
    // stores, a tile's end took 20 us.) All scales are read before the first store: stores count among the loads.
    const uint32_t n = n0 + wn * (32 * RN) + lane % 32, m = m0 + wm * (32 * RM) + lane / 32 * 4;
    // Y (or the part's sums) from this tile on: rows behind M are behind the buffer's end, columns behind N are sent there.
    // What differs between a lane's results is the same for all lanes, so that a store takes no address arithmetic of its
    // own (with it, and a branch for each row, the end of a tile of 256 x 256 took 9 us more).
    const uint32_t rows = min(a.M - m0, S::M + 0u), pitch = SPLIT ? a.N * 4 : static_cast<uint32_t>(a.ldy) * 4;
    void* const out = SPLIT ? static_cast<void*>(a.parts + (static_cast<size_t>(blockIdx.y) * a.M + m0) * a.N + n0) : a.Y + m0 * a.ldy + n0;
    const __amdgpu_buffer_rsrc_t Y = __builtin_amdgcn_make_buffer_rsrc(out, 0, (rows - 1) * pitch + min(a.N - n0, S::N + 0u) * 4, 0x20000);
    const __amdgpu_buffer_rsrc_t x_scales = __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(a.x_scales) + m0, 0, rows * 4, 0x20000);
    float w_scale[RN], bias[RN];
    f32x4 x_scale[RM][4];
    uint32_t y_at[RN];
#pragma unroll
    for (int r = 0; r < RN; ++r) {
        const uint32_t row = min(n + r * 32, a.N - 1);
        y_at[r] = n + r * 32 < a.N ? (m - m0) * pitch + (n - n0 + r * 32) * 4 : kBufferBytes;
        if constexpr (!SPLIT) w_scale[r] = a.w_scales[row], bias[r] = bias_at(a.bias, row);
    }
    if constexpr (!SPLIT) {
#pragma unroll
        for (int c = 0; c < RM; ++c)
#pragma unroll
            for (int q = 0; q < 4; ++q)
                x_scale[c][q] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(x_scales, (m - m0 + c * 32 + q * 8) * 4, 0, 0));
    }
#pragma unroll
    for (int c = 0; c < RM; ++c)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const uint32_t down = (c * 32 + e / 4 * 8 + e % 4) * pitch;
#pragma unroll
            for (int r = 0; r < RN; ++r) {
                uint32_t value = sum[r][c][e];
                if constexpr (!SPLIT) value = __float_as_uint(finish(sum[r][c][e], x_scale[c][e / 4][e % 4], w_scale[r], bias[r]));
                __builtin_amdgcn_raw_buffer_store_b32(value, Y, y_at[r], down, LONG ? kOnce : 0);
            }
        }
}

// Adds the parts of a split K and finishes them, four results of a row of Y a thread.
__global__ __launch_bounds__(256) void linear_i8_join_kernel(LinearI8Args a, uint32_t splits) {
    const uint32_t quads = (a.N + 3) / 4;
    const size_t size = static_cast<size_t>(a.M) * a.N;
    for (uint32_t i = blockIdx.x * 256 + threadIdx.x; i < quads * a.M; i += gridDim.x * 256) {
        const uint32_t m = i / quads, n = i % quads * 4;
        const int* p = a.parts + static_cast<size_t>(m) * a.N + n;
        i32x4 v = {0, 0, 0, 0};
        if (a.N % 4 == 0) {
            for (uint32_t z = 0; z < splits; ++z) v += *reinterpret_cast<const i32x4*>(p + z * size);
        } else {
            for (uint32_t z = 0; z < splits; ++z)
                for (int j = 0; j < 4; ++j)
                    if (n + j < a.N) v[j] += p[z * size + j];
        }
        store4(a, m, n, v);
    }
}

template <int RN, int RM, int ST, bool LONG = false>
hipError_t launch_tile(const LinearI8Args& a, hipStream_t s) {
    using S = TileShape<RN, RM, ST>;
    if constexpr (!LONG && RN * RM >= 4 && ST == 2) {  // (others hardly ever have a long Y)
        if (a.long_y) return launch_tile<RN, RM, ST, true>(a, s);
    }
    const uint64_t tiles = ((uint64_t{a.N} + S::N - 1) / S::N) * ((uint64_t{a.M} + S::M - 1) / S::M);
    static std::atomic<uint64_t> ready{0};
    const auto kernel = linear_i8_tile_kernel<RN, RM, ST, false, LONG>;
    const hipError_t set = allow_lds(reinterpret_cast<const void*>(kernel), S::Lds, ready);
    if (set != hipSuccess) return set;
    return vlaunch(kernel, dim3(static_cast<uint32_t>(tiles)), dim3(kTileThreads), S::Lds, s, a);
}
// K in `splits` parts (at most; each has steps), their sums in the workspace.
template <int RN, int RM, int ST>
hipError_t launch_tile_split(LinearI8Args a, uint32_t splits, hipStream_t s) {
    using S = TileShape<RN, RM, ST>;
    const uint32_t tiles = ((a.N + S::N - 1) / S::N) * ((a.M + S::M - 1) / S::M), steps = (a.K + 127) / 128;
    static std::atomic<uint64_t> ready{0};
    const hipError_t set = allow_lds(reinterpret_cast<const void*>(linear_i8_tile_kernel<RN, RM, ST, true, false>), S::Lds, ready);
    if (set != hipSuccess) return set;
    a.split_steps = (steps + splits - 1) / splits;
    splits = (steps + a.split_steps - 1) / a.split_steps;
    const hipError_t e = vlaunch(linear_i8_tile_kernel<RN, RM, ST, true, false>, dim3(tiles, splits), dim3(kTileThreads), S::Lds, s, a);
    if (e != hipSuccess) return e;
    const uint32_t quads = (a.N + 3) / 4 * a.M;
    return vlaunch(linear_i8_join_kernel, dim3(std::min((quads + 255) / 256, 2048u)), dim3(256), 0, s, a, splits);
}

template <uint32_t I>
hipError_t launch_kernel(const LinearI8Args& a, const I8Plan& plan, hipStream_t s) {
    constexpr I8Kernel k = kI8Kernels[I];
    if constexpr (k.kind == kI8Stream) return launch_stream<k.r, k.m, k.stages, k.waves>(a, s);
    else if constexpr (k.split) return launch_tile_split<k.r, k.m, k.stages>(a, plan.splits, s);
    else return launch_tile<k.r, k.m, k.stages>(a, s);
}
template <uint32_t... I>
hipError_t launch_plan(const LinearI8Args& a, const I8Plan& plan, hipStream_t s, std::integer_sequence<uint32_t, I...>) {
    hipError_t e = hipErrorInvalidValue;
    (void)((plan.kernel == I && (e = launch_kernel<I>(a, plan, s), true)) || ...);
    return e;
}

hipError_t launch_linear(const LinearI8Args& a, hipStream_t s) {
    hipError_t e = hipSuccess;
    auto launch = [&](const I8Plan& plan, uint64_t m0, uint64_t M, uint64_t n0, uint64_t N) {
        LinearI8Args b = a;
        b.M = static_cast<uint32_t>(M), b.N = static_cast<uint32_t>(N);
        b.W += n0 * a.ldw, b.w_scales += n0, b.X += m0 * a.ldx, b.x_scales += m0, b.Y += m0 * a.ldy + n0;
        if (b.bias) b.bias += n0;
        e = launch_plan(b, plan, s, std::make_integer_sequence<uint32_t, kI8KernelCount>{});
        return e == hipSuccess;
    };
    i8_launches(a.M, a.N, a.K, std::max(std::max(a.ldw, a.ldx), a.ldy * 4), gemm_cus(), launch);
    return e;
}

bool sizes_ok(uint32_t M, uint32_t N, uint32_t K) {
    return M < kPagedMost && N > 0 && N < kPagedMost && K > 0 && K <= kMostK && K % kCodesPerUnit == 0;
}

}  // namespace

extern "C" {

size_t vvli_gpu_linear_i8_workspace(uint32_t M, uint32_t N, uint32_t K) { return sizes_ok(M, N, K) ? i8_part_bytes(M, N, K) : 0; }

int vvli_gpu_linear_i8(const int8_t* W, uint64_t ldw, const float* w_scales, const int8_t* X, uint64_t ldx,
                       const float* x_scales, const uint16_t* bias, float* Y, uint64_t ldy, uint32_t M, uint32_t N,
                       uint32_t K, void* workspace, size_t workspace_bytes, void* stream) {
    const char* who = "vvli_gpu_linear_i8";
    if (!W || !w_scales || !X || !x_scales || !Y) return set_error(VVLI_NULL_ARG, "NULL argument to %s", who);
    if (!sizes_ok(M, N, K))
        return set_error(VVLI_INVALID_CONFIG, "%s: bad sizes M=%u N=%u K=%u (K: whole 16s up to %u)", who, M, N, K, kMostK);
    int rc;
    if ((rc = check_row_units(W, ldw, K, 1, "W", who)) || (rc = check_row_units(X, ldx, K, 1, "X", who))) return rc;
    if (ldy < N || ldy >= kPagedMost)
        return set_error(VVLI_INVALID_CONFIG, "%s: rows of Y of %u (stride %llu)", who, N, static_cast<unsigned long long>(ldy));
    const size_t need = vvli_gpu_linear_i8_workspace(M, N, K);
    if (need && !workspace) return set_error(VVLI_NULL_ARG, "%s: NULL workspace", who);
    if (need && (!aligned16(workspace) || workspace_bytes < need))
        return set_error(VVLI_INVALID_CONFIG, "%s: workspace of %zu bytes", who, workspace_bytes);
    const RowBytes y{Y, ldy * 4, uint64_t{N} * 4, M}, space{workspace, need, need, 1};
    const RowBytes inputs[] = {{W, ldw, K, N}, {X, ldx, K, M}, {w_scales, 4, 4, N}, {x_scales, 4, 4, M}, {bias, 2, 2, N}};
    for (const RowBytes& in : inputs)
        if (rows_meet(y, in) || rows_meet(space, in)) return set_error(VVLI_INVALID_CONFIG, "%s: Y or the workspace overlaps an input", who);
    if (rows_meet(y, space)) return set_error(VVLI_INVALID_CONFIG, "%s: Y overlaps the workspace", who);
    if (M == 0) return VVLI_OK;
    LinearI8Args a{};
    a.W = W, a.X = X, a.w_scales = w_scales, a.x_scales = x_scales, a.bias = bias, a.Y = Y;
    a.ldw = ldw, a.ldx = ldx, a.ldy = ldy, a.M = M, a.N = N, a.K = K;
    a.parts = static_cast<int*>(workspace);
    a.vector = aligned16(Y) && ldy % 4 == 0 && aligned16(w_scales), a.long_y = uint64_t{M} * N * 4 > kLongY;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    PAGED_TRY(launch_linear(a, st));
    return VVLI_OK;
}

}  // extern "C"
