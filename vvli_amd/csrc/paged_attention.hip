// paged_attention.hip -- attention of the new rows of several requests over
// their pages (vvli_gpu_paged_attention).
//
// For a row at position p, with j over the positions that it sees,
//   o = sum_j e^(s_j) v_j / sum_j e^(s_j),   s_j = scale q . k_j,
// in one pass over the keys: a running maximum m, the sum l of 2^(s_j - m)
// (scores in base 2 for v_exp_f32) and the output so far, both rescaled where
// m grows; parts over different keys join by the same rescaling.
//
// A vector is one (row, query head); the G vectors of a row that share a kv
// head, and the rows behind one another, stand together so that a key is read
// once for all of them. An item is up to M such vectors of one request and kv
// head. Its keys are counted in units of UK positions from position 0, and the
// units of all items, in the order (request, kv head, vectors, keys), are cut
// into equal runs, one for each block: no batch, whatever its lengths, leaves
// blocks with more to do than others. An item that a run's end cuts leaves its
// parts in the workspace, and the block whose part is there last joins all of
// them in order of keys, so results do not depend on timing.
//
// Two kernels: one for few rows a request (single tokens, drafts), which reads
// the cache at memory's rate, and one for prompts' chunks, which matrix products
// bound. What they do not take from either is the chain of a short call: some
// 3 us to find a block's run, 2 to an item's first keys, 1 to 2 a step and 5 to
// 10 for an item's parts.
#include <hip/hip_fp16.h>

#include <algorithm>

#include "device_common.hpp"
#include "paged.hpp"
#include "paged_runs.hpp"

using namespace vvli;

namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kThreads = 256;
struct PagedAttnArgs {
    const void *k, *v;
    const int32_t *table, *row_start, *start_pos;
    const float* q;
    float* out;
    uint32_t* arrived;  // of each block: parts that are there of the item that its run's end cut; 0 between calls
    float* parts;       // two slots for each block: [slot_vecs][HD] outputs, [slot_vecs] maxima and sums
    uint64_t slot_stride, ldq, ldo;
    uint32_t stride, requests, rows, kv_heads, window, pages, room, slot_vecs;
    PageDiv ps, group;
    float scale;
};

// ---------------------------------------------------------------------------
// Items and runs
// ---------------------------------------------------------------------------
__device__ __forceinline__ Request request_at(const PagedAttnArgs& a, uint32_t r) {
    const RowSpan s = row_span(a.row_start[r], a.row_start[r + 1], a.rows);
    return Request{s.first, s.count * a.group.d, a.start_pos[r]};
}

__device__ __forceinline__ uint64_t wave_scan(uint64_t v) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint64_t u = __shfl_up(v, o, 64);
        if (lane >= o) v += u;
    }
    return v;
}

// Units of one kv head of each lane's request, summed over its items: by the
// lane itself where they are few, else by its wave.
template <class S>
__device__ __forceinline__ uint64_t request_units(const PagedAttnArgs& a, const Request& q) {
    const uint32_t lane = threadIdx.x & 63, items = (q.vecs + S::M - 1) / S::M;
    uint64_t sum = 0;
    if (items <= 2)
        for (uint32_t i = 0; i < items; ++i) sum += units_of<S>(a, q, i * S::M).count;
    for (uint64_t todo = __ballot(items > 2); todo; todo &= todo - 1) {
        const int from = __builtin_ctzll(todo);
        const Request f{static_cast<uint32_t>(__shfl(q.first, from, 64)), static_cast<uint32_t>(__shfl(q.vecs, from, 64)),
                        __shfl(q.start, from, 64)};
        uint64_t s = 0;
        for (uint32_t i = lane; i < (f.vecs + S::M - 1) / S::M; i += 64) s += units_of<S>(a, f, i * S::M).count;
#pragma unroll
        for (int o = 32; o; o >>= 1) s += __shfl_xor(s, o, 64);
        if (static_cast<int>(lane) == from) sum = s;
    }
    return sum;
}

// A block's run (see Borders).
struct Run {
    uint64_t from, to;                // global units, before the borders move
    Borders at;
    uint32_t r, kvh, m0, unit;        // the item that holds unit `from`, and which unit of it that is
    uint32_t index;
    Request req;  // of r
    bool any;
};

struct RunScratch {
    uint64_t sums[kThreads / 64], found_rest, found_units;
    Request found;
    uint32_t found_r, last;
};

template <class S>
__device__ Run find_run(const PagedAttnArgs& a, RunScratch& sc) {
    const uint32_t blocks = gridDim.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const uint32_t chunks = (a.requests + kThreads - 1) / kThreads;
    uint64_t mine = 0, end = 0, before = 0;
    Request own{};
    auto chunk = [&](uint32_t c) {  // this thread's request's units, and the sum up to it
        const uint32_t r = c * kThreads + tid;
        own = r < a.requests ? request_at(a, r) : Request{0, 0, 0};
        mine = request_units<S>(a, own);
        const uint64_t s = wave_scan(mine);
        __syncthreads();
        if (lane == 63) sc.sums[wave] = s;
        __syncthreads();
        end = before + s;
        for (uint32_t w = 0; w < kThreads / 64; ++w) {
            if (w < wave) end += sc.sums[w];
            before += sc.sums[w];
        }
    };
    for (uint32_t c = 0; c < chunks; ++c) chunk(c);
    const uint64_t total = before * a.kv_heads;
    Run run{};
    run.at = borders_of<S>(total, blocks);
    run.index = run_of_block(blockIdx.x, blocks, run.at.runs);
    if (run.index >= run.at.runs) return run;
    run.from = run.at.per * run.index;
    run.to = min(run.from + run.at.per, total);
    run.any = true;
    before = 0;
    for (uint32_t c = 0; c < chunks; ++c) {
        if (chunks > 1) chunk(c);
        const uint64_t lo = (end - mine) * a.kv_heads;
        if (mine && run.from >= lo && run.from < end * a.kv_heads)
            sc.found_r = c * kThreads + tid, sc.found = own, sc.found_rest = run.from - lo, sc.found_units = mine;
    }
    __syncthreads();
    run.r = __builtin_amdgcn_readfirstlane(sc.found_r);
    const uint64_t rest = sc.found_rest, units = sc.found_units;
    run.kvh = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(quotient(rest, units)));
    uint64_t v = rest - run.kvh * units;
    const Request q{static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(sc.found.first)),
                    static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(sc.found.vecs)),
                    __builtin_amdgcn_readfirstlane(static_cast<int32_t>(sc.found.start))};
    run.req = q;
    for (uint32_t i = 0;; i += 64) {  // every wave by itself: the item that holds unit v
        const uint32_t m = (i + lane) * S::M;
        const uint64_t s = wave_scan(m < q.vecs ? units_of<S>(a, q, m).count : 0);
        const uint64_t past = __ballot(s > v);
        if (past || (i + 64) * S::M >= q.vecs) {
            const int at = past ? __builtin_ctzll(past) : 0;
            const uint64_t prev = __shfl(s, at ? at - 1 : 0, 64);
            run.m0 = __builtin_amdgcn_readfirstlane((i + at) * S::M);
            run.unit = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(at ? v - prev : v));
            return run;
        }
        v -= __shfl(s, 63, 64);
    }
}

// A block's way through its run: the item that it is at, and which of the
// item's units are its own.
template <class S>
struct Walk {
    Run run;
    Request req;
    uint64_t start;  // global unit where the item starts
    bool begun;      // the run starts inside the item
    Units un;
    Part part;
    __device__ __forceinline__ uint32_t first_unit() const { return un.first + (part.t0 > S::kItem ? part.t0 - S::kItem : 0); }  // of its keys
    __device__ __forceinline__ uint32_t end_unit() const { return un.first + (part.t1 > S::kItem ? part.t1 - S::kItem : 0); }

    __device__ __forceinline__ explicit Walk(const PagedAttnArgs& a, const Run& r) : run(r) {
        req = run.req;
        start = run.from - run.unit;
        begun = true;
    }
    // The first request from r on that has rows. (Idle ones are looked at 64 at a time: one after the other, 254
    // between two that have rows made 22 us 56 us.)
    __device__ __forceinline__ static uint32_t with_rows(const PagedAttnArgs& a, uint32_t r) {
        for (; r < a.requests; r += 64) {
            const uint32_t i = r + (threadIdx.x & 63);
            const uint64_t some = __ballot(i < a.requests && row_span(a.row_start[i], a.row_start[i + 1], a.rows).count != 0);
            if (some) return r + __builtin_ctzll(some);
        }
        return a.requests;
    }
    __device__ __forceinline__ bool item(const PagedAttnArgs& a) {  // false: the run has ended
        for (;; begun = false) {
            if (start >= run.to) return false;
            while (run.m0 >= req.vecs) {  // the next item with vectors
                run.m0 = 0;
                if (req.vecs == 0 || ++run.kvh == a.kv_heads) {
                    run.kvh = 0;
                    if (++run.r == a.requests) return false;
                    req = request_at(a, run.r);
                    if (__builtin_expect(req.vecs == 0, 0)) {
                        run.r = __builtin_amdgcn_readfirstlane(with_rows(a, run.r));
                        if (run.r == a.requests) return false;
                        req = request_at(a, run.r);
                    }
                }
            }
            un = units_of<S>(a, req, run.m0);
            const Share share = part_of<S>(run.at, un, start, run.to, run.unit, begun, part);
            if (share == Share::kNone) {
                next();
                continue;
            }
            return share == Share::kPart;
        }
    }
    __device__ __forceinline__ void next() { start += un.count, run.m0 += S::M, begun = false; }
    __device__ __forceinline__ uint32_t vecs() const { return min(static_cast<uint32_t>(S::M), req.vecs - run.m0); }
    __device__ __forceinline__ bool whole() const { return part.t0 == 0 && part.t1 == un.count; }
    __device__ __forceinline__ uint64_t border() const { return first_border(run.at, start); }
    __device__ __forceinline__ uint32_t parts() const { return parts_of(run.at, start, un.count); }
};

// Parts go through to memory (agent-scope stores and loads): other XCDs read them.
__device__ __forceinline__ void publish(float* p, float x, float y) {
    __hip_atomic_store(reinterpret_cast<uint64_t*>(p), static_cast<uint64_t>(__float_as_uint(y)) << 32 | __float_as_uint(x),
                       __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float2 fetch(const float* p) {
    const uint64_t w = __hip_atomic_load(reinterpret_cast<const uint64_t*>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return make_float2(__uint_as_float(static_cast<uint32_t>(w)), __uint_as_float(static_cast<uint32_t>(w >> 32)));
}
// Whether this block's part, which all its threads have published, is the item's last.
__device__ __forceinline__ bool last_part(uint32_t* arrived, uint32_t n, uint32_t& shared) {
    __builtin_amdgcn_s_waitcnt(0);  // this thread's stores are in memory
    __syncthreads();
    if (threadIdx.x == 0) {
        shared = __hip_atomic_fetch_add(arrived, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == n - 1;
        if (shared) __hip_atomic_store(arrived, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);  // for the next call
    }
    __syncthreads();
    if (!shared) return false;
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");
    return true;
}

// ---------------------------------------------------------------------------
// Cache types. 16-bit caches go through 16x16x32 products; an f32 operand is
// split into TERMS values of the type whose sum is it: x = t0 + t1 + ..., each
// the rounding of what is left. bf16 has 8 bits, so three terms hold 24; f16
// has 11, so two hold 22 (the rest, 2^-22 of x at most and half of that on
// average, is what rounding a product to f32 leaves too). f16 has few
// exponents: q is scaled by a power of two to below 2^13 (and the scores back),
// and the largest weight to 2^15 or, in chunks, whose scale follows the largest
// at a distance, 2^11 at least: terms are off by half of f16's smallest
// step, 2^-25, so that a weight is by 2^-36 of the largest at most. (With the
// largest at 2^5, a key 2^31 times as heavy as thousands of others hid them.)
// 2^15 times f16's largest value times the number of keys stays far below f32's
// end. An f32 cache goes through 16x16x4 products of f32.
// ---------------------------------------------------------------------------
template <int KIND> struct Kind;
template <> struct Kind<VVLI_CACHE_F32> {
    static constexpr int TERMS = 1, BYTES = 4, U = 1;
    static constexpr float TOP = 0.f;
};
template <> struct Kind<VVLI_CACHE_BF16> {
    static constexpr int TERMS = 3, BYTES = 2, U = 2;
    static constexpr float TOP = 0.f;
    typedef __bf16 T;
    typedef bf16x8 T8;
    static __device__ __forceinline__ f32x4 mfma(T8 x, T8 y, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, y, c, 0, 0, 0); }
    static __device__ __forceinline__ f32x16 mfma(T8 x, T8 y, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(x, y, c, 0, 0, 0); }
};
template <> struct Kind<VVLI_CACHE_F16> {
    static constexpr int TERMS = 2, BYTES = 2, U = 2;
    static constexpr float TOP = 15.f;
    typedef _Float16 T;
    typedef f16x8 T8;
    static __device__ __forceinline__ f32x4 mfma(T8 x, T8 y, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(x, y, c, 0, 0, 0); }
    static __device__ __forceinline__ f32x16 mfma(T8 x, T8 y, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(x, y, c, 0, 0, 0); }
};

template <typename K>
__device__ __forceinline__ void split(float x, int e, typename K::T8 (&t)[K::TERMS]) {
#pragma unroll
    for (int i = 0; i < K::TERMS; ++i) {
        const typename K::T h = static_cast<typename K::T>(x);
        t[i][e] = h;
        x -= static_cast<float>(h);
    }
}

// Maximum over the four lanes that hold a vector's scores (l % 16 alike).
__device__ __forceinline__ float rows_max(float x) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    const float y = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(y), __float_as_uint(y), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

// Terms of two neighbouring values. bf16: the first two by cutting off, so that
// what is left is exact and one v_perm packs a pair, the last (8 bits are left)
// by rounding.
template <typename K>
__device__ __forceinline__ void split2(float x, float y, int e, typename K::T8 (&t)[K::TERMS]) {
    if constexpr (K::TERMS == 3) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint32_t a = __float_as_uint(x), b = __float_as_uint(y);
            u32x4 w = __builtin_bit_cast(u32x4, t[i]);
            w[e / 2] = __builtin_amdgcn_perm(b, a, 0x07060302u);
            t[i] = __builtin_bit_cast(typename K::T8, w);
            x -= __uint_as_float(a & 0xffff0000u), y -= __uint_as_float(b & 0xffff0000u);
        }
        t[2][e] = static_cast<typename K::T>(x), t[2][e + 1] = static_cast<typename K::T>(y);
    } else {
        split<K>(x, e, t), split<K>(y, e + 1, t);
    }
}
// What is added to scores for weights of 2^bias at m. Where f32's steps at m are over 1, bias - m is rounded, and weights
// that are 2^16 or more for it are none in f16: there it is -m.
template <typename K>
__device__ __forceinline__ float shift_of(float bias, float m) {
    const float x = bias - m;
    return K::TOP > 0.f && x + m > bias + 0.5f ? -m : x;
}
// The power of two that brings a row of q with this largest value below 2^13.
__device__ __forceinline__ int f16_exponent(float top) {
    const int ex = top > 0.f && top < INFINITY ? 13 - (ilogbf(top) + 1) : 0;
    return min(max(ex, -120), 120);
}

// A product's result may be read so many wait states behind it (18 for the
// longest, 32 x 32 x 2 in f32). The compiler counts these along one way to a
// read; where a branch lies between the two, the other way can be shorter, and
// the last register of a result was then read before it was written. Here they
// are spent before any branch: behind chunks' scores and, in both kernels,
// behind the loop over the keys (inside it outputs are read behind the next
// step's scores). Behind the scores of few rows they cost one row behind 8000
// 0.5 of 21.1 us in bf16, so that there it is the compiler's count, as a test
// of the kernels' listing finds it.
template <typename V, int N>
__device__ __forceinline__ void mfma_done(V (&x)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) asm volatile("" : "+v"(x[i]));
    asm volatile("s_nop 15\n\ts_nop 3");
#pragma unroll
    for (int i = 0; i < N; ++i) asm volatile("" : "+v"(x[i]));
}

// ---------------------------------------------------------------------------
// A wave holds WV = 16 vectors of an item and takes WK = 16 U positions a
// step; waves that share vectors join at the item's end. Nothing is shared
// between waves on the way, so keys and values go from memory (or the caches,
// where waves read the same ones) straight into the registers that the products
// read, the next step's keys and values in flight behind this one's:
//   S^T = K Q^T  A: lane l has key l % 16, dims 32 s + 8 (l / 16) .. + 7 (16-bit)
//                   or 16 s + 4 (l / 16) + e (f32); D: lane l has keys
//                   4 (l / 16) + j of vector l % 16
//   O^T += V^T P^T  B: a lane's own scores, keys 16 u + 4 (l / 16) + j as the
//                   k index (u, j); A: row i of tile e is dim DV i + e, so that
//                   a lane loads DV = HD / 16 adjacent dims of each of its
//                   keys; 16-bit pairs of keys are put together by v_perm
// The first term of q stays in registers, the others in LDS: two waves fit a
// SIMD, one's products beside the other's exponentials.
//
// Keys and values from memory bound it where requests are many or long: 40 rows
// behind up to 8000 positions, 28 heads over 4 of 128, bf16, 83 us, 4.4 TB/s (a
// copy reaches 4.8 to 5.4), and 144 us, 5.0 TB/s, in f32; 64 behind up to 4000,
// 16 heads over 16 of 128, 232 us, 5.5 TB/s, and 418 us, 6.1 TB/s, in f32. The
// chain named above does where they are few: 1 row behind 230, 8 kv heads of
// 64, f32, 11 us; behind 8000, 4 kv heads of 128, bf16, 21 us; 24 x 5 rows
// behind up to 4100, f16, 40 us, 2.8 TB/s.
// ---------------------------------------------------------------------------
template <int HD, int KIND>
struct Form {
    using K = Kind<KIND>;
    static constexpr int WV = 16, M = 4 * WV, U = K::U, WK = 16 * U, DV = HD / 16;
    using S = FewCuts<U>;
    static_assert(S::M == M && S::WK == WK);
    static constexpr int KL = HD * K::BYTES / 64;   // 16-byte loads of a key row by a lane
    static constexpr int VW = DV * K::BYTES / 4;    // 32-bit words of a value row in a lane
    struct Step {
        u32x4 k[U][KL];
        uint32_t v[U][4][VW];
    };
    // What a wave leaves in LDS of an item at its end, in the place of q's
    // terms: [WV][HD] outputs with rows ROW apart, so that 16 rows' 16-byte
    // writes fall on different banks, [WV] maxima, [WV] sums.
    static constexpr int ROW = HD + 4, kWave = WV * (ROW + 2);
    static constexpr int kQ = KL * (K::TERMS - 1) * 64;         // of a wave, in 16-byte units
    static constexpr int kShared = std::max(4 * kWave, 4 * 4 * kQ);  // 32-bit words
};

template <int W>
__device__ __forceinline__ void load_words(uint32_t (&d)[W], const char* p) {
    if constexpr (W == 1) d[0] = *as_global(reinterpret_cast<const uint32_t*>(p));
    else if constexpr (W == 2) {
        const vvli_u32x2 x = *as_global(reinterpret_cast<const vvli_u32x2*>(p));
        d[0] = x.x, d[1] = x.y;
    } else {
#pragma unroll
        for (int i = 0; i < W; i += 4) {
            const vvli_u32x4 x = *as_global(reinterpret_cast<const vvli_u32x4*>(p + 4 * i));
            d[i] = x.x, d[i + 1] = x.y, d[i + 2] = x.z, d[i + 3] = x.w;
        }
    }
}

template <int KIND>
__device__ __forceinline__ uint32_t word_finite(uint32_t w) {  // values that are not finite become 0
    if constexpr (KIND == VVLI_CACHE_F32) return (w & 0x7f800000u) == 0x7f800000u ? 0u : w;
    constexpr uint32_t e = KIND == VVLI_CACHE_BF16 ? 0x7f80u : 0x7c00u;
    const uint32_t lo = (w & e) == e ? 0u : w & 0xffffu, hi = (w & (e << 16)) == (e << 16) ? 0u : w & 0xffff0000u;
    return lo | hi;
}
template <int KIND>
__device__ __forceinline__ float value_at(const uint32_t* words, int i) {
    if constexpr (KIND == VVLI_CACHE_F32) return __uint_as_float(words[i]);
    const uint16_t h = reinterpret_cast<const uint16_t*>(words)[i];
    if constexpr (KIND == VVLI_CACHE_BF16) return __uint_as_float(static_cast<uint32_t>(h) << 16);
    else return static_cast<float>(__builtin_bit_cast(_Float16, h));
}

// A value that is not finite spoils its dimension of every vector of an item,
// also of those that do not see its key (0 times it is NaN) and, through split
// terms of either sign, an infinity of those that do. That shows in the
// outputs, so no step looks for it: where outputs are not finite, the keys are
// gone over once more with such values taken as 0, and then they go straight
// to the outputs of the vectors that see them, whose sums they are whatever
// their weights. add(at, row) takes key `at` of a step of WK whose values
// hold one; `slots` as in filled().
template <int HD, int KIND, int WK, typename Add>
__device__ __forceinline__ void odd_values(const char* vbase, uint64_t row_bytes, uint32_t slots, uint64_t none, Add&& add) {
    constexpr int CHUNKS = HD * Kind<KIND>::BYTES / 16;
    static_assert(WK * CHUNKS % 64 == 0, "whole waves");
    bool odd = false;
    for (uint32_t i = threadIdx.x & 63; i < WK * CHUNKS; i += 64) {
        uint32_t w[4];
        load_words<4>(w, vbase + static_cast<uint32_t>(__shfl(slots, i / CHUNKS, 64)) * row_bytes + i % CHUNKS * 16);
#pragma unroll
        for (int e = 0; e < 4; ++e) odd |= word_finite<KIND>(w[e]) != w[e];
    }
    if (!__any(odd)) return;
    for (int at = 0; at < WK; ++at)
        if (!(none >> at & 1)) add(at, reinterpret_cast<const uint32_t*>(vbase + static_cast<uint32_t>(__shfl(slots, at, 64)) * row_bytes));
}

template <int HD, int KIND>
__global__ __launch_bounds__(kThreads, HD == 128 ? 2 : 3) void paged_attn_kernel(PagedAttnArgs a) {
    using F = Form<HD, KIND>;
    using K = Kind<KIND>;
    constexpr int WV = F::WV, U = F::U, WK = F::WK, DV = F::DV, KL = F::KL, VW = F::VW, ROW = F::ROW;
    constexpr bool F32 = KIND == VVLI_CACHE_F32;
    __shared__ RunScratch sc;
    __shared__ __attribute__((aligned(16))) float shared[F::kShared];

    const Run from = find_run<typename F::S>(a, sc);
    if (!from.any) return;
    const int tid = threadIdx.x, lane = tid & 63, fr = lane & 15, fq = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint64_t row_bytes = a.slot_stride * K::BYTES;
    const uint32_t slot_words = a.slot_vecs * (HD + 2);
    for (Walk<typename F::S> walk(a, from); walk.item(a); walk.next()) {
        const Run& run = walk.run;
        const Request& req = walk.req;
        const Units& un = walk.un;
        const uint32_t t0 = walk.part.t0;
        const uint32_t sets = 4u >> un.wide, UK = WK * sets;      // sets of waves with all of the item's vectors
        const uint32_t qw = wave & ((1u << un.wide) - 1), ks = wave >> un.wide;
        u32x4* const q_mine = reinterpret_cast<u32x4*>(shared) + qw * F::kQ + lane;  // (the sets write the same values)
        const int32_t* table = a.table + static_cast<size_t>(run.r) * a.stride;
        const char* kbase = static_cast<const char*>(a.k) + static_cast<size_t>(run.kvh) * HD * K::BYTES + 16 * fq;
        const char* vbase = static_cast<const char*>(a.v) + static_cast<size_t>(run.kvh) * HD * K::BYTES + 4 * VW * fr;

        // The first step's keys and values are on their way before q is taken apart.
        const uint32_t wm0 = run.m0 + qw * WV;  // the wave's first vector
        // Keys w_lo .. w_hi - 1 are seen by some vector of the wave, all_lo .. all_hi - 1 by
        // every one of them (no test needed there).
        uint32_t w_lo = 0, w_hi = 0, all_lo = 0, all_hi = 0;
        if (wm0 < req.vecs) {
            const int64_t p0 = req.start + page_of(a.group, wm0), p1 = req.start + page_of(a.group, min(wm0 + WV, req.vecs) - 1);
            const KeySpan s0 = key_span(p0, a.window, a.room), s1 = key_span(p1, a.window, a.room);
            w_lo = max(un.lo, a.window && p0 + 1 > a.window ? static_cast<uint32_t>(min(p0 + 1 - a.window, static_cast<int64_t>(a.room))) : 0);
            w_hi = p1 < 0 ? 0 : static_cast<uint32_t>(min(p1 + 1, static_cast<int64_t>(a.room)));
            all_lo = s1.lo, all_hi = min(s0.hi, s1.hi);
        }
        // The wave's steps: those units of the run whose WK keys from t * UK + ks * WK on meet w_lo .. w_hi - 1.
        uint32_t ta = walk.first_unit(), tb = walk.end_unit();
        if (w_lo >= (ks + 1) * WK) ta = max(ta, (w_lo - (ks + 1) * WK) / UK + 1);
        tb = w_lo < w_hi && w_hi > ks * WK ? min(tb, (w_hi - ks * WK + UK - 1) / UK) : 0;

        f32x4 o[DV];
        float m_run, l_run;

        // Slot of key t * UK + ks * WK + lane (of WK lanes), -1 where no vector of the wave sees it.
        auto slot_of = [&](uint32_t t) -> int32_t {
            const uint32_t key = t * UK + ks * WK + (lane & (WK - 1));
            return t < tb && key >= w_lo && key < w_hi ? page_slot(table, a.stride, a.pages, a.ps, key) : -1;
        };
        // Slots that there are none of read another key of the step, whose score is then not used: they
        // need neither a test at every load nor memory of their own.
        auto filled = [&](int32_t slot, uint64_t& none) -> uint32_t {
            none = __ballot(slot < 0);
            const int32_t other = ~none ? __builtin_amdgcn_readlane(slot, __builtin_ctzll(~none)) : 0;
            return slot < 0 ? other : slot;
        };
        typename F::Step st;
        auto load_k = [&](uint32_t slots) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const uint32_t s = __shfl(slots, 16 * u + fr, 64);
                const char* p = kbase + s * row_bytes;
#pragma unroll
                for (int i = 0; i < KL; ++i) {
                    uint32_t w[4];
                    load_words<4>(w, p + 64 * i);
                    st.k[u][i] = u32x4{w[0], w[1], w[2], w[3]};
                }
            }
        };
        auto load_v = [&](uint32_t slots) {
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t s = __shfl(slots, 16 * u + 4 * fq + j, 64);
                    load_words<VW>(st.v[u][j], vbase + s * row_bytes);
                }
        };
        uint64_t none;
        uint32_t slots = filled(slot_of(ta), none);
        int32_t ahead = slot_of(ta + 1);
        if (ta < tb) load_k(slots), load_v(slots);

        // The lane's vector: its keys and q.
        float inv = 1.f;  // scores are this times the products (f16's power of two)
        u32x4 qf[KL];
        const uint32_t m = wm0 + fr;
        const bool there = m < req.vecs;
        const uint32_t row = page_of(a.group, there ? m : 0), g = (there ? m : 0) - row * a.group.d;
        const KeySpan see = there ? key_span(req.start + row, a.window, a.room) : KeySpan{0, 0};
        const float* qp = a.q + (req.first + row) * a.ldq + (static_cast<size_t>(run.kvh) * a.group.d + g) * HD;
        const float f = a.scale * 1.44269504088896341f;
        if constexpr (F32) {
#pragma unroll
            for (int s = 0; s < KL; ++s) {
                const float4 x = load_f32x4(qp + 16 * s + 4 * fq);
                qf[s] = __builtin_bit_cast(u32x4, f32x4{x.x * f, x.y * f, x.z * f, x.w * f});
            }
        } else {
            float x[KL][8];
            float top = 0.f;
#pragma unroll
            for (int s = 0; s < KL; ++s) {
                const float4 x0 = load_f32x4(qp + 32 * s + 8 * fq), x1 = load_f32x4(qp + 32 * s + 8 * fq + 4);
                x[s][0] = x0.x, x[s][1] = x0.y, x[s][2] = x0.z, x[s][3] = x0.w;
                x[s][4] = x1.x, x[s][5] = x1.y, x[s][6] = x1.z, x[s][7] = x1.w;
#pragma unroll
                for (int e = 0; e < 8; ++e) x[s][e] *= f, top = fmaxf(top, fabsf(x[s][e]));
            }
            if constexpr (KIND == VVLI_CACHE_F16) {
                const int ex = f16_exponent(rows_max(top));
                const float up = ldexpf(1.f, ex);
                inv = ldexpf(1.f, -ex);
#pragma unroll
                for (int s = 0; s < KL; ++s)
#pragma unroll
                    for (int e = 0; e < 8; ++e) x[s][e] *= up;
            }
#pragma unroll
            for (int s = 0; s < KL; ++s) {
                typename K::T8 t[K::TERMS];
#pragma unroll
                for (int e = 0; e < 8; e += 2) split2<K>(x[s][e], x[s][e + 1], e, t);
                qf[s] = __builtin_bit_cast(u32x4, t[0]);
#pragma unroll
                for (int i = 1; i < K::TERMS; ++i) q_mine[(s * (K::TERMS - 1) + i - 1) * 64] = __builtin_bit_cast(u32x4, t[i]);
            }
        }
        bool spoilt = false;
        for (int careful = 0; careful < 2; ++careful) {
            m_run = -INFINITY, l_run = 0.f;
#pragma unroll
            for (int e = 0; e < DV; ++e) o[e] = f32x4{0, 0, 0, 0};
            if (ta >= tb) break;
            uint64_t none_next;
            uint32_t slots_next;
            if (careful) {
                slots = filled(slot_of(ta), none), ahead = slot_of(ta + 1);
                load_k(slots);
                load_v(slots);
            }
            for (uint32_t t = ta; t < tb; ++t) {
                slots_next = filled(ahead, none_next);
                ahead = slot_of(t + 2);
                const uint32_t key0 = t * UK + ks * WK;
                if (careful) {
#pragma unroll
                    for (int u = 0; u < U; ++u)
#pragma unroll
                        for (int j = 0; j < 4; ++j)
#pragma unroll
                            for (int i = 0; i < VW; ++i) st.v[u][j][i] = word_finite<KIND>(st.v[u][j][i]);
                }
                f32x4 s[U];
#pragma unroll
                for (int u = 0; u < U; ++u) s[u] = f32x4{0, 0, 0, 0};
#pragma unroll
                for (int i = 0; i < KL; ++i) {
                    if constexpr (F32) {
#pragma unroll
                        for (int e = 0; e < 4; ++e)
#pragma unroll
                            for (int u = 0; u < U; ++u)
                                s[u] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(st.k[u][i][e]), __uint_as_float(qf[i][e]),
                                                                            s[u], 0, 0, 0);
                    } else {
#pragma unroll
                        for (int x = 0; x < K::TERMS; ++x) {
                            const u32x4 qx = x == 0 ? qf[i] : q_mine[(i * (K::TERMS - 1) + x - 1) * 64];
#pragma unroll
                            for (int u = 0; u < U; ++u)
                                s[u] = K::mfma(__builtin_bit_cast(typename K::T8, st.k[u][i]),
                                               __builtin_bit_cast(typename K::T8, qx), s[u]);
                        }
                    }
                }
                if (t + 1 < tb) load_k(slots_next);
                // Holes in the table and the ends of spans need the test.
                if (key0 < all_lo || key0 + WK > all_hi || none) {
#pragma unroll
                    for (int u = 0; u < U; ++u)
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const uint32_t at = 16 * u + 4 * fq + j, key = key0 + at;
                            const bool hole = none >> at & 1;
                            if (hole || key < see.lo || key >= see.hi) s[u][j] = -INFINITY;
                        }
                }
                u32x4 pf[F32 ? U : K::TERMS];
                float mx = -INFINITY;
#pragma unroll
                for (int u = 0; u < U; ++u)
#pragma unroll
                    for (int j = 0; j < 4; ++j) mx = fmaxf(mx, s[u][j]);
                const float m_new = fmaxf(m_run, rows_max(mx) * inv);
                const float m_sub = m_new == -INFINITY ? 0.f : m_new;
                const bool grew = m_new != m_run;
                const float corr = __builtin_amdgcn_exp2f(m_run - m_sub), shift = shift_of<K>(K::TOP, m_sub);
                float sum = 0.f;
#pragma unroll
                for (int u = 0; u < U; ++u)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float p = __builtin_amdgcn_exp2f(fmaf(s[u][j], inv, shift));
                        s[u][j] = p;
                        sum += p;
                    }
                if constexpr (F32) {
#pragma unroll
                    for (int u = 0; u < U; ++u) pf[u] = __builtin_bit_cast(u32x4, s[u]);
                } else {
                    typename K::T8 t8[K::TERMS];
#pragma unroll
                    for (int u = 0; u < U; ++u)
#pragma unroll
                        for (int j = 0; j < 4; j += 2) split2<K>(s[u][j], s[u][j + 1], 4 * u + j, t8);
#pragma unroll
                    for (int x = 0; x < K::TERMS; ++x) pf[x] = __builtin_bit_cast(u32x4, t8[x]);
                }
                l_run = l_run * corr + sum;
                m_run = m_new;
                if (__any(grew)) {
#pragma unroll
                    for (int e = 0; e < DV; ++e) o[e] *= corr;
                }
#pragma unroll
                for (int e = 0; e < DV; ++e) {
                    if constexpr (F32) {
#pragma unroll
                        for (int u = 0; u < U; ++u)
#pragma unroll
                            for (int j = 0; j < 4; ++j)
                                o[e] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(st.v[u][j][e]), __uint_as_float(pf[u][j]),
                                                                            o[e], 0, 0, 0);
                    } else {
                        u32x4 w;
#pragma unroll
                        for (int u = 0; u < U; ++u)
#pragma unroll
                            for (int jp = 0; jp < 2; ++jp)  // keys 2 jp and 2 jp + 1, dim e of the lane's
                                w[2 * u + jp] = __builtin_amdgcn_perm(st.v[u][2 * jp + 1][e / 2], st.v[u][2 * jp][e / 2],
                                                                      e % 2 ? 0x07060302u : 0x05040100u);
#pragma unroll
                        for (int x = 0; x < K::TERMS; ++x)
                            o[e] = K::mfma(__builtin_bit_cast(typename K::T8, w), __builtin_bit_cast(typename K::T8, pf[x]), o[e]);
                    }
                }
                if (t + 1 < tb) load_v(slots_next);
                slots = slots_next, none = none_next;
            }
            mfma_done(o);
            float sum = 0.f;  // NaN if one of them is not finite
#pragma unroll
            for (int e = 0; e < DV; ++e)
#pragma unroll
                for (int j = 0; j < 4; ++j) sum = fmaf(o[e][j], 0.f, sum);
            if (careful) {
                spoilt = true;
            } else if (!__any(sum != sum)) {  // see odd_values
                break;
            }
        }
        if (spoilt)
            for (uint32_t t = ta; t < tb; ++t) {
                uint64_t none;
                const uint32_t slots = filled(slot_of(t), none);
                odd_values<HD, KIND, WK>(vbase - 4 * VW * fr, row_bytes, slots, none, [&](int at, const uint32_t* p) {
                    const uint32_t key = t * UK + ks * WK + at;
                    const bool sees = key >= see.lo && key < see.hi;
#pragma unroll
                    for (int e = 0; e < DV; ++e)
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const float x = value_at<KIND>(p, DV * (4 * fq + j) + e);
                            if (sees && !(fabsf(x) < INFINITY)) o[e][j] += x;
                        }
                });
            }

        // The waves' parts: outputs [WV][HD], maxima, sums.
        __syncthreads();  // (q's terms are read)
        float* mine = shared + wave * F::kWave;
        float l = l_run;
        l += __shfl_xor(l, 16, 64);
        l += __shfl_xor(l, 32, 64);
        if (fq == 0) mine[WV * ROW + fr] = m_run, mine[WV * ROW + WV + fr] = l;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float* p = mine + fr * ROW + DV * (4 * fq + j);
            if constexpr (DV >= 4) {
#pragma unroll
                for (int e = 0; e < DV; e += 4)
                    *reinterpret_cast<f32x4*>(p + e) = f32x4{o[e][j], o[e + 1][j], o[e + 2][j], o[e + 3][j]};
            } else {
                p[0] = o[0][j], p[1] = o[1][j];
            }
        }
        __syncthreads();
        const bool whole = walk.whole();
        const uint32_t vecs = walk.vecs();
        auto write = [&](uint32_t v, uint32_t d, f32x4 x, float l) {
            const uint32_t m = run.m0 + v, row = page_of(a.group, m), g = m - row * a.group.d;
            float* op = a.out + (req.first + row) * a.ldo + (static_cast<size_t>(run.kvh) * a.group.d + g) * HD + d;
            const float r = 1.f / l;
            *reinterpret_cast<f32x4*>(op) = l == 0.f ? f32x4{0, 0, 0, 0} : x * r;
        };
        float* slot = a.parts + (2 * static_cast<size_t>(run.index) + (t0 == 0)) * slot_words;
        for (uint32_t i = tid; i < vecs * (HD / 4); i += kThreads) {
            const uint32_t v = i / (HD / 4), d = i % (HD / 4) * 4, vq = v / WV, vv = v % WV;
            float top = -INFINITY;
            for (uint32_t w = vq; w < 4; w += 4 / sets) top = fmaxf(top, shared[w * F::kWave + WV * ROW + vv]);
            const float base = top == -INFINITY ? 0.f : top;
            float l = 0.f;
            f32x4 x = {0, 0, 0, 0};
            for (uint32_t w = vq; w < 4; w += 4 / sets) {
                const float* p = shared + w * F::kWave;
                const float c = __builtin_amdgcn_exp2f(p[WV * ROW + vv] - base);
                l += p[WV * ROW + WV + vv] * c;
                x += *reinterpret_cast<const f32x4*>(p + vv * ROW + d) * c;
            }
            if (whole) {
                write(v, d, x, l);
            } else {
                publish(slot + v * HD + d, x[0], x[1]);
                publish(slot + v * HD + d + 2, x[2], x[3]);
                if (d == 0) publish(slot + a.slot_vecs * HD + 2 * v, top, l);
            }
        }
        if (!whole) {
            const uint32_t n = walk.parts();
            const uint64_t border = walk.border();
            if (last_part(a.arrived + border - 1, n, sc.last)) {
                const float* first = a.parts + (2 * border - 1) * slot_words;
                auto part_at = [&](uint32_t i) { return i == 0 ? first : first + (2 * static_cast<size_t>(i) - 1) * slot_words; };
                // Two 16-byte pieces of the outputs a thread, four parts of each in flight.
                constexpr uint32_t NP = 4, NI = 2;
                for (uint32_t i0 = tid; i0 < vecs * (HD / 4); i0 += NI * kThreads) {
                    float top[NI], l[NI];
                    f32x4 x[NI];
                    uint32_t at[NI], at_ml[NI];
#pragma unroll
                    for (uint32_t k = 0; k < NI; ++k) {
                        const uint32_t i = min(i0 + k * kThreads, vecs * (HD / 4) - 1);
                        at[k] = 4 * i, at_ml[k] = static_cast<uint32_t>(a.slot_vecs) * HD + 2 * (i / (HD / 4));
                        top[k] = -INFINITY, l[k] = 0.f, x[k] = f32x4{0, 0, 0, 0};
                    }
                    for (uint32_t w0 = 0; w0 < n; w0 += NP) {
                        float2 ml[NI][NP], u0[NI][NP], u1[NI][NP];
#pragma unroll
                        for (uint32_t w = 0; w < NP; ++w) {
                            const float* p = part_at(min(w0 + w, n - 1));
#pragma unroll
                            for (uint32_t k = 0; k < NI; ++k)
                                ml[k][w] = fetch(p + at_ml[k]), u0[k][w] = fetch(p + at[k]), u1[k][w] = fetch(p + at[k] + 2);
                        }
#pragma unroll
                        for (uint32_t k = 0; k < NI; ++k) {
                            float more = top[k];
#pragma unroll
                            for (uint32_t w = 0; w < NP; ++w) more = fmaxf(more, ml[k][w].x);
                            const float base = more == -INFINITY ? 0.f : more, old = __builtin_amdgcn_exp2f(top[k] - base);
                            top[k] = more, l[k] *= old, x[k] *= old;
#pragma unroll
                            for (uint32_t w = 0; w < NP; ++w) {
                                const float c = w0 + w < n ? __builtin_amdgcn_exp2f(ml[k][w].x - base) : 0.f;
                                if (w0 + w < n) l[k] += ml[k][w].y * c, x[k] += f32x4{u0[k][w].x, u0[k][w].y, u1[k][w].x, u1[k][w].y} * c;
                            }
                        }
                    }
#pragma unroll
                    for (uint32_t k = 0; k < NI; ++k) {
                        const uint32_t i = i0 + k * kThreads;
                        if (i < vecs * (HD / 4)) write(i / (HD / 4), i % (HD / 4) * 4, x[k], l[k]);
                    }
                }
            }
            if (walk.part.cut) return;
        }
        __syncthreads();
    }
}

// ---------------------------------------------------------------------------
// Chunks: items of 128 vectors, 32 to a wave, and steps of 32 keys that the
// block's waves share through LDS (a wave's own loads of every key would be
// 16 KiB a step and wave in 16 bits). The block loads the next step's keys and
// values into registers while it computes this one, and stores them into the
// other of two stages behind it: one barrier a step. Products are 32 x 32 x 16
// (16-bit caches) or 32 x 32 x 2 (f32), a lane l with vector l % 32:
//   S^T = K Q^T    A: key l % 32, dims 16 s + 8 (l / 32) .. + 7, or
//                  8 s + 4 (l / 32) + e; D: register r has key
//                  8 (r / 4) + 4 (l / 32) + r % 4
//   O^T += V^T P^T B: registers 8 c .. 8 c + 7 of the weights are step c's 8
//                  values of k (f32: register r is step r's), as they stand;
//                  A: dim 32 n + l % 32, the same keys, in 16 bits 4 at a time
//                  by a transposed read of LDS (ds_read_b64_tr_b16); D: dims
//                  32 n + 8 (r / 4) + 4 (l / 32) + r % 4
// Rows lie in LDS as in memory, their 16-byte chunks permuted by the row so that
// the rows of a fragment read fall on different banks (no conflict is counted).
//
// Products bound it: 4000 rows behind 8000, 28 heads over 4 of 128, 4.6 ms in f32
// (125 of the 133 TFLOP/s that a large product reaches), 1.19 ms in f16 (480, times
// two terms 960 of 1310: a step's vector instructions, among them some 30 that
// bring spilled values back, weigh more beside fewer products) and 1.47 ms in
// bf16 (390, times three terms 1170 of 1200). Short chunks are bound by the runs'
// ends: 2 x up to 2000 rows behind up to 2100 in bf16 265 to 275 us (335 to 347,
// 1000 to 1040 with terms).
// ---------------------------------------------------------------------------
template <int HD, int KIND>
struct Wide {
    using K = Kind<KIND>;
    static constexpr bool F32 = KIND == VVLI_CACHE_F32;
    static constexpr int WV = 32, M = 128, WK = 32, NT = HD / 32, DS = HD * K::BYTES / 32;
    using S = ChunkCuts<F32>;
    static_assert(S::M == M && S::WK == WK);
    static constexpr int RB = HD * K::BYTES, CH = RB / 16, RPL = RB < 256 ? 256 / RB : 1;  // bytes and 16-byte chunks of a row, rows of 256 bytes
    static constexpr int TILE = WK * RB, LOADS = 2 * TILE / (16 * kThreads), ROWS = LOADS > 1 ? LOADS / 2 : 1;
    static constexpr int QR = F32 ? 1 : 2;  // terms of q in registers; the rest in LDS
    // A vector's weights are 2^(s + BIAS - base) with a base that follows the maximum of its scores only where that is
    // more than SLACK above it: weights stay in range, and few steps have outputs to rescale.
    static constexpr float SLACK = K::TOP > 0.f ? 4.f : 8.f, BIAS = K::TOP > 0.f ? K::TOP - SLACK : 0.f;
    static constexpr int kQ = (K::TERMS - QR) * 4 * DS * 1024;
    static __device__ __forceinline__ uint32_t kswz(uint32_t r) { return r / RPL % (CH < 16 ? CH : 16); }
    static __device__ __forceinline__ uint32_t vswz(uint32_t r) { return F32 ? (CH >= 16 ? r / 4 % 2 * 8 : 0) : 4 * (r / RPL % (CH / 4)); }
};
typedef short s16x4 __attribute__((ext_vector_type(4)));

template <int HD, int KIND>
__global__ __launch_bounds__(kThreads, 2) void paged_wide_kernel(PagedAttnArgs a) {
    using F = Wide<HD, KIND>;
    using K = Kind<KIND>;
    constexpr int WV = F::WV, M = F::M, WK = F::WK, NT = F::NT, DS = F::DS, CH = F::CH, RB = F::RB, TILE = F::TILE;
    constexpr int LOADS = F::LOADS, ROWS = F::ROWS, QR = F::QR;
    constexpr bool F32 = F::F32;
    __shared__ RunScratch sc;
    __shared__ __attribute__((aligned(1024))) char stage[2][2 * TILE];  // keys, then values
    __shared__ __attribute__((aligned(16))) char q_rest[F::kQ ? F::kQ : 16];

    const Run from = find_run<typename F::S>(a, sc);
    if (!from.any) return;
    const int tid = threadIdx.x, lane = tid & 63, fr = lane & 31, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint64_t row_bytes = a.slot_stride * K::BYTES;
    const uint32_t slot_words = a.slot_vecs * (HD + 2);
    u32x4* const q_mine = reinterpret_cast<u32x4*>(q_rest) + wave * ((K::TERMS - QR) * DS * 64) + lane;
    // Where the lane's fragments lie in a stage (products' step s and tile n are put in by ^ and +).
    const uint32_t k_at = fr * RB + ((half ^ F::kswz(fr)) << 4);
    const uint32_t v_row = 4 * half + (F32 ? 0 : (lane & 15) / 4);
    const uint32_t v_chunk = F32 ? fr / 4 : 2 * (lane / 16 % 2) + lane / 2 % 2;
    const uint32_t v_at = TILE + v_row * RB + ((v_chunk ^ F::vswz(v_row)) << 4) + (F32 ? 4 * (fr & 3) : 8 * (lane & 1));
    // This thread's rows of a step (the same of keys and of values; HD = 32: of one of the two) and its chunk.
    const uint32_t my_row = tid % (WK * CH / ROWS) / CH, my_c = tid % CH;

    for (Walk<typename F::S> walk(a, from); walk.item(a); walk.next()) {
        const Run& run = walk.run;
        const Request& req = walk.req;
        const Units& un = walk.un;
        const int32_t* table = a.table + static_cast<size_t>(run.r) * a.stride;
        const char* kbase = static_cast<const char*>(a.k) + static_cast<size_t>(run.kvh) * RB;
        const char* vbase = static_cast<const char*>(a.v) + static_cast<size_t>(run.kvh) * RB;

        // The lane's vector: its keys and q.
        const uint32_t wm0 = run.m0 + wave * WV, m = wm0 + fr;
        const bool there = m < req.vecs;
        const uint32_t row = page_of(a.group, there ? m : 0);
        const KeySpan see = there ? key_span(req.start + row, a.window, a.room) : KeySpan{0, 0};
        const size_t head = (static_cast<size_t>(run.kvh) * a.group.d + (there ? m : 0) - row * a.group.d) * HD;
        float inv = 1.f;
        u32x4 qf[QR][DS];
        if constexpr (F32) {
            const float* qp = a.q + (req.first + row) * a.ldq + head + 4 * half;
            const float f = a.scale * 1.44269504088896341f;
#pragma unroll
            for (int s = 0; s < DS; ++s) {
                const float4 x = load_f32x4(qp + 8 * s);
                qf[0][s] = __builtin_bit_cast(u32x4, f32x4{x.x * f, x.y * f, x.z * f, x.w * f});
            }
        } else {
            const float* qp = a.q + (req.first + row) * a.ldq + head + 8 * half;
            const float f = a.scale * 1.44269504088896341f;
            float x[DS][8];
            float top = 0.f;
#pragma unroll
            for (int s = 0; s < DS; ++s) {
                const float4 x0 = load_f32x4(qp + 16 * s), x1 = load_f32x4(qp + 16 * s + 4);
                x[s][0] = x0.x, x[s][1] = x0.y, x[s][2] = x0.z, x[s][3] = x0.w;
                x[s][4] = x1.x, x[s][5] = x1.y, x[s][6] = x1.z, x[s][7] = x1.w;
#pragma unroll
                for (int e = 0; e < 8; ++e) x[s][e] *= f, top = fmaxf(top, fabsf(x[s][e]));
            }
            if constexpr (KIND == VVLI_CACHE_F16) {
                const int ex = f16_exponent(fmaxf(top, __shfl_xor(top, 32, 64)));
                const float up = ldexpf(1.f, ex);
                inv = ldexpf(1.f, -ex);
#pragma unroll
                for (int s = 0; s < DS; ++s)
#pragma unroll
                    for (int e = 0; e < 8; ++e) x[s][e] *= up;
            }
#pragma unroll
            for (int s = 0; s < DS; ++s) {
                typename K::T8 t[K::TERMS];
#pragma unroll
                for (int e = 0; e < 8; e += 2) split2<K>(x[s][e], x[s][e + 1], e, t);
#pragma unroll
                for (int i = 0; i < K::TERMS; ++i) {
                    if (i < QR) qf[i < QR ? i : 0][s] = __builtin_bit_cast(u32x4, t[i]);
                    else q_mine[((i - QR) * DS + s) * 64] = __builtin_bit_cast(u32x4, t[i]);
                }
            }
        }
        // Keys w_lo .. w_hi - 1 are seen by some vector of the wave, all_lo .. all_hi - 1 by every one of them.
        uint32_t w_lo = 0, w_hi = 0, all_lo = 0, all_hi = 0;
        if (wm0 < req.vecs) {
            const int64_t p0 = req.start + page_of(a.group, wm0), p1 = req.start + page_of(a.group, min(wm0 + WV, req.vecs) - 1);
            const KeySpan s0 = key_span(p0, a.window, a.room), s1 = key_span(p1, a.window, a.room);
            w_lo = a.window && p0 + 1 > a.window ? static_cast<uint32_t>(min(p0 + 1 - a.window, static_cast<int64_t>(a.room))) : 0;
            w_hi = p1 < 0 ? 0 : static_cast<uint32_t>(min(p1 + 1, static_cast<int64_t>(a.room)));
            all_lo = s1.lo, all_hi = min(s0.hi, s1.hi);
        }
        const uint32_t ta = walk.first_unit(), tb = un.hi ? walk.end_unit() : 0;

        f32x16 o[NT];
        float m_run, l_run, shift;  // base of the weights (-inf: none yet), their sum, what is added to scores
        auto slot_of = [&](uint32_t t) -> int32_t {
            const uint32_t key = t * WK + fr;
            return t < tb && key >= un.lo && key < un.hi ? page_slot(table, a.stride, a.pages, a.ps, key) : -1;
        };
        auto filled = [&](int32_t slot, uint32_t& none) -> uint32_t {
            const uint64_t n = __ballot(slot < 0);
            none = static_cast<uint32_t>(n);
            const int32_t other = ~n ? __builtin_amdgcn_readlane(slot, __builtin_ctzll(~n)) : 0;
            return slot < 0 ? other : slot;
        };
        u32x4 next[LOADS];
        auto load = [&](uint32_t slots) {
#pragma unroll
            for (int r = 0; r < ROWS; ++r) {
                const uint64_t at = static_cast<uint32_t>(__shfl(slots, my_row + WK / ROWS * r, 64)) * row_bytes + 16 * my_c;
#pragma unroll
                for (int v = 0; v < LOADS / ROWS; ++v) {
                    uint32_t w[4];
                    load_words<4>(w, (LOADS == 1 ? (tid >= WK * CH ? vbase : kbase) : v ? vbase : kbase) + at);
                    next[ROWS * v + r] = u32x4{w[0], w[1], w[2], w[3]};
                }
            }
        };
        auto store = [&](uint32_t st, bool careful) {
#pragma unroll
            for (int r = 0; r < ROWS; ++r)
#pragma unroll
                for (int v = 0; v < LOADS / ROWS; ++v) {
                    const uint32_t rw = my_row + WK / ROWS * r;
                    const bool val = LOADS == 1 ? tid >= WK * CH : v;
                    u32x4& x = next[ROWS * v + r];
                    if (careful && val) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) x[e] = word_finite<KIND>(x[e]);
                    }
                    *reinterpret_cast<u32x4*>(stage[st] + (val ? TILE : 0) + rw * RB + ((my_c ^ (val ? F::vswz(rw) : F::kswz(rw))) << 4)) = x;
                }
        };
        bool spoilt = false;
        for (int careful = 0; careful < 2; ++careful) {
            m_run = -INFINITY, l_run = 0.f, shift = F::BIAS;
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int r = 0; r < 16; ++r) o[n][r] = 0.f;
            if (ta >= tb) break;
            uint32_t none, none_next;
            uint32_t slots = filled(slot_of(ta), none);
            int32_t ahead = slot_of(ta + 1);
            load(slots);
            store(0, careful);
            __syncthreads();
            uint32_t st = 0;
            for (uint32_t t = ta; t < tb; ++t, st ^= 1) {
                const uint32_t slots_next = filled(ahead, none_next);
                if (t + 1 < tb) load(slots_next);
                ahead = slot_of(t + 2);
                const uint32_t key0 = t * WK;
                if (key0 < w_hi && key0 + WK > w_lo) {
                    const char* base = stage[st];
                    // Two sums, of even and odd steps, and below the tiles of O^T in turn: a product waits for the
                    // one before it on the same sum about as long as it takes.
                    f32x16 sums[2];
#pragma unroll
                    for (int r = 0; r < 16; ++r) sums[0][r] = sums[1][r] = 0.f;
#pragma unroll
                    for (int i = 0; i < DS; i += 2) {
                        const u32x4 k0 = *reinterpret_cast<const u32x4*>(base + (k_at ^ (32 * i)));
                        const u32x4 k1 = *reinterpret_cast<const u32x4*>(base + (k_at ^ (32 * i + 32)));
                        if constexpr (F32) {
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                sums[0] = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(k0[e]), __uint_as_float(qf[0][i][e]), sums[0], 0, 0, 0);
                                sums[1] = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(k1[e]), __uint_as_float(qf[0][i + 1][e]), sums[1], 0, 0, 0);
                            }
                        } else {
#pragma unroll
                            for (int x = 0; x < K::TERMS; ++x) {
                                u32x4 q0, q1;
                                if (x < QR) q0 = qf[x < QR ? x : 0][i], q1 = qf[x < QR ? x : 0][i + 1];
                                else q0 = q_mine[((x - QR) * DS + i) * 64], q1 = q_mine[((x - QR) * DS + i + 1) * 64];
                                sums[0] = K::mfma(__builtin_bit_cast(typename K::T8, k0), __builtin_bit_cast(typename K::T8, q0), sums[0]);
                                sums[1] = K::mfma(__builtin_bit_cast(typename K::T8, k1), __builtin_bit_cast(typename K::T8, q1), sums[1]);
                            }
                        }
                    }
                    mfma_done(sums);
                    f32x16 s = sums[0] + sums[1];
                    if (key0 < all_lo || key0 + WK > all_hi || none) {
#pragma unroll
                        for (int r = 0; r < 16; ++r) {
                            const uint32_t at = 8 * (r / 4) + 4 * half + r % 4, key = key0 + at;
                            if ((none >> at & 1) || key < see.lo || key >= see.hi) s[r] = -INFINITY;
                        }
                    }
                    float mx = fmaxf(s[0], s[1]);
#pragma unroll
                    for (int r = 2; r < 16; ++r) mx = fmaxf(mx, s[r]);
                    const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(mx), __float_as_uint(mx), false, false);
                    mx = fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1])) * inv;
                    const bool grew = mx - m_run > F::SLACK;
                    if (__any(grew)) {
                        const float m_new = grew ? mx : m_run, m_sub = m_new == -INFINITY ? 0.f : m_new;
                        const float corr = __builtin_amdgcn_exp2f(m_run - m_sub);
                        m_run = m_new, shift = shift_of<K>(F::BIAS, m_sub), l_run *= corr;
#pragma unroll
                        for (int n = 0; n < NT; ++n) o[n] *= corr;
                    }
                    float sum[2] = {0.f, 0.f};
                    if constexpr (F32) {
#pragma unroll
                        for (int r = 0; r < 16; ++r) s[r] = __builtin_amdgcn_exp2f(s[r] + shift), sum[r & 1] += s[r];
#pragma unroll
                        for (int r = 0; r < 16; ++r)
#pragma unroll
                            for (int n = 0; n < NT; ++n) {
                                const float x = *reinterpret_cast<const float*>(base + ((v_at ^ (128 * n)) + (8 * (r / 4) + r % 4) * RB));
                                o[n] = __builtin_amdgcn_mfma_f32_32x32x2f32(x, s[r], o[n], 0, 0, 0);
                            }
                    } else {
                        typename K::T8 pf[2][K::TERMS];
#pragma unroll
                        for (int c = 0; c < 2; ++c)
#pragma unroll
                            for (int e = 0; e < 8; e += 2) {
                                const float p0 = __builtin_amdgcn_exp2f(fmaf(s[8 * c + e], inv, shift));
                                const float p1 = __builtin_amdgcn_exp2f(fmaf(s[8 * c + e + 1], inv, shift));
                                sum[0] += p0, sum[1] += p1;
                                split2<K>(p0, p1, e, pf[c]);
                            }
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            u32x4 w[NT];
#pragma unroll
                            for (int n = 0; n < NT; ++n)
#pragma unroll
                                for (int h = 0; h < 2; ++h) {
                                    const s16x4 v = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                        (__attribute__((address_space(3))) s16x4*)(base + ((v_at ^ (64 * n)) + (16 * c + 8 * h) * RB)));
                                    const uint2 d = __builtin_bit_cast(uint2, v);
                                    w[n][2 * h] = d.x, w[n][2 * h + 1] = d.y;
                                }
#pragma unroll
                            for (int x = 0; x < K::TERMS; ++x)
#pragma unroll
                                for (int n = 0; n < NT; ++n) o[n] = K::mfma(__builtin_bit_cast(typename K::T8, w[n]), pf[c][x], o[n]);
                        }
                    }
                    l_run += sum[0] + sum[1];
                }
                if (t + 1 < tb) store(st ^ 1, careful);
                none = none_next;
                __syncthreads();
            }
            mfma_done(o);
            float sum = 0.f;  // NaN if one of them is not finite
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int r = 0; r < 16; ++r) sum = fmaf(o[n][r], 0.f, sum);
            if (careful) {
                spoilt = true;
            } else if (!__syncthreads_or(sum != sum)) {  // see odd_values
                break;
            }
        }
        if (spoilt)
            for (uint32_t t = max(ta, w_lo / WK); t < min(tb, (w_hi + WK - 1) / WK); ++t) {
                uint32_t none;
                const uint32_t slots = filled(slot_of(t), none);
                odd_values<HD, KIND, WK>(vbase, row_bytes, slots, none, [&](int at, const uint32_t* p) {
                    const bool sees = t * WK + at >= see.lo && t * WK + at < see.hi;
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int r = 0; r < 16; ++r) {
                            const float x = value_at<KIND>(p, 32 * n + 8 * (r / 4) + 4 * half + r % 4);
                            if (sees && !(fabsf(x) < INFINITY)) o[n][r] += x;
                        }
                });
            }

        l_run += __shfl_xor(l_run, 32, 64);
        // Registers 4 i .. 4 i + 3 of tile n are dims 32 n + 8 i + 4 half .. + 3.
        auto write = [&]() {
            if (!there) return;
            float* op = a.out + (req.first + row) * a.ldo + head + 4 * half;
            const float r = 1.f / l_run;
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    *reinterpret_cast<f32x4*>(op + 32 * n + 8 * i) =
                        l_run == 0.f ? f32x4{0, 0, 0, 0}
                                      : f32x4{o[n][4 * i] * r, o[n][4 * i + 1] * r, o[n][4 * i + 2] * r, o[n][4 * i + 3] * r};
        };
        if (walk.whole()) {
            write();
            continue;
        }
        // A part is an image of the threads' registers, 8 bytes of each thread side by side; then maxima and sums.
        constexpr int IMAGE = NT * 16 * kThreads;
        static_assert(IMAGE == M * HD, "a part has its slot");
        float* slot = a.parts + (2 * static_cast<size_t>(run.index) + (walk.part.t0 == 0)) * slot_words;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int r = 0; r < 16; r += 2) publish(slot + (16 * n + r) * kThreads + 2 * tid, o[n][r], o[n][r + 1]);
        if (half == 0) publish(slot + IMAGE + 2 * (wave * WV + fr), m_run, l_run);
        const uint32_t parts = walk.parts();
        const uint64_t border = walk.border();
        if (last_part(a.arrived + border - 1, parts, sc.last)) {
            const float* first = a.parts + (2 * border - 1) * slot_words;
            m_run = -INFINITY, l_run = 0.f;
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int r = 0; r < 16; ++r) o[n][r] = 0.f;
            for (uint32_t w = 0; w < parts; ++w) {
                const float* p = w == 0 ? first : first + (2 * static_cast<size_t>(w) - 1) * slot_words;
                const float2 ml = fetch(p + IMAGE + 2 * (wave * WV + fr));
                float2 x[NT][8];
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int r = 0; r < 16; r += 2) x[n][r / 2] = fetch(p + (16 * n + r) * kThreads + 2 * tid);
                const float m_new = fmaxf(m_run, ml.x), base = m_new == -INFINITY ? 0.f : m_new;
                const float c0 = __builtin_amdgcn_exp2f(m_run - base), c1 = __builtin_amdgcn_exp2f(ml.x - base);
                m_run = m_new, l_run = l_run * c0 + ml.y * c1;
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int r = 0; r < 16; ++r) o[n][r] = o[n][r] * c0 + (r % 2 ? x[n][r / 2].y : x[n][r / 2].x) * c1;
            }
            write();
        }
        if (walk.part.cut) return;
    }
}

// What a call runs: an item's vectors, blocks, the kernel.
struct Plan {
    uint32_t m, blocks;
    bool wide;
};

// Chunks (many vectors of an average request and kv head), or not: a chunk's block takes 128 vectors a key read, but
// shares steps of 32 keys behind a barrier each, and in a batch of prompts and single tokens most of its vectors are
// none. Eight requests with up to so many rows behind up to 2000 positions, not as chunks | as chunks, bf16 (f32):
//   28 heads over 4 of 128   20 rows  51 | 59 us (70 | 91)   100 rows  63 | 63 us (109 | 113)   200 rows  105 | 84 us (228 | 200)
//   32 heads over 8 of 64    10 rows  26 | 30 us (43 | 45)    15 rows  29 | 29 us  (44 | 45)     80 rows   49 | 36 us  (77 | 70)
// and 63 single tokens with one prompt of 500 rows, heads of 128: 99 | 144 us.
// Blocks: as many as the registers of their waves leave room for, two or three on a CU (three and not two, 32 heads over 8
// of 64: 24 x 5 rows behind up to 4100 in f32 49 and not 52 us, 300 x 1 row behind up to 1000 in bf16 95 and not 103, 64 x 1
// behind 8000 195 and not 198, but 361 and not 352 in f32).
Plan plan_of(uint32_t rows, uint32_t requests, uint32_t group, uint32_t hd) {
    const bool wide = static_cast<uint64_t>(rows) * group > uint64_t{hd == 128 ? 384u : 48u} * requests;
    return Plan{wide ? 128u : 64u, gemm_cus() * (wide || hd == 128 ? 2 : 3), wide};
}

// Vectors that a part has room for (chunks' parts are images of all of an item's), and the bytes of a call's
// workspace: counters, then two parts for each block.
uint32_t slot_vecs(const Plan& p, uint32_t rows, uint32_t group) {
    return p.wide ? p.m : static_cast<uint32_t>(std::min<uint64_t>(p.m, (static_cast<uint64_t>(rows) * group + 1) & ~uint64_t{1}));
}
size_t plan_bytes(const Plan& p, uint32_t vecs, uint32_t hd) {
    return p.blocks * sizeof(float) * (4 + 2 * static_cast<size_t>(vecs) * (hd + 2));
}

bool sizes_ok(uint32_t rows, uint32_t requests, uint32_t heads, uint32_t kv_heads) {
    return requests != 0 && heads != 0 && kv_heads != 0 && heads % kv_heads == 0 && heads <= 65535 &&
           static_cast<uint64_t>(rows) * heads < kPagedMost;
}

template <int HD, int KIND>
hipError_t launch(const PagedAttnArgs& a, const Plan& p, hipStream_t s) {
    const dim3 grid(p.blocks), block(kThreads);
    return p.wide ? vlaunch(paged_wide_kernel<HD, KIND>, grid, block, 0, s, a)
                  : vlaunch(paged_attn_kernel<HD, KIND>, grid, block, 0, s, a);
}

template <int HD>
hipError_t launch(const PagedAttnArgs& a, uint32_t kind, const Plan& p, hipStream_t s) {
    return kind == VVLI_CACHE_F32 ? launch<HD, VVLI_CACHE_F32>(a, p, s)
           : kind == VVLI_CACHE_BF16 ? launch<HD, VVLI_CACHE_BF16>(a, p, s)
                                     : launch<HD, VVLI_CACHE_F16>(a, p, s);
}

}  // namespace

extern "C" {

size_t vvli_gpu_paged_attention_workspace(uint32_t rows, uint32_t requests, uint32_t heads, uint32_t kv_heads,
                                          uint32_t head_dim) {
    if (!sizes_ok(rows, requests, heads, kv_heads) || (head_dim != 32 && head_dim != 64 && head_dim != 128)) return 0;
    // Of however few requests, and of no fewer than any.
    const uint32_t group = heads / kv_heads;
    size_t most = 0;
    for (uint32_t n : {1u, ~0u}) {
        const Plan p = plan_of(rows, n, group, head_dim);
        most = std::max(most, plan_bytes(p, slot_vecs(p, rows, group), head_dim));
    }
    return most;
}

int vvli_gpu_paged_attention(const vvli_gpu_paged_cache* cache, const int32_t* table, uint32_t table_stride,
                             const int32_t* row_start, const int32_t* start_pos, uint32_t requests, const float* q,
                             uint64_t ldq, float* out, uint64_t ldo, uint32_t rows, uint32_t heads, float scale,
                             uint32_t window, void* workspace, size_t workspace_bytes, void* stream) {
    const char* who = "vvli_gpu_paged_attention";
    int rc = check_cache(cache, who);
    if (rc) return rc;
    if (!table || !row_start || !start_pos || !workspace) return set_error(VVLI_NULL_ARG, "NULL argument to %s", who);
    if (!sizes_ok(rows, requests, heads, cache->kv_heads) || table_stride == 0 ||
        static_cast<uint64_t>(table_stride) * cache->page_size >= kPagedMost ||
        static_cast<uint64_t>(table_stride) * requests >= kPagedMost || !std::isfinite(scale))
        return set_error(VVLI_INVALID_CONFIG, "%s: bad sizes (%u rows of %u requests, %u heads of %u, table rows of %u)", who,
                         rows, requests, heads, cache->kv_heads, table_stride);
    const uint64_t width = static_cast<uint64_t>(heads) * cache->head_dim;
    if ((rc = check_rows(q, ldq, width, "q", who)) || (rc = check_rows(out, ldo, width, "out", who))) return rc;
    if (!aligned16(workspace) ||
        workspace_bytes < vvli_gpu_paged_attention_workspace(rows, requests, heads, cache->kv_heads, cache->head_dim))
        return set_error(VVLI_INVALID_CONFIG, "%s: workspace of %zu bytes", who, workspace_bytes);
    if (q == out) return set_error(VVLI_INVALID_CONFIG, "%s: out is q", who);
    if (rows == 0) return VVLI_OK;
    const uint32_t group = heads / cache->kv_heads;
    const Plan p = plan_of(rows, requests, group, cache->head_dim);
    PagedAttnArgs a{};
    a.k = cache->k, a.v = cache->v, a.table = table, a.row_start = row_start, a.start_pos = start_pos, a.q = q, a.out = out;
    a.arrived = static_cast<uint32_t*>(workspace);
    a.parts = static_cast<float*>(workspace) + 4 * p.blocks;
    a.slot_vecs = slot_vecs(p, rows, group);
    a.slot_stride = cache->slot_stride, a.ldq = ldq, a.ldo = ldo;
    a.stride = table_stride, a.requests = requests, a.rows = rows, a.kv_heads = cache->kv_heads, a.window = window;
    a.pages = cache->pages, a.room = table_stride * cache->page_size, a.ps = page_div(cache->page_size), a.group = page_div(group);
    a.scale = scale;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    PAGED_TRY(cache->head_dim == 128 ? launch<128>(a, cache->kind, p, s)
              : cache->head_dim == 64 ? launch<64>(a, cache->kind, p, s)
                                      : launch<32>(a, cache->kind, p, s));
    return VVLI_OK;
}

}  // extern "C"
