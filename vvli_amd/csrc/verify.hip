// verify.hip -- drafted tokens against the target's probabilities
// (vvli_gpu_verify_drafts).
//
// With p the target's and q the draft's row behind a token, draft x stays
// while u q(x) < p(x); where one is refused the next token follows
// max(p - q, 0), which makes every given token one of p's. The token is the
// lowest v with sum(w[0..v]) > u sum(w). Sums are f64: an f32 sum over a
// vocabulary is off by more than a token's weight, so that tokens near a
// border would follow the order of adding.
#include <algorithm>

#include "device_common.hpp"
#include "paged.hpp"

using namespace vvli;

namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;
// A row is cut into chunks of whole kStep tokens (8 a lane of a wave), at most
// one for each thread of the block that searches their sums; a block sums some
// of them: enough blocks for the GPU, each with a chunk for every wave if there
// are as many. (256 requests of 32000 tokens: 28 us with 512 blocks, 54 with
// 2048; 64 of 128256 the same with either, 1 of 151936 too.)
constexpr uint32_t kStep = 512, kChunksMost = kThreads, kBlocks = 512;
// 8-byte words of a request in the workspace, the same for every vocabulary and
// number of requests: a workspace serves calls of other sizes too, and where a
// counter is for one of them no sum may be for another.
constexpr uint32_t kRecord = 1 + kChunksMost;

struct VerifyArgs {
    const float *target, *draft, *u_accept, *u_sample;
    const int32_t *tokens, *row_start;
    int32_t *accepted, *out;
    uint64_t* space;  // of each request kRecord words: blocks whose sums are there (0 between calls), then the chunks' sums
    uint64_t ldt, ldd;
    uint32_t rows, vocab, chunks, chunk, per_block;  // chunk: in tokens
};

// The weights of a row: what the draft leaves of the target's, or the target's.
struct Weights {
    const float *p, *q;  // (q null: none)
    uint32_t vocab, without;
    bool aligned;
};

__device__ __forceinline__ void load8(const Weights& w, uint32_t v, float (&p)[8], float (&q)[8]) {
    if (w.aligned && v + 8 <= w.vocab) {
#pragma unroll
        for (int i = 0; i < 8; i += 4) {
            const float4 x = load_f32x4(w.p + v + i), y = w.q ? load_f32x4(w.q + v + i) : make_float4(0, 0, 0, 0);
            p[i] = x.x, p[i + 1] = x.y, p[i + 2] = x.z, p[i + 3] = x.w;
            q[i] = y.x, q[i + 1] = y.y, q[i + 2] = y.z, q[i + 3] = y.w;
        }
        return;
    }
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) {
        const bool in = v < w.vocab && i < w.vocab - v;
        p[i] = in ? w.p[v + i] : 0.f, q[i] = in && w.q ? w.q[v + i] : 0.f;
    }
}
// A negative value of the draft counts 0, one that is not finite leaves nothing of the target's.
__device__ __forceinline__ float draft_value(float q) { return fabsf(q) < INFINITY ? fmaxf(q, 0.f) : INFINITY; }
__device__ __forceinline__ double weight(const Weights& w, uint32_t v, float p, float q) {
    // (finite and positive: also of a difference, which is f64 since f32 would round it)
    const double d = v == w.without ? 0.0 : static_cast<double>(p) - static_cast<double>(q);
    return d > 0 && d < INFINITY ? d : 0.0;
}
__device__ __forceinline__ double weight8(const Weights& w, uint32_t v, const float (&p)[8], float (&q)[8], double (&x)[8]) {
    uint32_t signs = 0;  // (values without a sign are right as they are: weight() leaves out what is not finite)
#pragma unroll
    for (int i = 0; i < 8; ++i) signs |= __float_as_uint(q[i]);
    if (__builtin_expect(__any(signs >> 31), 0)) {
#pragma unroll
        for (int i = 0; i < 8; ++i) q[i] = draft_value(q[i]);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = weight(w, v + i, p[i], q[i]);
    return ((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7]));
}

__device__ __forceinline__ double wave_total(double v) {
#pragma unroll
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}
__device__ __forceinline__ double wave_scan(double v) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const double u = __shfl_up(v, o, 64);
        if (lane >= o) v += u;
    }
    return v;
}

// A wave's sum of tokens from .. from + chunk - 1, two steps' loads in flight where a chunk has two (vocabularies over
// kStep * kChunksMost = 131072).
__device__ __forceinline__ double chunk_sum(const Weights& w, uint32_t from, uint32_t chunk) {
    const uint32_t lane = threadIdx.x & 63;
    double s = 0, x[8];
    for (uint32_t t = 0; t < chunk; t += 2 * kStep) {
        const uint32_t v0 = from + t + 8 * lane, v1 = v0 + kStep;
        const bool more = t + kStep < chunk;
        float p0[8], q0[8], p1[8], q1[8];
        load8(w, v0, p0, q0);
        if (more) load8(w, v1, p1, q1);
        s += weight8(w, v0, p0, q0, x);
        if (more) s += weight8(w, v1, p1, q1, x);
    }
    return wave_total(s);
}

// Block (some chunks, request). Every block finds where the request's drafts
// end (a few gathered values, less than a launch of its own would cost) and
// sums its chunks of that row; the block whose sums are the request's last
// finds the token's chunk among the sums and, with one wave, the token in it.
// One pass over one row of target and draft for each request bounds it where
// there are many requests (64 with 4 drafts, 128256 tokens: 21 us, 2.4 TB/s),
// the chain of dependent loads where there are few (1, 151936 tokens: 7.5 us).
// By blocks that walk the row in strides of the grid, each search over the
// whole row again, the two took 55 and 9.8 us.
__global__ __launch_bounds__(kThreads) void verify_kernel(VerifyArgs a) {
    __shared__ double sums[kChunksMost], waves[kWaves];
    __shared__ uint32_t found[kWaves], stop, last;
    const uint32_t r = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const RowSpan span = row_span(a.row_start[r], a.row_start[r + 1], a.rows);
    if (span.count == 0) {
        if (tid == 0 && blockIdx.x == 0) a.accepted[r] = 0;
        return;
    }
    const uint32_t drafts = span.count - 1;
    if (tid == 0) stop = drafts;
    __syncthreads();
    for (uint32_t i = tid; i < drafts; i += kThreads) {
        const uint64_t row = span.first + i;
        const uint32_t x = a.tokens[row + 1];
        bool ok = false;
        if (x < a.vocab) {
            const float p = a.target[row * a.ldt + x], q = a.draft ? draft_value(a.draft[row * a.ldd + x]) : 1.f;
            ok = p > 0 && p < INFINITY && q < INFINITY && static_cast<double>(a.u_accept[row]) * q < p;
        }
        if (!ok) atomicMin(&stop, i);
    }
    __syncthreads();
    const uint32_t acc = stop;
    const bool refused = acc < drafts;
    const uint64_t row = span.first + acc;
    Weights w;
    w.p = a.target + row * a.ldt, w.q = refused && a.draft ? a.draft + row * a.ldd : nullptr;
    w.vocab = a.vocab, w.without = refused && !a.draft ? a.tokens[row + 1] : ~0u;
    w.aligned = (reinterpret_cast<uintptr_t>(w.p) | reinterpret_cast<uintptr_t>(w.q)) % 16 == 0;
    const uint32_t c0 = blockIdx.x * a.per_block, c1 = min(c0 + a.per_block, a.chunks);
    uint64_t* const mine = a.space + static_cast<size_t>(r) * kRecord + 1;
    uint32_t* const arrived = reinterpret_cast<uint32_t*>(mine - 1);
    for (uint32_t c = c0 + wave; c < c1; c += kWaves) {
        const double s = chunk_sum(w, c * a.chunk, a.chunk);
        if (lane == 0) __hip_atomic_store(mine + c, __builtin_bit_cast(uint64_t, s), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __builtin_amdgcn_s_waitcnt(0);  // the sums are in memory (agent-scope stores go through)
    __syncthreads();
    if (tid == 0) {
        last = __hip_atomic_fetch_add(arrived, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == gridDim.x - 1;
        if (last) __hip_atomic_store(arrived, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);  // for the next call
    }
    __syncthreads();
    if (!last) return;
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");
    double s = 0;
    if (tid < a.chunks) s = __builtin_bit_cast(double, __hip_atomic_load(mine + tid, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
    double total, end;
    for (bool again = refused;; again = false) {
        // Sums up to each chunk, thread c having chunk c.
        end = wave_scan(s);
        __syncthreads();
        if (lane == 63) waves[wave] = end;
        __syncthreads();
        total = 0;
        for (uint32_t k = 0; k < kWaves; ++k) {
            if (k == wave) end += total;
            total += waves[k];
        }
        if (total > 0 || !again) break;
        // Nothing is left of the target's row: the row itself.
        w.q = nullptr, w.without = ~0u, w.aligned = reinterpret_cast<uintptr_t>(w.p) % 16 == 0;
        for (uint32_t c = wave; c < a.chunks; c += kWaves) {
            const double x = chunk_sum(w, c * a.chunk, a.chunk);
            if (lane == 0) sums[c] = x;
        }
        __syncthreads();
        s = tid < a.chunks ? sums[tid] : 0;
    }
    // The lowest token whose running sum is over the border; for numbers of 1 and more, and where no sum is, the last
    // token with a weight. Sums of different orders of adding are an ulp apart, so that a sum may be over the border
    // where no weight was added to it: only chunks, lanes and tokens that have a weight are taken. (A border below 0
    // is under all sums, that of token 0 too.)
    int32_t token = -1;
    if (total > 0) {
        const double u = a.u_sample[r], border = u * total;
        const uint64_t some = __ballot(s > 0), yes = __ballot(s > 0 && end > border);
        if (lane == 0) found[wave] = yes ? __builtin_ctzll(yes) : 64;
        sums[tid] = end - s;
        if (tid == 0) last = 0;
        __syncthreads();
        uint32_t at = kThreads;
        for (int k = kWaves - 1; k >= 0; --k)
            if (found[k] < 64) at = k * 64 + found[k];
        const bool behind = at == kThreads || u >= 1;
        if (behind) {
            if (lane == 0 && some) atomicMax(&last, wave * 64 + 63 - __builtin_clzll(some));
            __syncthreads();
            at = last;
        }
        if (!(u >= 0)) {
            token = 0;
        } else if (wave == 0) {
            double before = sums[at];
            uint32_t best = 0;  // 1 + the last token with a weight in the lane
            bool done = false;
            for (uint32_t t = 0; t < a.chunk && !done; t += kStep) {
                const uint32_t v = at * a.chunk + t + 8 * lane;
                float p[8], q[8];
                double x[8];
                load8(w, v, p, q);
                const double sum = weight8(w, v, p, q, x), upto = before + wave_scan(sum);
                const uint64_t over = behind ? 0 : __ballot(sum > 0 && upto > border);
                if (over) {
                    double run = upto - sum;
                    uint32_t tok = 0;
                    bool there = false;
#pragma unroll
                    for (uint32_t i = 0; i < 8; ++i) {
                        run += x[i];
                        if (x[i] > 0 && !there) tok = v + i, there = run > border;
                    }
                    best = __shfl(tok, __builtin_ctzll(over), 64) + 1;
                    done = true;
                } else {
#pragma unroll
                    for (uint32_t i = 0; i < 8; ++i)
                        if (x[i] > 0) best = v + i + 1;
                    before = __shfl(upto, 63, 64);
                }
            }
            // (not found: behind the last token, also where the chunk's sum was rounded up to it)
#pragma unroll
            for (int o = 32; o; o >>= 1) best = max(best, static_cast<uint32_t>(__shfl_xor(best, o, 64)));
            token = static_cast<int32_t>(best) - 1;
        }
    }
    if (tid == 0) {
        a.accepted[r] = static_cast<int32_t>(acc);
        a.out[span.first + acc] = token;
    }
    for (uint32_t i = tid; i < span.count; i += kThreads)
        if (i != acc) a.out[span.first + i] = i < acc ? a.tokens[span.first + i + 1] : -1;
}

uint32_t chunk_tokens(uint32_t vocab) { return ((vocab - 1) / (kStep * kChunksMost) + 1) * kStep; }
uint32_t chunks_of(uint32_t vocab) { return (vocab - 1) / chunk_tokens(vocab) + 1; }

}  // namespace

extern "C" {

size_t vvli_gpu_verify_drafts_workspace(uint32_t requests, uint32_t vocab) {
    return vocab ? static_cast<size_t>(requests) * kRecord * 8 : 0;
}

int vvli_gpu_verify_drafts(const float* target, uint64_t ldt, const float* draft, uint64_t ldd, const int32_t* tokens,
                           const int32_t* row_start, uint32_t requests, uint32_t rows, uint32_t vocab,
                           const float* u_accept, const float* u_sample, int32_t* accepted, int32_t* out,
                           void* workspace, size_t workspace_bytes, void* stream) {
    const char* who = "vvli_gpu_verify_drafts";
    if (!target || !tokens || !row_start || !u_accept || !u_sample || !accepted || !out || !workspace)
        return set_error(VVLI_NULL_ARG, "NULL argument to %s", who);
    if (requests == 0 || vocab == 0 || rows >= kPagedMost || requests > 65535 || vocab >= kPagedMost || ldt < vocab ||
        ldt >= kPagedMost || (draft && (ldd < vocab || ldd >= kPagedMost)))
        return set_error(VVLI_INVALID_CONFIG, "%s: bad sizes (%u requests, %u rows of %u)", who, requests, rows, vocab);
    // (Blocks read tokens while others write out.)
    const uintptr_t from = reinterpret_cast<uintptr_t>(tokens), to = reinterpret_cast<uintptr_t>(out), size = rows * sizeof(int32_t);
    if (to == from || (to < from + size && from < to + size)) return set_error(VVLI_INVALID_CONFIG, "%s: out overlaps tokens", who);
    if (!aligned16(workspace) || workspace_bytes < vvli_gpu_verify_drafts_workspace(requests, vocab))
        return set_error(VVLI_INVALID_CONFIG, "%s: workspace of %zu bytes", who, workspace_bytes);
    VerifyArgs a{};
    a.target = target, a.draft = draft, a.u_accept = u_accept, a.u_sample = u_sample, a.tokens = tokens, a.row_start = row_start;
    a.accepted = accepted, a.out = out, a.space = static_cast<uint64_t*>(workspace);
    a.ldt = ldt, a.ldd = ldd, a.rows = rows, a.vocab = vocab;
    a.chunks = chunks_of(vocab), a.chunk = chunk_tokens(vocab);
    const uint32_t blocks = std::min((a.chunks - 1) / kWaves + 1, (kBlocks - 1) / requests + 1);
    a.per_block = (a.chunks - 1) / blocks + 1;
    const dim3 grid((a.chunks - 1) / a.per_block + 1, requests);
    PAGED_TRY(vlaunch(verify_kernel, grid, dim3(kThreads), 0, static_cast<hipStream_t>(stream), a));
    return VVLI_OK;
}

}  // extern "C"
