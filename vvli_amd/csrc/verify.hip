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

#include "paged.hpp"

using namespace vvli;

namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;
// Slices of a row: at most kSliceMost tokens for each block, fewer where the
// requests alone leave most of the GPU idle (kBlocks blocks in all), not under
// kSliceLeast. 64 rows of 128256: 16 slices each; one row of 151936: 149.
constexpr uint32_t kSliceMost = 8192, kSliceLeast = 1024, kBlocks = 1024, kSlicesMost = 256;

struct VerifyArgs {
    const float *target, *draft, *u_accept, *u_sample;
    const int32_t *tokens, *row_start;
    int32_t *accepted, *out;
    uint32_t* arrived;  // of each request: slices whose sums are there; 0 between calls
    double* sums;       // [request][slice]: of what the draft left, of the target row
    uint64_t ldt, ldd;
    uint32_t rows, vocab, slices, slice;
};

__device__ inline double weight_of(double w) { return w > 0 && w < INFINITY ? w : 0; }

// The value of thread 0..; inclusive over the block's threads in their order, and the sum of all.
__device__ inline double block_scan(double v, double* waves, double& total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const double u = __shfl_up(v, o, 64);
        if (lane >= o) v += u;
    }
    __syncthreads();
    if (lane == 63) waves[wave] = v;
    __syncthreads();
    double before = 0;
    total = 0;
    for (int w = 0; w < kWaves; ++w) {
        if (w == wave) before = total;
        total += waves[w];
    }
    return before + v;
}
// Lowest thread for which `yes`, kThreads if none.
__device__ inline uint32_t first_thread(bool yes, uint32_t* waves) {
    const uint64_t b = __ballot(yes);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = b ? __builtin_ctzll(b) : 64;
    __syncthreads();
    for (uint32_t w = 0; w < kWaves; ++w)
        if (waves[w] < 64) return w * 64 + waves[w];
    return kThreads;
}
__device__ inline uint32_t last_thread(bool yes, uint32_t* waves) {
    const uint64_t b = __ballot(yes);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = b ? 63 - __builtin_clzll(b) : 64;
    __syncthreads();
    for (int w = kWaves - 1; w >= 0; --w)
        if (waves[w] < 64) return w * 64 + waves[w];
    return kThreads;
}

// Block (slice, request). Every block finds where the request's drafts end (a
// few gathered values, less than a launch of its own would cost) and sums its
// slice of that row, of both weights at once; the block whose sums are the
// request's last finds the token's slice and the token in it, which is what a
// second pass over one slice costs. One pass over one row of target and draft
// for each request bounds it.
__global__ __launch_bounds__(kThreads) void verify_kernel(VerifyArgs a) {
    __shared__ double waves[kWaves];
    __shared__ uint32_t found[kWaves], stop, last;
    __shared__ double slice_before;
    const uint32_t r = blockIdx.y, sl = blockIdx.x, tid = threadIdx.x;
    const RowSpan span = row_span(a.row_start[r], a.row_start[r + 1], a.rows);
    if (span.count == 0) {
        if (tid == 0 && sl == 0) a.accepted[r] = 0;
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
            const double q = a.draft ? a.draft[row * a.ldd + x] : 1.0;
            ok = static_cast<double>(a.u_accept[row]) * q < static_cast<double>(a.target[row * a.ldt + x]);
        }
        if (!ok) atomicMin(&stop, i);
    }
    __syncthreads();
    const uint32_t acc = stop;
    const uint64_t row = span.first + acc;
    const float* p = a.target + row * a.ldt;
    const float* q = a.draft && acc < drafts ? a.draft + row * a.ldd : nullptr;
    const uint32_t x = acc < drafts ? a.tokens[row + 1] : a.vocab;
    // What the draft leaves of token v; the target row itself where all drafts were accepted.
    auto left = [&](uint32_t v, float pv, float qv) {
        return weight_of(q ? static_cast<double>(pv) - static_cast<double>(qv) : v == x ? 0.0 : static_cast<double>(pv));
    };
    double s0 = 0, s1 = 0;
    {
        const uint32_t from = sl * a.slice, to = min(from + a.slice, a.vocab);
        constexpr int N = 4;  // loads in flight
        uint32_t v = from + tid;
        for (; v + (N - 1) * kThreads < to; v += N * kThreads) {
            float pv[N], qv[N];
#pragma unroll
            for (int i = 0; i < N; ++i) pv[i] = p[v + i * kThreads], qv[i] = q ? q[v + i * kThreads] : 0.f;
#pragma unroll
            for (int i = 0; i < N; ++i) s0 += left(v + i * kThreads, pv[i], qv[i]), s1 += weight_of(pv[i]);
        }
        for (; v < to; v += kThreads) {
            const float pv = p[v], qv = q ? q[v] : 0.f;
            s0 += left(v, pv, qv), s1 += weight_of(pv);
        }
    }
    double t0, t1;
    block_scan(s0, waves, t0);
    block_scan(s1, waves, t1);
    if (a.slices > 1) {
        if (tid == 0) {
            uint64_t* out = reinterpret_cast<uint64_t*>(a.sums + 2 * (static_cast<size_t>(r) * a.slices + sl));
            __hip_atomic_store(out, __builtin_bit_cast(uint64_t, t0), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            __hip_atomic_store(out + 1, __builtin_bit_cast(uint64_t, t1), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            __builtin_amdgcn_s_waitcnt(0);  // both are in memory (agent-scope stores go through)
            last = __hip_atomic_fetch_add(a.arrived + r, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == a.slices - 1;
            if (last) __hip_atomic_store(a.arrived + r, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);  // for the next call
        }
        __syncthreads();
        if (!last) return;
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");
        s0 = s1 = 0;
        if (tid < a.slices) {
            const uint64_t* in = reinterpret_cast<const uint64_t*>(a.sums + 2 * (static_cast<size_t>(r) * a.slices + tid));
            s0 = __builtin_bit_cast(double, __hip_atomic_load(in, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
            s1 = __builtin_bit_cast(double, __hip_atomic_load(in + 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
        }
    } else {
        s0 = tid ? 0 : t0, s1 = tid ? 0 : t1;
    }
    // Thread s has slice s. The lowest token whose running sum is not at or below the border; behind the last one
    // (a number of 1 or more) the last token with a weight.
    const double e0 = block_scan(s0, waves, t0), e1 = block_scan(s1, waves, t1);
    const bool less = acc < drafts && t0 > 0;
    const double total = less ? t0 : t1, mine = less ? s0 : s1, end = less ? e0 : e1;
    int32_t token = -1;
    if (total > 0) {
        const double border = static_cast<double>(a.u_sample[r]) * total;
        uint32_t at = first_thread(tid < a.slices && !(end <= border), found);
        const bool behind = at == kThreads;
        if (behind) at = last_thread(mine > 0, found);
        if (tid == at) slice_before = end - mine;
        __syncthreads();
        const double before = slice_before;
        // Thread t has the slice's run t of tokens.
        const uint32_t from = at * a.slice, to = min(from + a.slice, a.vocab), per = (to - from + kThreads - 1) / kThreads;
        const uint32_t a0 = min(from + tid * per, to), a1 = min(a0 + per, to);
        auto weight = [&](uint32_t v) { return less ? left(v, p[v], q ? q[v] : 0.f) : weight_of(p[v]); };
        double run = 0;
        for (uint32_t v = a0; v < a1; ++v) run += weight(v);
        double sum;
        const double upto = before + block_scan(run, waves, sum);
        uint32_t who = behind ? kThreads : first_thread(a0 < a1 && !(upto <= border), found);
        const bool over = who == kThreads;  // behind the last token, also where the slice's sum was rounded up to it
        if (over) who = last_thread(run > 0, found);
        if (tid == who) {
            double sofar = upto - run;
            uint32_t best = a0;
            for (uint32_t v = a0; v < a1; ++v) {
                const double w = weight(v);
                if (w > 0) best = v;
                sofar += w;
                if (!over && !(sofar <= border)) {
                    best = v;
                    break;
                }
            }
            last = best;
        }
        __syncthreads();
        if (who < kThreads) token = static_cast<int32_t>(last);
    }
    if (tid == 0) a.accepted[r] = static_cast<int32_t>(acc);
    for (uint32_t i = tid; i < span.count; i += kThreads) a.out[span.first + i] = i < acc ? a.tokens[span.first + i + 1] : i == acc ? token : -1;
}

struct Slices {
    uint32_t count, tokens;
};
Slices slices_of(uint32_t requests, uint32_t vocab) {
    const uint32_t few = (vocab - 1) / kSliceMost + 1, many = std::min((vocab - 1) / kSliceLeast + 1, (kBlocks - 1) / requests + 1);
    const uint32_t n = std::min(std::max(few, many), kSlicesMost), tokens = (vocab - 1) / n + 1;
    return Slices{(vocab - 1) / tokens + 1, tokens};
}

size_t counter_bytes(uint32_t requests) { return (static_cast<size_t>(requests) * 4 + 15) / 16 * 16; }

}  // namespace

extern "C" {

size_t vvli_gpu_verify_drafts_workspace(uint32_t requests, uint32_t vocab) {
    // (slices of fewer requests: no more than kBlocks and one each)
    const size_t few = vocab ? (vocab - 1) / kSliceMost + 1 : 0;
    return counter_bytes(requests) + 16 * (requests * std::min<size_t>(few, kSlicesMost) + requests + kBlocks);
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
    if (out == tokens) return set_error(VVLI_INVALID_CONFIG, "%s: out is tokens", who);
    if (!aligned16(workspace) || workspace_bytes < vvli_gpu_verify_drafts_workspace(requests, vocab))
        return set_error(VVLI_INVALID_CONFIG, "%s: workspace of %zu bytes", who, workspace_bytes);
    const Slices sl = slices_of(requests, vocab);
    VerifyArgs a{};
    a.target = target, a.draft = draft, a.u_accept = u_accept, a.u_sample = u_sample, a.tokens = tokens, a.row_start = row_start;
    a.accepted = accepted, a.out = out, a.arrived = static_cast<uint32_t*>(workspace);
    a.sums = reinterpret_cast<double*>(static_cast<char*>(workspace) + counter_bytes(requests));
    a.ldt = ldt, a.ldd = ldd, a.rows = rows, a.vocab = vocab, a.slices = sl.count, a.slice = sl.tokens;
    PAGED_TRY(vlaunch(verify_kernel, dim3(sl.count, requests), dim3(kThreads), 0, static_cast<hipStream_t>(stream), a));
    return VVLI_OK;
}

}  // extern "C"
