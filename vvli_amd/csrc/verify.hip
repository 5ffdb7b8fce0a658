// verify.hip -- drafted tokens against the target's probabilities
// (vvli_gpu_verify_drafts).
//
// With p the target's and q the draft's row behind a token, draft x stays
// while u q(x) < p(x); where one is refused the next token follows
// max(p - q, 0), which makes every given token one of p's. The token is the
// lowest v with sum(w[0..v]) > u sum(w). Sums are f64: an f32 sum over a
// vocabulary is off by more than a token's weight, so that tokens near a
// border would follow the order of adding.
#include "paged.hpp"

using namespace vvli;

namespace {

struct VerifyArgs {
    const float *target, *draft, *u_accept, *u_sample;
    const int32_t *tokens, *row_start;
    int32_t *accepted, *out;
    uint64_t ldt, ldd;
    uint32_t rows, vocab;
};

constexpr int kThreads = 256;

__device__ inline double weight_of(double w) { return w > 0 && w < INFINITY ? w : 0; }

// One block per request, the row in pieces of 256 tokens.
__global__ __launch_bounds__(kThreads) void verify_kernel(VerifyArgs a) {
    __shared__ uint32_t stop;
    __shared__ double sums[kThreads];
    const uint32_t r = blockIdx.x, tid = threadIdx.x;
    const RowSpan span = row_span(a.row_start[r], a.row_start[r + 1], a.rows);
    if (span.count == 0) {
        if (tid == 0) a.accepted[r] = 0;
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
    const float* q = a.draft ? a.draft + row * a.ldd : nullptr;
    const uint32_t x = acc < drafts ? a.tokens[row + 1] : a.vocab;
    auto weight = [&](uint32_t v, bool less) {
        const double w = p[v];
        return weight_of(!less ? w : q ? w - static_cast<double>(q[v]) : v == x ? 0.0 : w);
    };
    int32_t token = -1;
    for (int less = acc < drafts ? 1 : 0; less >= 0; --less) {
        // Thread t sums tokens t * per ..; then the thread whose run holds the border looks for it.
        const uint32_t per = (a.vocab + kThreads - 1) / kThreads, from = min(tid * per, a.vocab), to = min(from + per, a.vocab);
        double mine = 0;
        for (uint32_t v = from; v < to; ++v) mine += weight(v, less);
        __syncthreads();
        sums[tid] = mine;
        __syncthreads();
        if (tid == 0) {
            double total = 0;
            for (int t = 0; t < kThreads; ++t) total += sums[t];
            if (total > 0) {
                const double border = static_cast<double>(a.u_sample[r]) * total;
                int t = 0, last = -1;
                double before = 0;
                for (; t < kThreads; ++t) {
                    if (sums[t] > 0) last = t;
                    if (!(before + sums[t] <= border)) break;
                    before += sums[t];
                }
                if (t == kThreads) {  // (u of 1 or more: the last token with a weight)
                    t = last;
                    before = INFINITY;
                }
                uint32_t found = 0, end = min((t + 1) * per, a.vocab);
                double run = before;
                for (uint32_t v = t * per; v < end; ++v) {
                    const double w = weight(v, less);
                    if (w > 0) found = v;
                    run += w;
                    if (!(run <= border) && before != INFINITY) { found = v; break; }
                }
                token = static_cast<int32_t>(found);
            }
            stop = token >= 0;
        }
        __syncthreads();
        if (stop) break;
    }
    if (tid == 0) a.accepted[r] = static_cast<int32_t>(acc);
    for (uint32_t i = tid; i < span.count; i += kThreads) {
        if (i != acc) a.out[span.first + i] = i < acc ? a.tokens[span.first + i + 1] : -1;
        else if (tid != 0) continue;
    }
    if (tid == 0) a.out[span.first + acc] = token;
}

}  // namespace

extern "C" {

size_t vvli_gpu_verify_drafts_workspace(uint32_t requests, uint32_t vocab) {
    (void)requests, (void)vocab;
    return 16;
}

int vvli_gpu_verify_drafts(const float* target, uint64_t ldt, const float* draft, uint64_t ldd, const int32_t* tokens,
                           const int32_t* row_start, uint32_t requests, uint32_t rows, uint32_t vocab,
                           const float* u_accept, const float* u_sample, int32_t* accepted, int32_t* out,
                           void* workspace, size_t workspace_bytes, void* stream) {
    const char* who = "vvli_gpu_verify_drafts";
    if (!target || !tokens || !row_start || !u_accept || !u_sample || !accepted || !out || !workspace)
        return set_error(VVLI_NULL_ARG, "NULL argument to %s", who);
    if (requests == 0 || vocab == 0 || rows >= kPagedMost || requests >= kPagedMost || vocab >= kPagedMost || ldt < vocab ||
        ldt >= kPagedMost || (draft && (ldd < vocab || ldd >= kPagedMost)))
        return set_error(VVLI_INVALID_CONFIG, "%s: bad sizes (%u requests, %u rows of %u)", who, requests, rows, vocab);
    if (out == tokens) return set_error(VVLI_INVALID_CONFIG, "%s: out is tokens", who);
    if (!aligned16(workspace) || workspace_bytes < vvli_gpu_verify_drafts_workspace(requests, vocab))
        return set_error(VVLI_INVALID_CONFIG, "%s: workspace of %zu bytes", who, workspace_bytes);
    VerifyArgs a{target, draft, u_accept, u_sample, tokens, row_start, accepted, out, ldt, ldd, rows, vocab};
    PAGED_TRY(vlaunch(verify_kernel, dim3(requests), dim3(kThreads), 0, static_cast<hipStream_t>(stream), a));
    return VVLI_OK;
}

}  // extern "C"
