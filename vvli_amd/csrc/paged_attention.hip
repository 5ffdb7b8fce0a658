// paged_attention.hip -- attention of the new rows of several requests over
// their pages (vvli_gpu_paged_attention).
#include <hip/hip_fp16.h>

#include "device_common.hpp"
#include "paged.hpp"

using namespace vvli;

namespace {

struct PagedAttnArgs {
    const void *k, *v;
    const int32_t *table, *row_start, *start_pos;
    const float* q;
    float* out;
    uint64_t slot_stride, ldq, ldo;
    uint32_t stride, requests, rows, heads, kv_heads, window, pages;
    PageDiv ps;
    float scale;
};

// One block per (row, head): each of its four waves takes every fourth key
// with a running maximum and sum, and wave 0 joins them.
template <int HD, typename T>
__global__ __launch_bounds__(256) void paged_attn_kernel(PagedAttnArgs a) {
    constexpr int E = (HD + 63) / 64;
    __shared__ float part[4][HD + 2];
    const uint32_t row = blockIdx.x, h = blockIdx.y, kvh = h / (a.heads / a.kv_heads);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t lo = 0, hi = a.requests;  // the request whose rows hold `row`
    while (lo < hi) {
        const uint32_t mid = (lo + hi) / 2;
        if (a.row_start[mid + 1] > static_cast<int64_t>(row)) hi = mid;
        else lo = mid + 1;
    }
    if (lo == a.requests) return;
    const RowSpan span = row_span(a.row_start[lo], a.row_start[lo + 1], a.rows);
    if (row < span.first || row >= span.first + span.count) return;
    const int32_t* table = a.table + static_cast<size_t>(lo) * a.stride;
    const KeySpan keys = key_span(static_cast<int64_t>(a.start_pos[lo]) + (row - span.first), a.window, a.stride * a.ps.d);
    const bool on = lane < HD;
    float q[E], o[E], m = -INFINITY, l = 0;
    for (int e = 0; e < E; ++e) q[e] = on ? a.q[row * a.ldq + static_cast<size_t>(h) * HD + lane + 64 * e] * a.scale : 0.f, o[e] = 0;
    for (uint32_t j = keys.lo + wave; j < keys.hi; j += 4) {
        const int32_t slot = page_slot(table, a.stride, a.pages, a.ps, j);
        if (slot < 0) continue;
        const uint64_t at = static_cast<uint64_t>(slot) * a.slot_stride + static_cast<size_t>(kvh) * HD + lane;
        float s = 0;
        for (int e = 0; e < E; ++e) s += on ? q[e] * static_cast<float>(static_cast<const T*>(a.k)[at + 64 * e]) : 0.f;
        s = wave_sum(s);
        const float m_new = fmaxf(m, s), base = m_new == -INFINITY ? 0.f : m_new;
        const float c = expf(m - base), p = expf(s - base);
        l = l * c + p;
        for (int e = 0; e < E; ++e) o[e] = o[e] * c + (on ? p * static_cast<float>(static_cast<const T*>(a.v)[at + 64 * e]) : 0.f);
        m = m_new;
    }
    for (int e = 0; e < E; ++e)
        if (on) part[wave][lane + 64 * e] = o[e];
    if (lane == 0) part[wave][HD] = m, part[wave][HD + 1] = l;
    __syncthreads();
    if (wave || !on) return;
    float top = -INFINITY;
    for (int w = 0; w < 4; ++w) top = fmaxf(top, part[w][HD]);
    if (top == -INFINITY) top = 0;
    float sum = 0;
    for (int e = 0; e < E; ++e) o[e] = 0;
    for (int w = 0; w < 4; ++w) {
        const float c = expf(part[w][HD] - top);
        sum += part[w][HD + 1] * c;
        for (int e = 0; e < E; ++e) o[e] += part[w][lane + 64 * e] * c;
    }
    for (int e = 0; e < E; ++e) a.out[row * a.ldo + static_cast<size_t>(h) * HD + lane + 64 * e] = sum == 0 ? 0.f : o[e] / sum;
}

template <int HD>
hipError_t launch(const PagedAttnArgs& a, uint32_t kind, hipStream_t s) {
    const dim3 grid(a.rows, a.heads), block(256);
    if (kind == VVLI_CACHE_F32) return vlaunch(paged_attn_kernel<HD, float>, grid, block, 0, s, a);
    if (kind == VVLI_CACHE_BF16) return vlaunch(paged_attn_kernel<HD, __bf16>, grid, block, 0, s, a);
    return vlaunch(paged_attn_kernel<HD, _Float16>, grid, block, 0, s, a);
}

bool sizes_ok(uint32_t rows, uint32_t requests, uint32_t heads, uint32_t kv_heads) {
    return requests != 0 && heads != 0 && kv_heads != 0 && heads % kv_heads == 0 && heads <= 65535 && rows < kPagedMost;
}

}  // namespace

extern "C" {

size_t vvli_gpu_paged_attention_workspace(uint32_t rows, uint32_t requests, uint32_t heads, uint32_t kv_heads,
                                          uint32_t head_dim) {
    if (!sizes_ok(rows, requests, heads, kv_heads) || (head_dim != 32 && head_dim != 64 && head_dim != 128)) return 0;
    return 16;
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
    PagedAttnArgs a{cache->k, cache->v, table,        row_start, start_pos, q,
                    out,      cache->slot_stride,     ldq,       ldo,       table_stride,
                    requests, rows,     heads,        cache->kv_heads, window, cache->pages,
                    page_div(cache->page_size),       scale};
    const hipStream_t s = static_cast<hipStream_t>(stream);
    PAGED_TRY(cache->head_dim == 128 ? launch<128>(a, cache->kind, s)
              : cache->head_dim == 64 ? launch<64>(a, cache->kind, s)
                                      : launch<32>(a, cache->kind, s));
    return VVLI_OK;
}

}  // extern "C"
