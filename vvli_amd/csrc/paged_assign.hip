// paged_assign.hip -- pages, cache slots and row numbers of one step's new
// rows (vvli_gpu_paged_assign).
#include "paged.hpp"

using namespace vvli;

namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64;

struct AssignArgs {
    int32_t *free_pages, *free_count, *table;
    const int32_t *held, *keep, *add;
    int32_t *len, *row_start, *start_pos, *row_pos;
    int64_t* slots;
    uint32_t requests, stride, pages, rows;
    PageDiv ps;
};

// Inclusive sums over the block of two values (64-bit: new rows, whose inputs
// are unchecked, and pages taken and given in the two halves of one word,
// which stay below 2^31 each).
__device__ uint64_t block_scan(uint64_t v, uint64_t* sums) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint64_t u = __shfl_up(v, o, 64);
        if (lane >= o) v += u;
    }
    __syncthreads();  // (an earlier scan's sums are read)
    if (lane == 63) sums[wave] = v;
    __syncthreads();
    uint64_t before = 0;
    for (int w = 0; w < wave; ++w) before += sums[w];
    return v + before;
}

// One request, with the sums over those up to it.
struct Need {
    uint32_t held, keep, n, have, want;
    bool ok;
    uint64_t row_end;
    uint32_t need, give, need_end, give_end;
};

__device__ Need look(const AssignArgs& a, uint32_t r, uint64_t rows_before, uint64_t pages_before, uint64_t* sums) {
    Need x{};
    int32_t held = 0, keep = 0, add = 0;
    const bool there = r < a.requests;
    if (there) held = a.held[r], keep = a.keep[r], add = a.add[r];
    x.n = add > 0 ? add : 0;
    x.row_end = rows_before + block_scan(x.n, sums);
    const uint64_t room = static_cast<uint64_t>(a.stride) * a.ps.d;
    x.held = held, x.keep = keep;
    x.ok = there && add >= 0 && keep >= 0 && keep <= held && static_cast<uint64_t>(held) <= room &&
           static_cast<uint64_t>(keep) + x.n <= room && x.row_end <= a.rows;
    if (x.ok) {
        x.have = pages_for(a.ps, held), x.want = pages_for(a.ps, keep + x.n);
        x.need = x.want > x.have ? x.want - x.have : 0;
        x.give = x.have > x.want ? x.have - x.want : 0;
    }
    const uint64_t p = pages_before + block_scan(static_cast<uint64_t>(x.give) << 32 | x.need, sums);
    x.need_end = static_cast<uint32_t>(p), x.give_end = static_cast<uint32_t>(p >> 32);
    return x;
}

// f(r, entry, k) for n consecutive entries of each lane's request in the table
// and places in L: by the lane itself where they are few, else by its wave.
template <typename F>
__device__ void each_page(uint32_t r, uint32_t n, uint32_t entry, uint32_t k, F&& f) {
    const uint32_t lane = threadIdx.x & 63;
    if (n <= 4)
        for (uint32_t i = 0; i < n; ++i) f(r, entry + i, k + i);
    for (uint64_t todo = __ballot(n > 4); todo; todo &= todo - 1) {
        const int from = __builtin_ctzll(todo);
        const uint32_t fr = __shfl(r, from, 64), fn = __shfl(n, from, 64), fe = __shfl(entry, from, 64), fk = __shfl(k, from, 64);
        for (uint32_t i = lane; i < fn; i += 64) f(fr, fe + i, fk + i);
    }
}

__global__ __launch_bounds__(kThreads) void assign_kernel(AssignArgs a) {
    __shared__ uint64_t sums[kWaves];
    __shared__ uint64_t carry[2];
    const uint32_t tid = threadIdx.x, chunks = (a.requests + kThreads - 1) / kThreads;
    // First the sums over all requests: pages are taken from what all of them give.
    uint64_t rows_before = 0, pages_before = 0;
    Need x{};
    for (uint32_t c = 0; c < chunks; ++c) {
        const uint32_t r = c * kThreads + tid;
        x = look(a, r, rows_before, pages_before, sums);
        if (r < a.requests) {
            if (r == 0) a.row_start[0] = 0;
            a.row_start[r + 1] = static_cast<int32_t>(x.row_end < a.rows ? x.row_end : a.rows);
        }
        if (tid == kThreads - 1) carry[0] = x.row_end, carry[1] = static_cast<uint64_t>(x.give_end) << 32 | x.need_end;
        __syncthreads();
        rows_before = carry[0], pages_before = carry[1];
    }
    int32_t count = a.free_count[0];
    count = count < 0 ? 0 : count > static_cast<int32_t>(a.pages) ? a.pages : count;
    // (never over the stack's room: requests hold different pages)
    const uint32_t given = static_cast<uint32_t>(pages_before >> 32);
    const uint32_t avail = min(static_cast<uint32_t>(count) + given, a.pages);
    __syncthreads();
    rows_before = pages_before = 0;
    for (uint32_t c = 0; c < chunks; ++c) {
        const uint32_t r = c * kThreads + tid;
        if (chunks > 1) {
            x = look(a, r, rows_before, pages_before, sums);
            if (tid == kThreads - 1) carry[0] = x.row_end, carry[1] = static_cast<uint64_t>(x.give_end) << 32 | x.need_end;
            __syncthreads();
            rows_before = carry[0], pages_before = carry[1];
        }
        each_page(r, x.give, x.want, x.give_end - x.give, [&](uint32_t q, uint32_t entry, uint32_t k) {
            int32_t* e = a.table + static_cast<size_t>(q) * a.stride + entry;
            if (k < avail) a.free_pages[avail - 1 - k] = *e;
            *e = -1;
        });
    }
    __syncthreads();
    rows_before = pages_before = 0;
    uint32_t taken = 0;
    for (uint32_t c = 0; c < chunks; ++c) {
        const uint32_t r = c * kThreads + tid;
        if (chunks > 1) {
            x = look(a, r, rows_before, pages_before, sums);
            if (tid == kThreads - 1) carry[0] = x.row_end, carry[1] = static_cast<uint64_t>(x.give_end) << 32 | x.need_end;
            __syncthreads();
            rows_before = carry[0], pages_before = carry[1];
        }
        const bool served = x.ok && (x.need == 0 || x.need_end <= avail);
        const uint32_t need = served ? x.need : 0;
        if (need) taken = x.need_end;
        each_page(r, need, x.have, x.need_end - x.need, [&](uint32_t q, uint32_t entry, uint32_t k) {
            a.table[static_cast<size_t>(q) * a.stride + entry] = a.free_pages[avail - 1 - k];
        });
        if (r < a.requests) {
            a.len[r] = served ? x.keep + x.n : x.held;
            a.start_pos[r] = served ? static_cast<int32_t>(x.keep) : -static_cast<int32_t>(x.n);
        }
    }
    // The served requests that need pages are the first ones that do.
    if (tid == 0) carry[0] = 0;
    __syncthreads();
    if (taken) atomicMax(reinterpret_cast<unsigned long long*>(&carry[0]), static_cast<unsigned long long>(taken));
    __syncthreads();
    if (tid == 0) a.free_count[0] = static_cast<int32_t>(avail - static_cast<uint32_t>(carry[0]));
}

// Positions and slots of the new rows: the request of a row by halving over row_start.
__global__ __launch_bounds__(256) void assign_rows_kernel(AssignArgs a) {
    const uint32_t i = blockIdx.x * 256 + threadIdx.x;
    if (i >= static_cast<uint32_t>(a.row_start[a.requests])) return;
    uint32_t lo = 0, hi = a.requests - 1;  // the first request whose rows end behind i
    while (lo < hi) {
        const uint32_t mid = (lo + hi) / 2;
        if (static_cast<uint32_t>(a.row_start[mid + 1]) > i) hi = mid;
        else lo = mid + 1;
    }
    int32_t pos = a.start_pos[lo];
    int32_t slot = -1;
    if (pos >= 0) {
        pos += static_cast<int32_t>(i - a.row_start[lo]);
        slot = page_slot(a.table + static_cast<size_t>(lo) * a.stride, a.stride, a.pages, a.ps, pos);
    } else {
        pos = -1;
    }
    a.row_pos[i] = pos;
    a.slots[i] = slot;
}

}  // namespace

extern "C" int vvli_gpu_paged_assign(const vvli_gpu_page_pool* pool, const int32_t* held, const int32_t* keep,
                                     const int32_t* add, uint32_t rows, int32_t* len, int32_t* row_start,
                                     int32_t* start_pos, int32_t* row_pos, int64_t* slots, void* stream) {
    const char* who = "vvli_gpu_paged_assign";
    if (!pool || !pool->free_pages || !pool->free_count || !pool->table || !held || !keep || !add || !len || !row_start ||
        !start_pos || (rows && (!row_pos || !slots)))
        return set_error(VVLI_NULL_ARG, "NULL argument to %s", who);
    const uint64_t r = pool->requests, st = pool->table_stride, ps = pool->page_size, n = pool->pages;
    if (r == 0 || st == 0 || ps == 0 || n == 0 || rows >= kPagedMost || r * st >= kPagedMost || st * ps >= kPagedMost ||
        n * ps >= kPagedMost)
        return set_error(VVLI_INVALID_CONFIG, "%s: bad sizes (%u requests, %u pages of %u slots, table rows of %u, %u rows)",
                         who, pool->requests, pool->pages, pool->page_size, pool->table_stride, rows);
    AssignArgs a{pool->free_pages, pool->free_count, pool->table,      held,           keep,
                 add,              len,              row_start,        start_pos,      row_pos,
                 slots,            pool->requests,   pool->table_stride, pool->pages, rows,
                 page_div(pool->page_size)};
    const hipStream_t s = static_cast<hipStream_t>(stream);
    PAGED_TRY(vlaunch(assign_kernel, dim3(1), dim3(kThreads), 0, s, a));
    if (rows) PAGED_TRY(vlaunch(assign_rows_kernel, dim3((rows + 255) / 256), dim3(256), 0, s, a));
    return VVLI_OK;
}
