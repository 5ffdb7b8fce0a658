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

// Inclusive sums over the threads of a wave, saturating (new rows, whose inputs
// are unchecked: a sum that does not fit is over any number of rows), by
// row shifts and broadcasts of DPP.
#define ASSIGN_DPP(v, ctrl, rows) static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), ctrl, rows, 0xf, false))
__device__ __forceinline__ uint32_t wave_scan(uint32_t v) {
    v = __builtin_elementwise_add_sat(v, ASSIGN_DPP(v, 0x111, 0xf));
    v = __builtin_elementwise_add_sat(v, ASSIGN_DPP(v, 0x112, 0xf));
    v = __builtin_elementwise_add_sat(v, ASSIGN_DPP(v, 0x114, 0xf));
    v = __builtin_elementwise_add_sat(v, ASSIGN_DPP(v, 0x118, 0xf));
    v = __builtin_elementwise_add_sat(v, ASSIGN_DPP(v, 0x142, 0xa));
    v = __builtin_elementwise_add_sat(v, ASSIGN_DPP(v, 0x143, 0xc));
    return v;
}

struct Scratch {
    uint32_t sums[3][kWaves], carry[3];
    uint32_t taken;
    uint32_t row_end[kThreads];
    int32_t start[kThreads];
};

// One request, with the sums over those up to it.
struct Need {
    uint32_t held, keep, n, have, want;
    bool ok;
    uint32_t row_end, need, give, need_end, give_end;
};

// Sums over the block's threads on top of `before`.
__device__ __forceinline__ uint32_t block_scan(uint32_t v, uint32_t before, uint32_t* sums) {
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    v = wave_scan(v);
    if (lane == 63) sums[wave] = v;
    __syncthreads();
    uint32_t waves = wave_scan(lane < wave ? sums[lane] : 0);
    waves = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(waves), 63));
    return __builtin_elementwise_add_sat(__builtin_elementwise_add_sat(v, waves), before);
}

__device__ Need look(const AssignArgs& a, uint32_t r, const uint32_t (&before)[3], Scratch& sc) {
    Need x{};
    int32_t held = 0, keep = 0, add = 0;
    const bool there = r < a.requests;
    if (there) held = a.held[r], keep = a.keep[r], add = a.add[r];
    x.n = add > 0 ? add : 0;
    __syncthreads();  // (an earlier look's sums are read)
    x.row_end = block_scan(x.n, before[0], sc.sums[0]);
    const uint64_t room = static_cast<uint64_t>(a.stride) * a.ps.d;
    x.held = held, x.keep = keep;
    x.ok = there && add >= 0 && keep >= 0 && keep <= held && static_cast<uint64_t>(held) <= room &&
           static_cast<uint64_t>(keep) + x.n <= room && x.row_end <= a.rows;
    if (x.ok) {
        x.have = pages_for(a.ps, held), x.want = pages_for(a.ps, keep + x.n);
        x.need = x.want > x.have ? x.want - x.have : 0;
        x.give = x.have > x.want ? x.have - x.want : 0;
    }
    x.need_end = block_scan(x.need, before[1], sc.sums[1]);
    x.give_end = block_scan(x.give, before[2], sc.sums[2]);
    return x;
}

// What the next chunk of requests adds to: the last thread's sums.
__device__ void carry(const Need& x, uint32_t (&before)[3], Scratch& sc) {
    if (threadIdx.x == kThreads - 1) sc.carry[0] = x.row_end, sc.carry[1] = x.need_end, sc.carry[2] = x.give_end;
    __syncthreads();
    for (int i = 0; i < 3; ++i) before[i] = sc.carry[i];
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

// Position and slot of new row i, which is request r's.
__device__ __forceinline__ void put_row(const AssignArgs& a, uint32_t i, uint32_t r, int32_t start, uint32_t first) {
    const int32_t pos = start >= 0 ? start + static_cast<int32_t>(i - first) : -1;
    a.row_pos[i] = pos;
    a.slots[i] = pos >= 0 ? page_slot(a.table + static_cast<size_t>(r) * a.stride, a.stride, a.pages, a.ps, pos) : -1;
}

// One block: what the pages of a request are depends on all requests before it.
// Sums over the requests (a chunk of 1024 at a time, one chunk kept in
// registers), the given pages, the taken ones and, where they are few, the new
// rows follow one another with a barrier between; latency bounds it (48 requests
// of one row each 9.2 us, 300 of up to 130 rows 13.9 with assign_rows_kernel).
__global__ __launch_bounds__(kThreads) void assign_kernel(AssignArgs a, bool with_rows) {
    __shared__ Scratch sc;
    const uint32_t tid = threadIdx.x, chunks = (a.requests + kThreads - 1) / kThreads;
    int32_t count = a.free_count[0];
    // First the sums over all requests: pages are taken from what all of them give.
    uint32_t before[3] = {0, 0, 0};
    Need x{};
    for (uint32_t c = 0; c < chunks; ++c) {
        const uint32_t r = c * kThreads + tid;
        x = look(a, r, before, sc);
        if (r < a.requests) {
            if (r == 0) a.row_start[0] = 0;
            a.row_start[r + 1] = static_cast<int32_t>(min(x.row_end, a.rows));
        }
        carry(x, before, sc);
    }
    count = count < 0 ? 0 : count > static_cast<int32_t>(a.pages) ? a.pages : count;
    // (never over the stack's room: requests hold different pages)
    const uint32_t avail = min(static_cast<uint32_t>(count) + before[2], a.pages);
    if (before[2]) {
        before[0] = before[1] = before[2] = 0;
        for (uint32_t c = 0; c < chunks; ++c) {
            const uint32_t r = c * kThreads + tid;
            if (chunks > 1) x = look(a, r, before, sc), carry(x, before, sc);
            each_page(r, x.give, x.want, x.give_end - x.give, [&](uint32_t q, uint32_t entry, uint32_t k) {
                int32_t* e = a.table + static_cast<size_t>(q) * a.stride + entry;
                if (k < avail) a.free_pages[avail - 1 - k] = *e;
                *e = -1;
            });
        }
        __syncthreads();
    }
    before[0] = before[1] = before[2] = 0;
    if (tid == 0) sc.taken = 0;
    uint32_t taken = 0;
    for (uint32_t c = 0; c < chunks; ++c) {
        const uint32_t r = c * kThreads + tid;
        if (chunks > 1) x = look(a, r, before, sc), carry(x, before, sc);
        const bool served = x.ok && (x.need == 0 || x.need_end <= avail);
        const uint32_t need = served ? x.need : 0;
        if (need) taken = x.need_end;
        each_page(r, need, x.have, x.need_end - x.need, [&](uint32_t q, uint32_t entry, uint32_t k) {
            a.table[static_cast<size_t>(q) * a.stride + entry] = a.free_pages[avail - 1 - k];
        });
        if (r < a.requests) {
            const int32_t start = served ? static_cast<int32_t>(x.keep) : -static_cast<int32_t>(x.n);
            a.len[r] = served ? x.keep + x.n : x.held;
            a.start_pos[r] = start;
            if (with_rows) sc.row_end[tid] = min(x.row_end, a.rows), sc.start[tid] = start;
        }
    }
    // The served requests that need pages are the first ones that do.
    __syncthreads();
    if (taken) atomicMax(&sc.taken, taken);
    __syncthreads();
    if (tid == 0) a.free_count[0] = static_cast<int32_t>(avail - sc.taken);
    if (!with_rows) return;
    const uint32_t rows = sc.row_end[a.requests - 1];
    for (uint32_t i = tid; i < rows; i += kThreads) {
        uint32_t lo = 0, hi = a.requests - 1;  // the first request whose rows end behind i
        while (lo < hi) {
            const uint32_t mid = (lo + hi) / 2;
            if (sc.row_end[mid] > i) hi = mid;
            else lo = mid + 1;
        }
        put_row(a, i, lo, sc.start[lo], lo ? sc.row_end[lo - 1] : 0);
    }
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
    put_row(a, i, lo, a.start_pos[lo], a.row_start[lo]);
}

// Rows that the one block places itself; more are worth a launch over the GPU
// (400 rows: 10.9 us in the block, 13.9 with the launch; 39000: 27 and 15).
constexpr uint32_t kRowsInBlock = 2048;

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
    const bool with_rows = rows != 0 && rows <= kRowsInBlock && pool->requests <= kThreads;
    PAGED_TRY(vlaunch(assign_kernel, dim3(1), dim3(kThreads), 0, s, a, with_rows));
    if (rows && !with_rows) PAGED_TRY(vlaunch(assign_rows_kernel, dim3((rows + 255) / 256), dim3(256), 0, s, a));
    return VVLI_OK;
}
