// A step's tables from its requests' lengths: block tables that grow and shrink with them out of a stack of free pages, and for
// every row its request, position and slot.
//
// Request r has L_r cached positions, brings n_r tokens and holds h_r pages of s positions. With need_r = ceil((L_r + n_r) / s) the
// pages need_r .. h_r - 1 of every request go back on the stack, the last request's last page first (so that pages taken in one call and
// given back whole in the next leave the stack as it was), then pages h_r .. need_r - 1 are popped for request after
// request. All or nothing: where pages or places are missing the status says so and nothing else is written.
//
// One block finds the sums over the requests (scans in shared memory) and moves the pages, a page a thread; the rows are written by the
// same block where they are few, by a second launch where they are many. What bounds it is the chain of dependent steps, not its bytes: 16 requests
// of up to five tokens 5.6 us, 1,024 of up to 128 (1.6 MB of rows) 7.3 + 5.0 us, with an empty launch at 2.5.
//
// Neither kernel lets the kernels behind it start early. The attention of single tokens reads positions, requests and block tables ahead of its wait (the
// engine's own steps have them copied in before their first kernel), and a wait is for the kernel right ahead only: a few kernels behind this one, with
// early starts all the way, it would read the tables of the step before.
#include <climits>

#include "common.cuh"

namespace gi {

constexpr int kTableThreads = 1024;            // also the requests of a turn
constexpr int kRowsHere = 4096;                // rows up to which the first launch writes them
constexpr int kRowsThreads = 256, kRowsEach = 2, kRowsStarts = 4096;

enum TableStatus : int { kTablesDone = 0, kTablesRows = -1, kTablesRequest = -2, kTablesValues = -3, kTablesStack = -4 };   // > 0: pages missing

struct TableArgs {
    const int* lengths;
    const int* counts;                         // not read where row_start is null (trimming)
    int* tables;
    int* held;
    int* free_pages;
    int* n_free;
    int* row_start;
    int* row_req;
    int* positions;
    int* slots;
    int* status;
    int R, stride, pool, page, rows;
};

// Exclusive scans of three numbers over the block at once; each returns its total, which every thread has.
struct Scan3 {
    long long v[3];
};
__device__ __forceinline__ Scan3 block_scan(long long (&x)[3], long long (&scratch)[3][32]) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    long long in[3];
#pragma unroll
    for (int k = 0; k < 3; ++k) {
        long long run = x[k];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long m = __shfl_up_sync(0xffffffffu, run, o);
            if (lane >= o) run += m;
        }
        in[k] = run - x[k];
        if (lane == 31) scratch[k][warp] = run;
    }
    __syncthreads();
    Scan3 total;
#pragma unroll
    for (int k = 0; k < 3; ++k) {
        long long run = scratch[k][lane];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long m = __shfl_up_sync(0xffffffffu, run, o);
            if (lane >= o) run += m;
        }
        total.v[k] = __shfl_sync(0xffffffffu, run, 31);
        const long long before = __shfl_sync(0xffffffffu, run, warp > 0 ? warp - 1 : 0);
        x[k] = in[k] + (warp > 0 ? before : 0);
    }
    __syncthreads();                           // the scratch is free again
    return total;
}

// The last of n ascending starts that is <= x (starts[0] <= x).
__device__ __forceinline__ int last_start(const int* starts, int n, int x) {
    int low = 0, high = n;
    while (high - low > 1) {
        const int mid = (low + high) >> 1;
        if (starts[mid] <= x) low = mid; else high = mid;
    }
    return low;
}

__device__ __forceinline__ void write_row(const TableArgs& a, int t, int r, int start) {
    const int pos = a.lengths[r] + (t - start);
    a.row_req[t] = r;
    a.positions[t] = pos;
    a.slots[t] = a.tables[static_cast<size_t>(r) * a.stride + pos / a.page] * a.page + pos % a.page;
}

__global__ void __launch_bounds__(kTableThreads, 1) step_tables_kernel(TableArgs a) {
    pdl_wait();
    __shared__ long long scratch[3][32];
    __shared__ int s_row[kTableThreads], s_page[kTableThreads], s_need[kTableThreads];
    __shared__ int s_wrong;
    const int n = *a.n_free, turns = (a.R + kTableThreads - 1) / kTableThreads;
    int length = 0, count = 0, need = 0, held = 0;
    bool fits = true;
    auto request = [&](int r) {                // the thread's request of a turn
        length = count = need = held = 0;
        fits = true;
        if (r >= a.R) return true;
        length = a.lengths[r];
        count = a.row_start ? a.counts[r] : 0;
        held = a.held[r];
        if (length < 0 || count < 0 || held < 0 || held > a.stride) return false;
        const long long end = static_cast<long long>(length) + count, pages = (end + a.page - 1) / a.page;
        fits = pages <= a.stride && end <= INT_MAX;             // (positions are 32-bit, also where a table has room for more)
        need = static_cast<int>(pages < a.stride ? pages : a.stride);
        return true;
    };
    // what a turn's scan gives: before this thread's request, and in all. One turn's is kept (1,024 requests: a pass over them 2 us shorter).
    long long kept[3];
    Scan3 kept_total;
    bool have = false, valid = true;
    auto scan = [&](int turn, long long (&x)[3]) {
        if (!(have && turns == 1)) {
            valid = request(turn * kTableThreads + threadIdx.x);
            x[0] = count;
            x[1] = max(held - need, 0);
            x[2] = max(need - held, 0);
            kept_total = block_scan(x, scratch);
            kept[0] = x[0]; kept[1] = x[1]; kept[2] = x[2];
            have = true;
        }
        x[0] = kept[0]; x[1] = kept[1]; x[2] = kept[2];
        return kept_total;
    };
    // ---- is there room for all of it?
    if (threadIdx.x == 0) s_wrong = n < 0 || n > a.pool ? kTablesValues : 0;
    __syncthreads();
    long long rows = 0, back = 0, take = 0;
    for (int turn = 0; turn < turns; ++turn) {
        long long x[3];
        const Scan3 total = scan(turn, x);
        if (!valid) s_wrong = kTablesValues;                // (the same from every thread that writes)
        else if (!fits) atomicCAS(&s_wrong, 0, static_cast<int>(kTablesRequest));
        rows += total.v[0]; back += total.v[1]; take += total.v[2];
    }
    __syncthreads();
    int wrong = s_wrong;
    if (!wrong && a.row_start && rows > a.rows) wrong = kTablesRows;
    if (!wrong && n + back > a.pool) wrong = kTablesStack;
    if (!wrong && take > n + back) wrong = static_cast<int>(take - n - back < INT_MAX ? take - n - back : INT_MAX);
    if (wrong) {
        if (threadIdx.x == 0) *a.status = wrong;
        return;
    }
    // ---- pages back on the stack, a page a thread
    const int top = n + static_cast<int>(back);
    long long first = 0;
    if (back > 0)
        for (int turn = 0; turn < turns; ++turn) {
            long long x[3];
            const Scan3 total = scan(turn, x);
            s_page[threadIdx.x] = static_cast<int>(x[1]);
            s_need[threadIdx.x] = need;
            __syncthreads();
            const int some = static_cast<int>(total.v[1]);
            for (int k = threadIdx.x; k < some; k += kTableThreads) {
                const int i = last_start(s_page, kTableThreads, k);
                int* entry = a.tables + static_cast<size_t>(turn * kTableThreads + i) * a.stride + s_need[i] + (k - s_page[i]);
                a.free_pages[top - 1 - static_cast<int>(first) - k] = *entry;
                *entry = -1;
            }
            first += some;
            __syncthreads();
        }
    // ---- pages from the stack, and the rows' starts
    first = 0;
    long long row = 0;
    for (int turn = 0; turn < turns; ++turn) {
        const int r = turn * kTableThreads + threadIdx.x;
        long long x[3];
        const Scan3 total = scan(turn, x);
        s_page[threadIdx.x] = static_cast<int>(x[2]);
        s_need[threadIdx.x] = held;
        s_row[threadIdx.x] = static_cast<int>(row + x[0]);
        __syncthreads();
        const int some = static_cast<int>(total.v[2]);
        for (int k = threadIdx.x; k < some; k += kTableThreads) {
            const int i = last_start(s_page, kTableThreads, k);
            a.tables[static_cast<size_t>(turn * kTableThreads + i) * a.stride + s_need[i] + (k - s_page[i])] = a.free_pages[top - 1 - static_cast<int>(first) - k];
        }
        if (r < a.R) {
            a.held[r] = need;
            if (a.row_start) a.row_start[r] = s_row[threadIdx.x];
        }
        first += some;
        row += total.v[0];
        __syncthreads();
    }
    if (threadIdx.x == 0) {
        *a.n_free = top - static_cast<int>(take);
        *a.status = kTablesDone;
        if (a.row_start) a.row_start[a.R] = static_cast<int>(rows);
    }
    if (!a.row_start || a.rows > kRowsHere || turns > 1) {
        __threadfence();
        return;
    }
    for (int t = threadIdx.x; t < a.rows; t += kTableThreads) {
        if (t < rows) {
            const int r = last_start(s_row, a.R, t);          // (of requests without rows at the same place the last: the one that has them)
            write_row(a, t, r, s_row[r]);
        } else {
            a.row_req[t] = -1;
            a.positions[t] = 0;
            a.slots[t] = -1;
        }
    }
    __threadfence();
}

// A block has neighbouring rows; the starts are searched in shared memory where that holds them.
__global__ void __launch_bounds__(kRowsThreads) step_rows_kernel(TableArgs a) {
    pdl_wait();
    __shared__ int s_start[kRowsStarts + 1];
    if (*a.status != kTablesDone) return;
    const int rows = a.row_start[a.R];
    const int* starts = a.row_start;
    if (a.R <= kRowsStarts) {
        for (int r = threadIdx.x; r <= a.R; r += kRowsThreads) s_start[r] = a.row_start[r];
        __syncthreads();
        starts = s_start;
    }
#pragma unroll
    for (int e = 0; e < kRowsEach; ++e) {
        const int t = (blockIdx.x * kRowsEach + e) * kRowsThreads + threadIdx.x;
        if (t < rows) {
            const int r = last_start(starts, a.R, t);
            write_row(a, t, r, starts[r]);
        } else if (t < a.rows) {
            a.row_req[t] = -1;
            a.positions[t] = 0;
            a.slots[t] = -1;
        }
    }
    __threadfence();
}

}  // namespace gi

using namespace gi;

// row_start null: the tables follow the lengths, no rows (counts, row_req, positions, slots are not used). pool: places of the stack.
static int gi_step_tables_impl(const int* lengths, const int* counts, int R, int* tables, int stride, int* held, int* free_pages, int* n_free, int pool,
                               int page, int* row_start, int* row_req, int* positions, int* slots, int rows, int* status, void* stream) {
    GI_REQUIRE(R >= 0 && stride >= 0 && pool >= 0 && rows >= 0, "step_tables: sizes must not be negative (R=%d, stride=%d, pool=%d, rows=%d)", R, stride, pool, rows);
    GI_REQUIRE(page > 0 && static_cast<long long>(pool) * page <= INT_MAX, "step_tables: %d pages of %d positions: slots must fit 32 bits", pool, page);
    const TableArgs a = {lengths, counts, tables, held, free_pages, n_free, row_start, row_req, positions, slots, status, R, stride, pool, page, rows};
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    launch_kernel((step_tables_kernel), dim3(1), dim3(kTableThreads), 0, st, a);
    if (check_launch("step_tables")) return 1;
    if (row_start && rows > 0 && (rows > kRowsHere || R > kTableThreads))
        launch_kernel((step_rows_kernel), dim3((rows + kRowsThreads * kRowsEach - 1) / (kRowsThreads * kRowsEach)), dim3(kRowsThreads), 0, st, a);
    return check_launch("step_tables");
}

extern "C" int gi_step_tables(const int* lengths, const int* counts, int R, int* tables, int stride, int* held, int* free_pages, int* n_free, int pool,
                              int page, int* row_start, int* row_req, int* positions, int* slots, int rows, int* status, void* stream) {
    return gi::dispatch(gi_step_tables_impl, lengths, counts, R, tables, stride, held, free_pages, n_free, pool, page, row_start, row_req, positions, slots,
                        rows, status, stream);
}
