// attn_plan.hip -- pages, lengths and slots of a serving step from its requests (gfx950).
//
// For sequences b in order, t_b = ceil((start_b + want_b) / page), held_b the pages of its table row:
//   back_b = max(0, held_b - t_b)     go on the stack of free pages, positions ascending
//   need_b = max(0, t_b - held_b)     if sum_{c <= b} need_c <= free + sum back, and the rows fit behind all that had pages
//   row_start_b = sum_{c < b} n_c;  row r of b: position start_b + r - row_start_b, slot page * size + token
// Four prefix sums over the sequences, and two lists (pages and rows) whose elements find their sequence in a prefix
// sum by bisection.  Bound by latency: one workgroup goes through the sequences, 1024 at a time, so that the
// order of sequences is the order of the sums and nothing depends on timing.
#include <hip/hip_runtime.h>

#include "attn_common.h"
#include "attn_kv.h"
#include "attn_launch.h"
#include "attn_scan.h"

namespace tkm {
namespace {

constexpr int T = 1024;

struct Request {
    int start, want, held, target, back, need;
    bool in_table;
};
__device__ __forceinline__ Request request_of(const PlanArgs& a, int b) {
    Request q{};
    if (b >= a.kv.B) return q;
    const int cap = a.kv.max_pages * a.kv.page, shift = __ffs(a.kv.page) - 1;
    q.start = a.start ? a.start[b] : a.kv.len[b];
    q.held = max(0, min(a.pages.held[b], a.kv.max_pages));
    q.in_table = q.start >= 0 && q.start <= cap;
    const int want = a.want[b];
    q.want = q.in_table && want > 0 && want <= cap - q.start ? want : 0;
    q.target = q.in_table ? (q.start + q.want + a.kv.page - 1) >> shift : q.held;
    q.back = max(0, q.held - q.target);
    q.need = q.want ? max(0, q.target - q.held) : 0;
    return q;
}

__device__ __forceinline__ int64_t slot_of(const tkm_attn_kv& kv, int b, int pos) {
    const int shift = __ffs(kv.page) - 1, page = kv.table[(long long)b * kv.max_pages + (pos >> shift)];
    return (unsigned)page < (unsigned)kv.num_pages ? ((int64_t)page << shift) + (pos & (kv.page - 1)) : -1;
}

// Where row k of a list of sequences' rows is, and its slot.
__device__ __forceinline__ void put_row(const PlanArgs& a, int r, int b, int pos) {
    a.plan.seq[r] = b;
    a.plan.pos[r] = pos;
    a.plan.slot[r] = b < 0 ? -1 : slot_of(a.kv, b, pos);
}

// SLOTS: also seq, pos and slot of every row.
template <bool SLOTS>
__global__ __launch_bounds__(T) void plan_kernel(PlanArgs a) {
    __shared__ Scan<T> lds;
    const tkm_attn_kv& kv = a.kv;
    int32_t* table = const_cast<int32_t*>(kv.table);
    const int tid = threadIdx.x, B = kv.B;
    const int64_t had = max(0, min(*a.pages.n_free, kv.num_pages));
    // what comes back
    int64_t top = had, all;
    for (int c = 0; c < B; c += T) {
        const Request q = request_of(a, c + tid);
        const int64_t s = lds.sum(0, q.back, all);
        if (all) {
            lds.list(s - q.back, q.back, all, q.target, [&](int k, int i, int p) {
                const long long at = (long long)(c + i) * kv.max_pages + p;
                if (top + k < kv.num_pages) a.pages.free[top + k] = table[at];
                table[at] = -1;
            });
        }
        top += all;
        __syncthreads();
    }
    top = min(top, (int64_t)kv.num_pages);

    // what is taken, and the rows: sums over the sequences before the chunk
    int64_t asked = 0, wanted = 0, taken = 0, rows = 0;
    for (int c = 0; c < B; c += T) {
        const int b = c + tid;
        const Request q = request_of(a, b);
        const int64_t ask = asked + lds.sum(0, q.need, all);
        asked += all;
        int n = q.need == 0 || ask <= top ? q.want : 0;
        const int64_t fill = wanted + lds.sum(1, n, all);
        wanted += all;
        if (fill > a.rows) n = 0;
        const int take = n ? q.need : 0;
        int64_t all_pages, all_rows;
        const int64_t pages_end = lds.sum(0, take, all_pages), rows_end = lds.sum(1, n, all_rows);
        if (b < B) {
            a.pages.held[b] = q.held - q.back + take;
            kv.len[b] = q.start + n;
            a.plan.n_new[b] = n;
            a.plan.row_start[b] = (int)(rows + rows_end - n);
        }
        if (all_pages) {
            lds.list(pages_end - take, take, all_pages, q.held, [&](int k, int i, int p) {
                const int64_t at = top - 1 - taken - k;
                table[(long long)(c + i) * kv.max_pages + p] = at >= 0 ? a.pages.free[at] : -1;
            });
        }
        if (SLOTS && all_rows)
            lds.list(rows_end - n, n, all_rows, q.start, [&](int k, int i, int pos) { put_row(a, (int)rows + k, c + i, pos); });
        taken += all_pages;
        rows += all_rows;
        __syncthreads();      // the sums' parts are written again
    }
    if (SLOTS)
        for (int64_t r = rows + tid; r < a.rows; r += T) put_row(a, (int)r, -1, -1);
    if (tid == 0) {
        a.plan.row_start[B] = (int)rows;
        *a.pages.n_free = (int)(top - taken);
    }
}

// Sequences whose first rows a workgroup holds in LDS.
constexpr int kHeld = 4096;

__global__ __launch_bounds__(256) void slots_kernel(PlanArgs a) {
    __shared__ int ends[kHeld];
    const int B = a.kv.B, r = blockIdx.x * 256 + threadIdx.x;
    const int32_t* end = a.plan.row_start + 1;
    if (B <= kHeld) {
        for (int i = threadIdx.x; i < B; i += 256) ends[i] = end[i];
        __syncthreads();
    }
    if (r >= a.rows) return;
    if (r >= end[B - 1]) return put_row(a, r, -1, -1);
    const int b = B <= kHeld ? first_above(ends, B, r) : first_above(end, B, r);
    // the position of a sequence's last row is its length less one
    put_row(a, r, b, a.kv.len[b] - (end[b] - r));
}

// Rows up to which the planning workgroup lays them out itself, in one launch (kernels, one launch and two: 64 rows 6.0 and
// 7.1 us, 3000 7.8 and 8.3, 6000 9.7 and 8.3, 12500 14.2 and 8.2).
constexpr int kOwnRows = 4096;

}  // namespace

int launch_plan(const PlanArgs& a) {
    note_kernels(kPlan);
    const bool own = a.rows <= kOwnRows;
    if (own) hipLaunchKernelGGL(plan_kernel<true>, dim3(1), dim3(T), 0, (hipStream_t)a.stream, a);
    else hipLaunchKernelGGL(plan_kernel<false>, dim3(1), dim3(T), 0, (hipStream_t)a.stream, a);
    if (hipGetLastError() != hipSuccess) return -1;
    if (own) return 0;
    hipLaunchKernelGGL(slots_kernel, dim3(((unsigned)a.rows + 255) / 256), dim3(256), 0, (hipStream_t)a.stream, a);
    return hipGetLastError() == hipSuccess ? 0 : -1;
}

}  // namespace tkm
