// attn_scan.h -- prefix sums over a workgroup, and lists whose elements find their owner in one (attn_plan.hip,
// attn_chunk.hip).
#pragma once

#include <limits.h>

#include "attn_common.h"

namespace tkm {

// The first i < n with end[i] > k (of a k below end[n - 1]).
__device__ __forceinline__ int first_above(const int* end, int n, int k) {
    int lo = 0, hi = n - 1;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (end[mid] > k) hi = mid;
        else lo = mid + 1;
    }
    return lo;
}

__device__ __forceinline__ int64_t lane_value64(int64_t v, int lane) {
    return (int64_t)(((uint64_t)(uint32_t)lane_value((int)(v >> 32), lane) << 32) | (uint32_t)lane_value((int)v, lane));
}

// A workgroup of T threads, each with an owner of some elements of a list.
template <int T>
struct Scan {
    static constexpr int WAVES = T / 64;
    int64_t part[2][WAVES];
    int end[T];          // behind each owner's last element,
    int arg[T][2];       // its first element, and what that stands for

    // Inclusive sum over the threads, and of all; `turn` alternates between calls.
    __device__ __forceinline__ int64_t sum(int turn, int64_t v, int64_t& all) {
        const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        const int64_t s = wave_scan(v);
        if (lane == 63) part[turn][wave] = s;
        __syncthreads();
        const int64_t p = wave_scan(lane < WAVES ? part[turn][lane] : (int64_t)0);
        all = lane_value64(p, 63);
        return s + (wave ? lane_value64(p, wave - 1) : 0);
    }

    // The owner's elements are first .. first + n of `all`: each(element, owner, what it stands for), the elements
    // of all owners dealt to the threads.  Ends with a barrier.
    template <class F>
    __device__ __forceinline__ void list(int64_t first, int n, int64_t all, int stands_for, F&& each) {
        constexpr int64_t most = INT_MAX;
        end[threadIdx.x] = (int)min(first + n, most);
        arg[threadIdx.x][0] = (int)min(first, most);
        arg[threadIdx.x][1] = stands_for;
        __syncthreads();
        const int total = (int)min(all, most);
#pragma unroll 1
        for (int64_t k = threadIdx.x; k < total; k += T) {
            const int i = first_above(end, T, (int)k);
            each((int)k, i, arg[i][1] + (int)k - arg[i][0]);
        }
        __syncthreads();
    }
};

}  // namespace tkm
