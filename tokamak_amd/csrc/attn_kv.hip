// attn_kv.hip -- the paged key-value cache's own kernels (gfx950): rows of packed QKV into it, and eviction
// from it by accumulated attention weight.  The layout is in attn_kv.h.
//
// All of these move data and are bound by HBM, or by the launch where there is little to move.
#include <hip/hip_runtime.h>
#include <limits.h>

#include "attn_common.h"
#include "attn_kv.h"
#include "attn_launch.h"

namespace tkm {
namespace {

// Elements before the 32-token tile of `tile` (within its page) of a page's kv head.
__device__ __forceinline__ long long tile_at(const tkm_attn_kv& kv, int page, int h, int tile) {
    return (((long long)page * kv.Hkv + h) * (kv.page / 32) + tile) * (32 * kv.D);
}
__device__ __forceinline__ bool in_pool(const tkm_attn_kv& kv, int page) { return (unsigned)page < (unsigned)kv.num_pages; }

// Rows a sequence receives and where they start; the length it then has. A start outside the table writes
// nothing and leaves a length that every reader refuses.
struct Rows {
    int start, n, len;
};
__device__ __forceinline__ Rows rows_of(const AppendArgs& a, int b) {
    Rows r;
    r.start = a.start ? a.start[b] : a.kv.len[b];
    r.n = a.S;
    if (a.n_new) r.n = max(0, min(a.n_new[b], a.S));
    if (r.start < 0) {
        r.n = 0;
        r.len = -1;
    } else {
        r.len = r.start > INT_MAX - r.n ? INT_MAX : r.start + r.n;
    }
    return r;
}

// One row a sequence (a decoding step): a workgroup copies all kv heads of one row. V's 16-bit values go to
// 64-byte rows of their own.
__global__ __launch_bounds__(256) void append_one_kernel(AppendArgs a) {
    const tkm_attn_kv& kv = a.kv;
    const int b = blockIdx.x, pos = rows_of(a, b).start;
    const Rows r = rows_of(a, b);
    const int cap = kv.max_pages * kv.page;
    if (r.n == 1 && pos < cap) {
        const int page = kv.table[(long long)b * kv.max_pages + pos / kv.page];
        const int tile = pos % kv.page / 32, t = pos % 32, chunks = kv.D / 8;
        if (in_pool(kv, page)) {
            const uint16_t* row = (const uint16_t*)a.qkv + ((long long)b * (a.Hq + 2 * kv.Hkv) + a.Hq) * kv.D;
            for (int i = threadIdx.x; i < 2 * kv.Hkv * chunks; i += 256) {
                const u32x4 x = ld_global16(row + i * 8);
                const int h = i / chunks % kv.Hkv, c = i % chunks;
                const long long at = tile_at(kv, page, h, tile) + c / 4 * 1024;
                if (i < kv.Hkv * chunks) {
                    *(u32x4*)((uint16_t*)kv.k + at + t * 32 + c % 4 * 8) = x;
                } else {
                    uint16_t* v = (uint16_t*)kv.v + at + c % 4 * 8 * 32 + t;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        v[2 * j * 32] = (uint16_t)x[j];
                        v[(2 * j + 1) * 32] = (uint16_t)(x[j] >> 16);
                    }
                }
            }
            if (kv.weight)
                for (int h = threadIdx.x; h < kv.Hkv; h += 256) kv.weight[((long long)b * kv.Hkv + h) * cap + pos] = 0.f;
        }
    }
    __syncthreads();      // every thread has its start: it may be the length itself
    if (threadIdx.x == 0) kv.len[b] = r.len;
}

// Several rows a sequence: a workgroup fills (its part of) one tile of one kv head; V is transposed through LDS.
__global__ __launch_bounds__(256) void append_rows_kernel(AppendArgs a, int tiles) {
    const tkm_attn_kv& kv = a.kv;
    __shared__ __attribute__((aligned(16))) uint16_t vt[128][40];   // [dim][token]: rows 80 bytes apart
    const int ti = blockIdx.x % tiles, h = blockIdx.x / tiles % kv.Hkv, b = blockIdx.x / tiles / kv.Hkv;
    const Rows r = rows_of(a, b);
    const int cap = kv.max_pages * kv.page;
    if (a.start && ti == 0 && h == 0 && threadIdx.x == 0) kv.len[b] = r.len;   // else advance_kernel does
    if (r.start < 0 || r.start >= cap) return;
    const int end = (int)min((long long)r.start + r.n, (long long)cap);      // first position not written
    const int t0 = (r.start / 32 + ti) * 32;
    if (t0 >= end) return;
    const int page = kv.table[(long long)b * kv.max_pages + t0 / kv.page];
    if (!in_pool(kv, page)) return;
    const long long at = tile_at(kv, page, h, t0 % kv.page / 32);
    uint16_t* kd = (uint16_t*)kv.k + at;
    uint16_t* vd = (uint16_t*)kv.v + at;
    const int W = (a.Hq + 2 * kv.Hkv) * kv.D, chunks = kv.D / 8;
    for (int i = threadIdx.x; i < 32 * chunks; i += 256) {
        const int t = i / chunks, c = i % chunks, pos = t0 + t;
        if (pos < r.start || pos >= end) continue;
        const uint16_t* src = (const uint16_t*)a.qkv + ((long long)b * a.S + (pos - r.start)) * W + (a.Hq + h) * kv.D + c * 8;
        *(u32x4*)(kd + c / 4 * 1024 + t * 32 + c % 4 * 8) = ld_global16(src);
        const u32x4 x = ld_global16(src + kv.Hkv * kv.D);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            vt[c * 8 + 2 * j][t] = (uint16_t)x[j];
            vt[c * 8 + 2 * j + 1][t] = (uint16_t)(x[j] >> 16);
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < kv.D * 4; i += 256) {
        const int d = i / 4, t = i % 4 * 8, pos = t0 + t;
        if (pos >= r.start && pos + 8 <= end) {
            *(u32x4*)(vd + d * 32 + t) = *(const u32x4*)&vt[d][t];
        } else {
            for (int j = 0; j < 8; ++j)
                if (pos + j >= r.start && pos + j < end) vd[d * 32 + t + j] = vt[d][t + j];
        }
    }
    if (kv.weight && threadIdx.x < 32) {
        const int pos = t0 + threadIdx.x;
        if (pos >= r.start && pos < end) kv.weight[((long long)b * kv.Hkv + h) * cap + pos] = 0.f;
    }
}

__global__ __launch_bounds__(256) void advance_kernel(AppendArgs a) {
    const int b = blockIdx.x * 256 + threadIdx.x;
    if (b < a.kv.B) a.kv.len[b] = rows_of(a, b).len;
}

// ---- eviction -----------------------------------------------------------------------------------

// A weight as an integer of the same order; NaN below all others, -0 as +0.
__device__ __forceinline__ uint32_t key_of(float w) {
    if (w != w) return 0u;
    const uint32_t u = __float_as_uint(w + 0.0f);
    return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

constexpr int kSel = 1024;   // threads of a selecting workgroup

struct SelectLds {
    int count[3][4];
    int wave[2][kSel / 64][2];
};

// The largest key K such that at least r of the n weights have a key >= K (r >= 1), and the number above K:
// 16 rounds of two bits, each counting three candidates at once by ballots.  E > 0: the keys stay in E
// registers a thread; E = 0: they are read again each round.
template <int E>
__device__ void find_key(const float* w, int n, int r, SelectLds& lds, uint32_t& key, int& above) {
    const int tid = threadIdx.x, lane = tid & 63;
    uint32_t k[E > 0 ? E : 1];
    if constexpr (E > 0) {
#pragma unroll
        for (int e = 0; e < E; ++e) k[e] = e * kSel + tid < n ? key_of(w[e * kSel + tid]) : 0u;
    }
    if (tid < 4) lds.count[0][tid] = 0;
    __syncthreads();
    key = 0u;
    above = 0;
    for (int i = 0; i < 16; ++i) {
        const uint32_t step = 1u << (30 - 2 * i);
        const uint32_t k1 = key + step, k2 = k1 + step, k3 = k2 + step;
        int c1 = 0, c2 = 0, c3 = 0;   // of the wave
        auto one = [&](uint32_t x) {  // candidates are above 0, the key of what is not there
            c1 += __popcll(__ballot(x >= k1));
            c2 += __popcll(__ballot(x >= k2));
            c3 += __popcll(__ballot(x >= k3));
        };
        if constexpr (E > 0) {
#pragma unroll
            for (int e = 0; e < E; ++e) one(k[e]);
        } else {
            for (int j = 0; j < n; j += kSel) one(j + tid < n ? key_of(w[j + tid]) : 0u);
        }
        if (lane == 0) {
            atomicAdd(&lds.count[i % 3][1], c1);
            atomicAdd(&lds.count[i % 3][2], c2);
            atomicAdd(&lds.count[i % 3][3], c3);
        }
        if (tid < 4) lds.count[(i + 1) % 3][tid] = 0;   // last read two rounds ago, before the last barrier
        __syncthreads();
        c1 = lds.count[i % 3][1];
        c2 = lds.count[i % 3][2];
        c3 = lds.count[i % 3][3];
        if (c3 >= r) {
            key = k3;
        } else if (c2 >= r) {
            key = k2;
            above = c3;
        } else if (c1 >= r) {
            key = k1;
            above = c2;
        } else {
            above = c1;
        }
    }
    __syncthreads();
}

// Chooses what one kv head of one sequence keeps: writes its old positions in ascending order to `kept`, and
// their weights to their new places.  A sequence with a length or a page that its tables cannot have gets -1s.
__global__ __launch_bounds__(kSel) void select_kernel(EvictArgs a) {
    __shared__ SelectLds lds;
    const tkm_attn_kv& s = a.src;
    const tkm_attn_kv& d = a.dst;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const long long row = blockIdx.x;
    const int b = (int)(row / s.Hkv);
    const long long cap = (long long)s.max_pages * s.page, cap_d = (long long)d.max_pages * d.page;
    const int n = s.len[b];
    int32_t* kept = a.kept + row * a.budget;
    int bad = n < 0 || n > cap;
    if (!bad) {
        const int most = min(n, a.budget);
        for (int i = tid; i < (n + s.page - 1) / s.page; i += kSel) bad |= !in_pool(s, s.table[(long long)b * s.max_pages + i]);
        for (int i = tid; i < (most + d.page - 1) / d.page; i += kSel) bad |= !in_pool(d, d.table[(long long)b * d.max_pages + i]);
    }
    if (__syncthreads_or(bad)) {
        for (int i = tid; i < a.budget; i += kSel) kept[i] = -1;
        return;
    }
    const float* w = s.weight + row * cap;
    float* wd = d.weight ? d.weight + row * cap_d : nullptr;
    if (n <= a.budget) {
        for (int i = tid; i < a.budget; i += kSel) {
            kept[i] = i < n ? i : -1;
            if (wd && wd != w && i < n) wd[i] = w[i];
        }
        return;
    }
    const int lo = a.sink, hi = n - a.recent, r = a.budget - a.sink - a.recent;
    uint32_t key = 0xffffffffu;
    int above = 0;
    if (r > 0) {
        if (hi - lo <= 8 * kSel) find_key<8>(w + lo, hi - lo, r, lds, key, above);
        else if (hi - lo <= 32 * kSel) find_key<32>(w + lo, hi - lo, r, lds, key, above);
        else find_key<0>(w + lo, hi - lo, r, lds, key, above);
    }
    const int ties = r - above;      // of the weights equal to the key, the first ones
    int sure = 0, equal = 0;         // before this chunk
    for (int c = 0; c < n; c += kSel) {
        const int i = c + tid, buf = (c / kSel) & 1;
        const float x = i < n ? w[i] : 0.f;
        const uint32_t k = key_of(x);
        const bool mid = i >= lo && i < hi;
        const bool g = i < n && (!mid || (r > 0 && k > key)), e = mid && r > 0 && k == key;
        const uint64_t mg = __ballot(g), me = __ballot(e), under = (1ull << lane) - 1;
        if (lane == 0) {
            lds.wave[buf][wave][0] = __popcll(mg);
            lds.wave[buf][wave][1] = __popcll(me);
        }
        __syncthreads();             // also: the chunk's weights are read before any is overwritten in place
        int ng = sure + __popcll(mg & under), ne = equal + __popcll(me & under);
        for (int v = 0; v < kSel / 64; ++v) {
            const int cg = lds.wave[buf][v][0], ce = lds.wave[buf][v][1];
            ng += v < wave ? cg : 0;
            ne += v < wave ? ce : 0;
            sure += cg;
            equal += ce;
        }
        if (g || (e && ne < ties)) {
            const int at = ng + min(ne, ties);
            kept[at] = i;
            if (wd) wd[at] = x;
        }
    }
}

// Moves K (kind 0) or V (kind 1) of 32 dims of the kept tokens of one kv head to their new places, 256 tokens
// a turn.  In place one workgroup goes through all turns: tokens only move down and keep their order, so what a
// turn overwrites no later turn reads, and within a turn all loads end before the first store.
__global__ __launch_bounds__(256) void move_kernel(EvictArgs a, int in_place, int turns) {
    const tkm_attn_kv& s = a.src;
    const tkm_attn_kv& d = a.dst;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    long long item = blockIdx.x;
    const int turn0 = in_place ? 0 : (int)(item % turns);
    if (!in_place) item /= turns;
    const int slices = s.D / 32 * 2;
    const int slice = (int)(item % slices), db = slice / 2, kind = slice % 2;
    const long long row = item / slices;
    const int b = (int)(row / s.Hkv), h = (int)(row % s.Hkv);
    const int32_t* kept = a.kept + row * a.budget;
    if (row % s.Hkv == 0 && slice == 0 && turn0 == 0 && tid == 0) {
        const int n = s.len[b];
        d.len[b] = n != 0 && kept[0] < 0 ? -1 : min(n, a.budget);
    }
    const uint16_t* from = (const uint16_t*)(kind ? s.v : s.k);
    uint16_t* to = (uint16_t*)(kind ? d.v : d.k);
    // element offset of a token's block of 32 dims
    auto block_of = [&](const tkm_attn_kv& kv, int t) {
        const int page = kv.table[(long long)b * kv.max_pages + t / kv.page];
        return tile_at(kv, page, h, t % kv.page / 32) + db * 1024;
    };
    for (int turn = turn0; turn < (in_place ? turns : turn0 + 1); ++turn) {
        const int t0 = turn * 256;
        if (in_place) {
            const int t = t0 + tid;
            if (!__syncthreads_or(t < a.budget && kept[t] >= 0 && kept[t] != t)) continue;
        }
        if (kind == 0) {
            u32x4 x[4];
            const int c = tid % 4 * 8;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int t = t0 + i * 64 + tid / 4, o = t < a.budget ? kept[t] : -1;
                x[i] = o >= 0 ? ld_global16(from + block_of(s, o) + o % 32 * 32 + c) : u32x4{0u, 0u, 0u, 0u};
            }
            if (in_place) {
                __builtin_amdgcn_s_waitcnt(0);
                __syncthreads();
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int t = t0 + i * 64 + tid / 4;
                if (t < a.budget && kept[t] >= 0) *(u32x4*)(to + block_of(d, t) + t % 32 * 32 + c) = x[i];
            }
        } else {
            uint16_t x[4][8];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int t = t0 + i * 64 + lane, o = t < a.budget ? kept[t] : -1;
                const uint16_t* p = from + (o >= 0 ? block_of(s, o) + wave * 8 * 32 + o % 32 : 0);
#pragma unroll
                for (int j = 0; j < 8; ++j) x[i][j] = o >= 0 ? p[j * 32] : (uint16_t)0;
            }
            if (in_place) {
                __builtin_amdgcn_s_waitcnt(0);
                __syncthreads();
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int t = t0 + i * 64 + lane;
                if (t >= a.budget || kept[t] < 0) continue;
                uint16_t* p = to + block_of(d, t) + wave * 8 * 32 + t % 32;
#pragma unroll
                for (int j = 0; j < 8; ++j) p[j * 32] = x[i][j];
            }
        }
    }
}

int status() { return hipGetLastError() == hipSuccess ? 0 : -1; }

}  // namespace

int launch_append(const AppendArgs& a) {
    hipStream_t st = (hipStream_t)a.stream;
    note_kernels(kAppend);
    if (a.S == 1) {
        hipLaunchKernelGGL(append_one_kernel, dim3((unsigned)a.kv.B), dim3(256), 0, st, a);
        return status();
    }
    const int tiles = (a.S + 30) / 32 + 1;     // that S rows starting anywhere may touch
    hipLaunchKernelGGL(append_rows_kernel, dim3((unsigned)a.kv.B * a.kv.Hkv * tiles), dim3(256), 0, st, a, tiles);
    if (!a.start) hipLaunchKernelGGL(advance_kernel, dim3((unsigned)(a.kv.B + 255) / 256), dim3(256), 0, st, a);
    return status();
}

int launch_evict(const EvictArgs& a) {
    hipStream_t st = (hipStream_t)a.stream;
    note_kernels(kEvict);
    const int in_place = a.src.table == a.dst.table, turns = (a.budget + 255) / 256;
    const unsigned rows = (unsigned)a.src.B * a.src.Hkv;
    hipLaunchKernelGGL(select_kernel, dim3(rows), dim3(kSel), 0, st, a);
    hipLaunchKernelGGL(move_kernel, dim3(rows * (a.src.D / 32 * 2) * (in_place ? 1 : turns)), dim3(256), 0, st, a, in_place,
                       turns);
    return status();
}

}  // namespace tkm
