// attn_kv.hip -- the paged key-value cache's own kernels (gfx950): rows of packed QKV into it, and eviction
// from it by accumulated attention weight.  The layout is in attn_kv.h.
//
// All of these move data and are bound by HBM, or by the launch where there is little to move.  us on one card: a
// row to each of 64 sequences, 8 kv heads of D 128: 3.3; up to 1531 rows to each of 6, 4 kv heads of D 64 (14 MB both
// ways): 5.8; eviction: see the kernels.
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

constexpr int kSel = 1024, kSelWaves = kSel / 64;   // threads and waves of a selecting workgroup
constexpr int kEach = 8, kChunk = kSel * kEach;      // weights a thread has at a time, and the workgroup
constexpr int kSelBits[3] = {12, 10, 10};            // of a weight's key, from the top

struct SelectLds {
    uint32_t bins[1 << kSelBits[0]];
    uint32_t tot[2][kSelWaves];
    uint32_t flags[2][kEach * kSelWaves];
    uint32_t bin, before, many;
};

// Chooses what one kv head of one sequence keeps: writes its old positions in ascending order to `kept`, and
// their weights to their new places.  A sequence with a length or a page that its tables cannot have gets -1s.
//
// The border among the weights is found by three histograms of their keys' bits (12, 10, 10; each narrows to the
// bin that holds the border, and the walk ends with a bin of which all are kept), of weights that stay in registers
// where 8192 hold them all.  Then ballots number what stays: 8192 positions a barrier.  Bound by the chain of
// barriers: as 16 rounds of counting three candidates, and 1024 positions a barrier, it took 19 us for 1180
// tokens and 30 for 8192.
__global__ __launch_bounds__(kSel) void select_kernel(EvictArgs a) {
    __shared__ SelectLds lds;
    const tkm_attn_kv& s = a.src;
    const tkm_attn_kv& d = a.dst;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const long long row = blockIdx.x;
    const int b = (int)(row / s.Hkv);
    const long long cap = (long long)s.max_pages * s.page, cap_d = (long long)d.max_pages * d.page;
    const int n = s.len[b];
    int32_t* kept = a.kept + row * a.budget;
    const float* w = s.weight + row * cap;
    float* wd = d.weight ? d.weight + row * cap_d : nullptr;
    int bad = n < 0 || n > cap;
    float held[kEach];
    const bool holds = n <= kChunk;
    if (!bad) {
        const int most = min(n, a.budget);
#pragma unroll
        for (int e = 0; e < kEach; ++e) held[e] = e * kSel + tid < n ? w[e * kSel + tid] : 0.f;
        for (int i = tid; i < (n + s.page - 1) / s.page; i += kSel) bad |= !in_pool(s, s.table[(long long)b * s.max_pages + i]);
        for (int i = tid; i < (most + d.page - 1) / d.page; i += kSel) bad |= !in_pool(d, d.table[(long long)b * d.max_pages + i]);
    }
    if (__syncthreads_or(bad)) {
        for (int i = tid; i < a.budget; i += kSel) kept[i] = -1;
        return;
    }
    if (n <= a.budget) {
        for (int i = tid; i < a.budget; i += kSel) {
            kept[i] = i < n ? i : -1;
            if (wd && wd != w && i < n) wd[i] = w[i];
        }
        return;
    }
    const int lo = a.sink, hi = n - a.recent, r = a.budget - a.sink - a.recent;
    auto load = [&](int c, float (&x)[kEach]) {      // the weights of positions c + e * kSel + tid
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
            const int i = c + e * kSel + tid;
            x[e] = holds ? held[e] : i < n ? w[i] : 0.f;
        }
    };
    // Of the positions in [lo, hi) those with a key >= sure stay, and the first `ties` of those with the key `tie`.
    uint32_t sure = 0xffffffffu, tie = 0xffffffffu;
    int ties = 0, flip = 0;
    if (r > 0) {
        uint32_t prefix = 0, before = 0;
        int low = 32;
        for (int level = 0; level < 3; ++level) {
            const int bits = kSelBits[level], bins = 1 << bits;
            low -= bits;
            if (tid * 4 < bins) *(uint4*)&lds.bins[tid * 4] = make_uint4(0, 0, 0, 0);
            __syncthreads();
            for (int c = 0; c < n; c += kChunk) {
                float x[kEach];
                load(c, x);
#pragma unroll
                for (int e = 0; e < kEach; ++e) {
                    const int i = c + e * kSel + tid;
                    const uint32_t k = key_of(x[e]);
                    if (i >= lo && i < hi && (uint32_t)((uint64_t)k >> (low + bits)) == prefix)
                        atomicAdd(&lds.bins[k >> low & (uint32_t)(bins - 1)], 1u);
                }
            }
            __syncthreads();
            // the bin, from the largest on, at which the running count reaches r
            uint4 v = make_uint4(0, 0, 0, 0);        // bins first .. first + 3
            const int first = bins - 4 - tid * 4;
            if (first >= 0) v = *(const uint4*)&lds.bins[first];
            const uint32_t sum = v.x + v.y + v.z + v.w, run = wave_scan(sum);
            if (lane == 63) lds.tot[flip][wave] = run;
            __syncthreads();
            const uint32_t all = wave_scan(lane < kSelWaves ? lds.tot[flip][lane] : 0u);
            flip ^= 1;
            uint32_t at = before + run - sum + (wave ? (uint32_t)lane_value((int)all, wave - 1) : 0u);
            if (at < (uint32_t)r && at + sum >= (uint32_t)r) {
                int bin = first + 3;
                if (at + v.w < (uint32_t)r) {
                    at += v.w;
                    --bin;
                    if (at + v.z < (uint32_t)r) {
                        at += v.z;
                        --bin;
                        if (at + v.y < (uint32_t)r) {
                            at += v.y;
                            --bin;
                        }
                    }
                }
                lds.bin = (uint32_t)bin;
                lds.before = at;
                lds.many = lds.bins[bin];
            }
            __syncthreads();
            before = lds.before;
            prefix = prefix << bits | lds.bin;
            if (before + lds.many == (uint32_t)r || level == 2) {
                sure = prefix << low;
                if (before + lds.many != (uint32_t)r) {
                    tie = sure++;                    // keys end below 0xffffffff
                    ties = r - (int)before;
                }
                break;
            }
            __syncthreads();
        }
    }
    uint32_t stay = 0, equal = 0;    // before this chunk
    const uint64_t under = (1ull << lane) - 1;
    for (int c = 0, buf = 0; c < n; c += kChunk, buf ^= 1) {
        float x[kEach];
        uint64_t g[kEach], t[kEach];
        load(c, x);
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
            const int i = c + e * kSel + tid;
            const uint32_t k = key_of(x[e]);
            const bool mid = i >= lo && i < hi;
            g[e] = __ballot(i < n && (!mid || k >= sure));
            t[e] = __ballot(mid && ties > 0 && k == tie);
            if (lane == 0) lds.flags[buf][e * kSelWaves + wave] = (uint32_t)(__popcll(g[e]) | __popcll(t[e]) << 16);
        }
        __builtin_amdgcn_s_waitcnt(0);
        __syncthreads();             // also: all of the chunk's weights are read before one is overwritten in place
        const uint32_t v0 = lds.flags[buf][lane * 2], v1 = lds.flags[buf][lane * 2 + 1], run = wave_scan(v0 + v1);
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
            const int at = e * kSelWaves + wave;
            const uint32_t before = (uint32_t)(lane_value((int)(run - v0 - v1), at / 2) + (at % 2 ? lane_value((int)v0, at / 2) : 0));
            const uint32_t ng = stay + (before & 0xffffu) + (uint32_t)__popcll(g[e] & under);
            const uint32_t nt = equal + (before >> 16) + (uint32_t)__popcll(t[e] & under);
            if ((g[e] >> lane & 1) || ((t[e] >> lane & 1) && nt < (uint32_t)ties)) {
                const uint32_t to = ng + min(nt, (uint32_t)ties);
                kept[to] = c + e * kSel + tid;
                if (wd) wd[to] = x[e];
            }
        }
        const uint32_t last = (uint32_t)lane_value((int)run, 63);
        stay += last & 0xffffu;
        equal += last >> 16;
    }
}

// Moves K and V of the kept tokens of one kv head to their new places, 256 tokens a turn and 32 dims at a time, the
// next 32 on their way while these are stored.  In place one workgroup goes through all turns of its dims: tokens
// only move down and keep their order, so what a turn overwrites no later turn reads, and within a turn all loads
// of a block of dims end before its first store.
// Bound by HBM: K's kept tokens are single 64-byte rows, V's lie in 64-byte rows of 32 tokens, kept or not, so
// nearly all of the source is read: 376 MB for 16 x 8 heads of 4096 kept of 6144 tokens (268 are the kept ones
// alone), 268 written, in 149 us: 4.3 TB/s, where a plain copy reaches 5.2.
template <bool K, bool V>
__device__ __forceinline__ void move_tokens(const EvictArgs& a, int in_place, int turns, int turn0, long long row, int db0, int blocks) {
    const tkm_attn_kv& s = a.src;
    const tkm_attn_kv& d = a.dst;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int b = (int)(row / s.Hkv), h = (int)(row % s.Hkv);
    const int32_t* kept = a.kept + row * a.budget;
    // element offset of a token's blocks of 32 dims, -1 for none
    auto block_of = [&](const tkm_attn_kv& kv, int t) {
        return t < 0 ? -1ll : tile_at(kv, kv.table[(long long)b * kv.max_pages + t / kv.page], h, t % kv.page / 32);
    };
    const uint16_t* vs = (const uint16_t*)s.v;
    const uint16_t* ks = (const uint16_t*)s.k;
    uint16_t* vd = (uint16_t*)d.v;
    uint16_t* kd = (uint16_t*)d.k;
    for (int turn = turn0; turn < (in_place ? turns : turn0 + 1); ++turn) {
        const int t0 = turn * 256;
        if (in_place) {
            const int t = t0 + tid;
            if (!__syncthreads_or(t < a.budget && kept[t] >= 0 && kept[t] != t)) continue;
        }
        // K: 4 threads a token, 16 bytes each; V: a lane a token, a wave 8 of the 32 dims
        long long kf[4], kt[4], vf[4], vt[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            int t = t0 + i * 64 + tid / 4, o = t < a.budget ? kept[t] : -1;
            kf[i] = block_of(s, o) + (o & 31) * 32 + tid % 4 * 8;
            kt[i] = block_of(d, o < 0 ? -1 : t) + (t & 31) * 32 + tid % 4 * 8;
            if (o < 0) kf[i] = -1;
            t = t0 + i * 64 + lane;
            o = t < a.budget ? kept[t] : -1;
            vf[i] = block_of(s, o) + wave * 8 * 32 + (o & 31);
            vt[i] = block_of(d, o < 0 ? -1 : t) + wave * 8 * 32 + (t & 31);
            if (o < 0) vf[i] = -1;
        }
        u32x4 kx[2][4];
        uint16_t vx[2][4][8];
        auto load = [&](int buf, int db) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (K && kf[i] >= 0) kx[buf][i] = ld_global16(ks + kf[i] + db * 1024);
                if (V && vf[i] >= 0)
#pragma unroll
                    for (int j = 0; j < 8; ++j) vx[buf][i][j] = vs[vf[i] + db * 1024 + j * 32];
            }
        };
        auto store = [&](int buf, int db) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (K && kf[i] >= 0) *(u32x4*)(kd + kt[i] + db * 1024) = kx[buf][i];
                if (V && vf[i] >= 0)
#pragma unroll
                    for (int j = 0; j < 8; ++j) vd[vt[i] + db * 1024 + j * 32] = vx[buf][i][j];
            }
        };
        load(0, db0);
        for (int i = 0; i < blocks; i += 2) {
            if (in_place) {
                __builtin_amdgcn_s_waitcnt(0);
                __syncthreads();
            }
            if (i + 1 < blocks) load(1, db0 + i + 1);
            store(0, db0 + i);
            if (i + 1 >= blocks) break;
            if (in_place) {
                __builtin_amdgcn_s_waitcnt(0);
                __syncthreads();
            }
            if (i + 2 < blocks) load(0, db0 + i + 2);
            store(1, db0 + i + 1);
        }
    }
}

// `parts` workgroups share a head's dims; with `apart` K and V have workgroups of their own.
__global__ __launch_bounds__(256) void move_kernel(EvictArgs a, int in_place, int turns, int parts, int apart) {
    long long item = blockIdx.x;
    const int kind = apart ? (int)(item & 1) : 2;
    if (apart) item >>= 1;
    const int part = (int)(item % parts);
    item /= parts;
    const int turn0 = in_place ? 0 : (int)(item % turns);
    const long long row = in_place ? item : item / turns;
    const int blocks = a.src.D / 32 / parts;
    if (row % a.src.Hkv == 0 && part == 0 && turn0 == 0 && kind != 1 && threadIdx.x == 0) {
        const int b = (int)(row / a.src.Hkv), n = a.src.len[b];
        a.dst.len[b] = n != 0 && a.kept[row * a.budget] < 0 ? -1 : min(n, a.budget);
    }
    if (kind == 0) move_tokens<true, false>(a, in_place, turns, turn0, row, part * blocks, blocks);
    else if (kind == 1) move_tokens<false, true>(a, in_place, turns, turn0, row, part * blocks, blocks);
    else move_tokens<true, true>(a, in_place, turns, turn0, row, part * blocks, blocks);
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
    // In place, and where there are few (head, turn) pairs, a workgroup has 32 dims of K or V of a head (64 pairs of
    // D 64: 6.3 us, against 10.8 of one workgroup for all), else all of both (2048 pairs of D 128: 149 us, against
    // 172 of one for K and one for V, and 215 of the finest).
    const bool few = in_place || (long long)rows * turns < 1024;
    const int parts = few ? a.src.D / 32 : 1, apart = few;
    hipLaunchKernelGGL(move_kernel, dim3(rows * parts * (apart ? 2 : 1) * (in_place ? 1 : turns)), dim3(256), 0, st, a, in_place, turns,
                       parts, apart);
    return status();
}

}  // namespace tkm
