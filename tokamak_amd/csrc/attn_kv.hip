// attn_kv.hip -- the paged key-value cache's own kernels (gfx950): rows of packed QKV into it, and eviction
// from it by accumulated attention weight.  The layout is in attn_kv.h.
//
// All of these move data and are bound by HBM, or by the launch where there is little to move.  us on one card: a
// row to each of 64 sequences, 8 kv heads of D 128: 3.3; up to 1531 rows to each of 6, 4 kv heads of D 64 (14 MB both
// ways): 5.7, and 1.5 to advance the lengths where they are the start; eviction: see the kernels.
#include <hip/hip_runtime.h>
#include <limits.h>

#include "attn_common.h"
#include "attn_kv.h"
#include "attn_launch.h"

namespace tkm {
namespace {

// Pages are powers of two, from 32 tokens on.
__device__ __forceinline__ int page_shift(const tkm_attn_kv& kv) { return __ffs(kv.page) - 1; }
// Elements before the 32-token tile that holds position t in a page's kv head.
__device__ __forceinline__ long long tile_at(const tkm_attn_kv& kv, int page, int h, int t) {
    return ((((long long)page * kv.Hkv + h) << (page_shift(kv) - 5)) + ((t & (kv.page - 1)) >> 5)) * (32 * kv.D);
}
__device__ __forceinline__ int page_of(const tkm_attn_kv& kv, int b, int t) { return kv.table[(long long)b * kv.max_pages + (t >> page_shift(kv))]; }
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
        const int page = page_of(kv, b, pos), t = pos % 32, chunks = kv.D / 8;
        if (in_pool(kv, page)) {
            const uint16_t* row = (const uint16_t*)a.qkv + ((long long)b * (a.Hq + 2 * kv.Hkv) + a.Hq) * kv.D;
            for (int i = threadIdx.x; i < 2 * kv.Hkv * chunks; i += 256) {
                const u32x4 x = ld_global16(row + i * 8);
                const int h = i / chunks % kv.Hkv, c = i % chunks;
                const long long at = tile_at(kv, page, h, pos) + c / 4 * 1024;
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
    const int page = page_of(kv, b, t0);
    if (!in_pool(kv, page)) return;
    const long long at = tile_at(kv, page, h, t0);
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

// A weight as an integer of the same order, at most that of +inf; NaN below all others, -0 as +0.
__device__ __forceinline__ uint32_t key_of(float w) {
    const uint32_t u = __float_as_uint(w + 0.0f);
    const uint32_t k = u ^ ((uint32_t)((int)u >> 31) | 0x80000000u);
    return w != w ? 0u : k;
}
// Keys that no weight has: of a position that stays without a choice, of one behind the sequence, and none's.
constexpr uint32_t kStays = 0xffffffffu, kGone = 0xfffffffeu, kNoKey = 0xfffffffdu;

__device__ __forceinline__ uint32_t rank_in(uint64_t mask, uint32_t from) {     // from + lanes of the mask below this one
    return __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, from));
}

// A selecting workgroup of T threads has EACH weights a thread at a time.
template <int T, int EACH>
struct Sel {
    static constexpr int WAVES = T / 64, CHUNK = T * EACH;
    static constexpr int BITS[3] = {T == 256 ? 11 : 12, T == 256 ? 11 : 10, 10};   // of a weight's key, from the top
    static constexpr int PER = (1 << BITS[0]) / T;                                  // bins a thread has
    uint32_t bins[1 << BITS[0]];
    uint32_t tot[2][WAVES];
    uint32_t flags[2][EACH][WAVES];
    uint32_t bin, before, many;
};

// Chooses what one kv head of one sequence of n > budget tokens keeps: writes its old positions in ascending order
// to `kept`, and their weights w to their new places wd.
//
// The border among the weights is found by three histograms of their keys' bits (12, 10, 10, or 11, 11, 10; each
// narrows to the bin that holds the border, and the walk ends with a bin of which all are kept), of weights that
// stay in registers where T * EACH hold them all.  Then ballots number what stays, T * EACH positions a barrier.
// Bound by the chain of barriers and dependent loads where sequences are short (6 to 8 us for 16 heads of 1180
// tokens, 12 for 128 of 6144), and by one workgroup's issue where they are long: 87 us for 2 heads of 110000.
template <int T, int EACH>
__device__ __forceinline__ void select_row(Sel<T, EACH>& lds, const EvictArgs& a, int n, const float* w, float* wd, int32_t* kept) {
    using S = Sel<T, EACH>;
    constexpr int PER = S::PER;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const bool holds = n <= S::CHUNK;
    const int lo = a.sink, hi = n - a.recent, r = a.budget - a.sink - a.recent;
    float x[EACH], y[EACH];      // a chunk's weights, and the next one's under way
    uint32_t key[EACH];
    // f(e) for the positions c + e * T + tid of a chunk, e < EACH; straight code where the chunk is full, as most
    // chunks of long sequences are
    auto each = [&](int c, auto f) {
        if (c + S::CHUNK <= n) {
#pragma unroll
            for (int e = 0; e < EACH; ++e) f(e);
        } else {
#pragma unroll
            for (int e = 0; e < EACH; ++e) {
                if (c + e * T >= n) break;
                f(e);
            }
        }
    };
    auto fetch = [&](int c) {
        if (c + S::CHUNK <= n) {
#pragma unroll
            for (int e = 0; e < EACH; ++e) y[e] = (w + c + e * T)[(unsigned)tid];
        } else {
#pragma unroll
            for (int e = 0; e < EACH; ++e) {
                y[e] = 0.f;
                if (c + e * T + tid < n) y[e] = (w + c + e * T)[(unsigned)tid];
            }
        }
    };
    auto take = [&](int c) {     // the chunk that was fetched last, and its keys; fetches the next, or the first again
#pragma unroll
        for (int e = 0; e < EACH; ++e) x[e] = y[e];
        if (!holds) fetch(c + S::CHUNK < n ? c + S::CHUNK : 0);
        if (c >= lo && c + S::CHUNK <= hi) {
#pragma unroll
            for (int e = 0; e < EACH; ++e) key[e] = key_of(x[e]);
        } else {
#pragma unroll
            for (int e = 0; e < EACH; ++e) {
                const int i = c + e * T + tid;
                key[e] = i >= lo && i < hi ? key_of(x[e]) : i < n ? kStays : kGone;
            }
        }
    };
    fetch(0);
    if (holds) take(0);
    // Positions with a key >= sure stay, but for kGone, and the first `ties` of those with the key `tie`.
    uint32_t sure = kStays, tie = kNoKey;
    int ties = 0, flip = 0;
    if (r > 0) {
        uint32_t prefix = 0, before = 0;
        int low = 32;
        for (int level = 0; level < 3; ++level) {
            const int bits = S::BITS[level], bins = 1 << bits;
            low -= bits;
            if (tid * PER < bins)
#pragma unroll
                for (int i = 0; i < PER; i += 4) *(uint4*)&lds.bins[tid * PER + i] = make_uint4(0, 0, 0, 0);
            __syncthreads();
            const uint32_t base = level ? prefix << (low + bits) : 0u, span = level ? 1u << (low + bits) : kGone;
            for (int c = 0; c < n; c += S::CHUNK) {
                if (!holds) take(c);
                each(c, [&](int e) {
                    const uint32_t k = key[e] - base;
                    if (k < span) atomicAdd(&lds.bins[k >> low], 1u);
                });
            }
            __syncthreads();
            // the bin, from the largest on, at which the running count reaches r
            uint32_t v[PER] = {}, sum = 0;           // bins first .. first + PER - 1
            const int first = bins - PER - tid * PER;
            if (first >= 0) __builtin_memcpy(v, __builtin_assume_aligned(&lds.bins[first], 16), sizeof v);
#pragma unroll
            for (int i = 0; i < PER; ++i) sum += v[i];
            const uint32_t run = wave_scan(sum);
            if (lane == 63) lds.tot[flip][wave] = run;
            __syncthreads();
            const uint32_t all = wave_scan(lane < S::WAVES ? lds.tot[flip][lane] : 0u);
            flip ^= 1;
            uint32_t at = before + run - sum + (wave ? (uint32_t)lane_value((int)all, wave - 1) : 0u);
            if (at < (uint32_t)r && at + sum >= (uint32_t)r) {
                int bin = first + PER - 1;
#pragma unroll
                for (int i = PER - 1; i > 0; --i)
                    if (bin == first + i && at + v[i] < (uint32_t)r) {
                        at += v[i];
                        --bin;
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
                    tie = sure++;
                    ties = r - (int)before;
                }
                break;
            }
            __syncthreads();
        }
    }
    uint32_t* wo = wd ? (uint32_t*)wd : (uint32_t*)kept;     // (written before kept's own value)
    uint32_t stay = 0, equal = 0;    // before this chunk
    for (int c = 0, buf = 0; c < n; c += S::CHUNK, buf ^= 1) {
        if (!holds) take(c);
        auto stays = [&](int e) { return __ballot(key[e] >= sure) & __ballot(key[e] != kGone); };
        uint32_t count = 0;          // of the positions of lane e in this wave: those that stay, and << 16 those at the border
        each(c, [&](int e) {
            const int of = __popcll(stays(e)) | __popcll(__ballot(key[e] == tie)) << 16;
            count = lane == e ? (uint32_t)of : count;
        });
        if (lane < EACH) lds.flags[buf][lane][wave] = count;
        __syncthreads();     // also: all of the chunk's weights are here before one is overwritten in place
        uint32_t sum = 0, mine = 0;  // of the positions of lane e: all waves', and those of the waves before this one
        if (lane < EACH)
#pragma unroll
            for (int v = 0; v < S::WAVES; ++v) {
                const uint32_t f = lds.flags[buf][lane][v];
                sum += f;
                mine += v < wave ? f : 0;
            }
        const uint32_t run = wave_scan(sum), before = run - sum + mine;
        const uint32_t at_border = equal + (before >> 16), at = stay + (before & 0xffffu) + min(at_border, (uint32_t)ties);
        each(c, [&](int e) {
            bool in = key[e] >= sure && key[e] != kGone;
            const uint64_t g = stays(e), t = __ballot(key[e] == tie);
            uint32_t to = rank_in(g, (uint32_t)lane_value((int)at, e));
            if (t) {
                const uint32_t b0 = (uint32_t)lane_value((int)at_border, e), b = rank_in(t, b0);
                to += min(b, (uint32_t)ties) - min(b0, (uint32_t)ties);
                in |= key[e] == tie && b < (uint32_t)ties;
            }
            if (in) {
                wo[to] = __float_as_uint(x[e]);
                kept[to] = c + e * T + tid;
            }
        });
        const uint32_t last = (uint32_t)lane_value((int)run, 63);
        stay += last & 0xffffu;
        equal += last >> 16;
    }
}

// One kv head of one sequence a workgroup.  A sequence with a length or a page that its tables cannot have gets -1s.
template <int T>
__global__ __launch_bounds__(T) void select_kernel(EvictArgs a) {
    constexpr int LONG = T == 256 ? 8 : 16;
    __shared__ union {
        Sel<T, 8> few;
        Sel<T, LONG> many;
    } lds;
    const tkm_attn_kv& s = a.src;
    const tkm_attn_kv& d = a.dst;
    const int tid = threadIdx.x;
    const long long row = blockIdx.x;
    const int b = (int)(row / s.Hkv);
    const long long cap = (long long)s.max_pages * s.page, cap_d = (long long)d.max_pages * d.page;
    const int n = s.len[b];
    int32_t* kept = a.kept + row * a.budget;
    const float* w = s.weight + row * cap;
    float* wd = d.weight ? d.weight + row * cap_d : nullptr;
    int bad = n < 0 || n > cap;
    if (!bad) {
        const int most = min(n, a.budget);
        for (int i = tid; i < (n + s.page - 1) / s.page; i += T) bad |= !in_pool(s, s.table[(long long)b * s.max_pages + i]);
        for (int i = tid; i < (most + d.page - 1) / d.page; i += T) bad |= !in_pool(d, d.table[(long long)b * d.max_pages + i]);
    }
    if (__syncthreads_or(bad)) {
        for (int i = tid; i < a.budget; i += T) kept[i] = -1;
        return;
    }
    if (n <= a.budget) {
        for (int i = tid; i < a.budget; i += T) {
            kept[i] = i < n ? i : -1;
            if (wd && wd != w && i < n) wd[i] = w[i];
        }
        return;
    }
    if (T == 256 || n <= T * 8) select_row<T, 8>(lds.few, a, n, w, wd, kept);
    else select_row<T, LONG>(lds.many, a, n, w, wd, kept);
}

// Moves K and V of the kept tokens of one kv head to their new places, 256 tokens a turn and 32 dims at a time, the
// next 32 on their way while these are stored.  In place one workgroup goes through all turns of its dims: tokens
// only move down and keep their order, so what a turn overwrites no later turn reads, and within a turn all loads
// of a block of dims end before its first store.
// Bound by HBM: K's kept tokens are single 64-byte rows, V's lie in 64-byte rows of 32 tokens, kept or not, so
// nearly all of the source is read: 376 MB for 16 x 8 heads of 4096 kept of 6144 tokens (268 are the kept ones
// alone), 268 written, in 149 us: 4.3 TB/s, where a plain copy reaches 5.2.  In place it is bound by the turns' chain of
// position, page, load, wait and store, 3.6 to 3.9 us each where heads are few: 251 us for 16384 tokens of 8 heads (49 into
// another table), 854 for 60000 of 2 heads (41), 222 for the 16 x 8 heads of 4096 above.
template <bool K, bool V>
__device__ __forceinline__ void move_tokens(const EvictArgs& a, int in_place, int turns, int turn0, long long row, int db0, int blocks) {
    const tkm_attn_kv& s = a.src;
    const tkm_attn_kv& d = a.dst;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int b = (int)(row / s.Hkv), h = (int)(row % s.Hkv);
    const int32_t* kept = a.kept + row * a.budget;
    // element offset of a token's blocks of 32 dims, -1 for none
    auto block_of = [&](const tkm_attn_kv& kv, int t) {
        return t < 0 ? -1ll : tile_at(kv, page_of(kv, b, t), h, t);
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

// Tiles that S rows starting anywhere may touch.
static int append_tiles(int S) { return S / 32 + (S % 32 > 1 ? 2 : 1); }

bool append_fits(const tkm_attn_kv& kv, int S) {
    return launch_fits(S == 1 ? (double)kv.B : (double)kv.B * kv.Hkv * append_tiles(S), 256);
}

int launch_append(const AppendArgs& a) {
    hipStream_t st = (hipStream_t)a.stream;
    note_kernels(kAppend);
    if (a.S == 1) {
        hipLaunchKernelGGL(append_one_kernel, dim3((unsigned)a.kv.B), dim3(256), 0, st, a);
        return status();
    }
    const int tiles = append_tiles(a.S);
    hipLaunchKernelGGL(append_rows_kernel, dim3((unsigned)a.kv.B * a.kv.Hkv * tiles), dim3(256), 0, st, a, tiles);
    if (status()) return -1;
    if (a.start) return 0;
    hipLaunchKernelGGL(advance_kernel, dim3((unsigned)(a.kv.B + 255) / 256), dim3(256), 0, st, a);
    return status();
}

// The choosing kernel's threads: small workgroups where they hold a row, for more rows at a time and cheaper barriers
// (1152 heads of 1226 tokens 12 us, against 41 with 1024 threads; 16 heads of 1180 8, against 11).
static int select_threads(const tkm_attn_kv& src) { return (long long)src.max_pages * src.page <= 2048 ? 256 : 1024; }

// The moving kernel's launch.  In place, and where there are few (head, turn) pairs, a workgroup has 32 dims of K or V
// of a head; where there are more, half of K's or V's dims; else all of both.  us of all / halves / 32 dims: 64 pairs
// of D 64 10.8 / 5.9 / 5.9, 176 of D 128 8.9 / 7.0 / 9.1, 320 of D 128 26 / 22 / 25, 480 of D 128 37 / 47 / 51, 1456 of
// D 64 57 / 75 / 75, 2048 of D 128 149 / 172 / 215.
struct MoveGrid {
    int in_place, turns, parts, apart;
    double groups;
};
static MoveGrid move_grid(const tkm_attn_kv& src, const tkm_attn_kv& dst, int budget) {
    MoveGrid g;
    g.in_place = src.table == dst.table;
    g.turns = (budget + 255) / 256;
    const double rows = (double)src.B * src.Hkv, pairs = rows * g.turns;
    const bool few = g.in_place || pairs < 128, some = pairs < 400;
    g.parts = few ? src.D / 32 : some ? 2 : 1;
    g.apart = few || some;
    g.groups = rows * g.parts * (g.apart ? 2 : 1) * (g.in_place ? 1 : g.turns);
    return g;
}

bool evict_fits(const tkm_attn_kv& src, const tkm_attn_kv& dst, int budget) {
    return launch_fits((double)src.B * src.Hkv, select_threads(src)) && launch_fits(move_grid(src, dst, budget).groups, 256);
}

int launch_evict(const EvictArgs& a) {
    hipStream_t st = (hipStream_t)a.stream;
    note_kernels(kEvict);
    const unsigned rows = (unsigned)a.src.B * a.src.Hkv;
    if (select_threads(a.src) == 256) hipLaunchKernelGGL(select_kernel<256>, dim3(rows), dim3(256), 0, st, a);
    else hipLaunchKernelGGL(select_kernel<1024>, dim3(rows), dim3(1024), 0, st, a);
    if (status()) return -1;      // move_kernel goes by what the choosing kernel wrote
    const MoveGrid g = move_grid(a.src, a.dst, a.budget);
    hipLaunchKernelGGL(move_kernel, dim3((unsigned)g.groups), dim3(256), 0, st, a, g.in_place, g.turns, g.parts, g.apart);
    return status();
}

}  // namespace tkm
