// attn_rope.hip -- rotary positions, and packed rows of Q, K and V into the paged cache (gfx950).
//
//   (x0, x1) -> factor (x0 cos a - x1 sin a, x0 sin a + x1 cos a),  a = pos * turns_i * 2^-64 of a circle
//
// An angle is the low 64 bits of pos * turns_i, of which the upper 32 are kept (two 32-bit products): off by 2^-33
// of a circle whatever the position is.  A row's rot/2 sines and cosines are formed once, in fp32, and shared by its
// heads through LDS; products and sums are fp32, rounded once on the way out.
//
// Both kernels move data and are bound by HBM, or by the launch where rows are few.
#include <hip/hip_runtime.h>

#include "attn_common.h"
#include "attn_kv.h"
#include "attn_launch.h"

namespace tkm {
namespace {

constexpr int kThreads = 256;

// N 16-bit values as one access of the memory pipe.
template <int N> struct Vec;
template <> struct Vec<8> { typedef u32x4 T; };
template <> struct Vec<4> { typedef u32x2 T; };
template <> struct Vec<2> { typedef uint32_t T; };
template <> struct Vec<1> { typedef uint16_t T; };
template <int N>
struct Part {
    uint16_t e[N];
    __device__ __forceinline__ void load(const uint16_t* p) {
        const typename Vec<N>::T v = *(const typename Vec<N>::T*)p;
        __builtin_memcpy(e, &v, 2 * N);
    }
    __device__ __forceinline__ void store(uint16_t* p) const {
        typename Vec<N>::T v;
        __builtin_memcpy(&v, e, 2 * N);
        *(typename Vec<N>::T*)p = v;
    }
};
template <int DT>
__device__ __forceinline__ uint16_t to_16(float x) { return (uint16_t)pack2<DT>(x, 0.f); }

// Cosine and sine of pair i at a position, times the factor.
__device__ __forceinline__ float2 turn(const tkm_attn_rope& rope, int i, int pos, float sign) {
    const uint64_t w = rope.turns[i];
    const uint32_t top = __umulhi((uint32_t)w, (uint32_t)pos) + (uint32_t)(w >> 32) * (uint32_t)pos;
    float s, c;
    sincospif((float)(int32_t)top * 0x1p-31f, &s, &c);      // half circles
    return float2{c * rope.factor, s * rope.factor * sign};
}

// A unit: V pairs of one head, as two parts of V values (HALVES: rot/2 apart) or as one of 2 V (PAIRS).
template <int DT, int LAYOUT, int V>
struct Unit {
    static constexpr int N = LAYOUT == TKM_ROPE_HALVES ? V : 2 * V;
    Part<N> x, y;
    __device__ __forceinline__ static int first(int u) { return u * N; }      // dim of x; y's is rot/2 behind it
    __device__ __forceinline__ void load(const uint16_t* p, int half) {
        x.load(p);
        if constexpr (LAYOUT == TKM_ROPE_HALVES) y.load(p + half);
    }
    __device__ __forceinline__ void rotate(const float2* cs) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
            uint16_t& e0 = LAYOUT == TKM_ROPE_HALVES ? x.e[j] : x.e[(2 * j) % N];
            uint16_t& e1 = LAYOUT == TKM_ROPE_HALVES ? y.e[j] : x.e[(2 * j + 1) % N];
            const float a = to_f32<DT>(e0), b = to_f32<DT>(e1);
            e0 = to_16<DT>(a * cs[j].x - b * cs[j].y);
            e1 = to_16<DT>(a * cs[j].y + b * cs[j].x);
        }
    }
};

// `T` threads have a row: their place in it, and the row's sines and cosines in LDS.
struct Row {
    int r, t, T, pos;
    const float2* cs;
};
__device__ __forceinline__ Row begin_row(float2 (*cs)[64], int T, int rows, const int32_t* pos, int S, const tkm_attn_rope& rope, float sign) {
    Row w;
    w.T = T;
    const int k = threadIdx.x / T;
    w.t = threadIdx.x % T;
    w.r = (int)blockIdx.x * (kThreads / T) + k;
    w.pos = w.r < rows ? (pos ? pos[w.r] : w.r % S) : -1;
    for (int i = w.t; i < rope.rot / 2; i += T) cs[k][i] = turn(rope, i, w.pos, sign);
    __syncthreads();
    w.cs = cs[k];
    return w;
}

// ---- rows to rows ---------------------------------------------------------------------------------

struct RopeK {
    tkm_attn_rope rope;
    const uint16_t* in;
    uint16_t* out;
    const int32_t* pos;
    long long in_stride, out_stride;
    int S, rows, heads, all, D, T;     // rotated heads, heads of a row
    float sign;
};

template <int DT, int LAYOUT, int V>
__global__ __launch_bounds__(kThreads) void rope_kernel(RopeK a) {
    __shared__ float2 cs[kThreads / 64][64];
    const Row w = begin_row(cs, a.T, a.rows, a.pos, a.S, a.rope, a.sign);
    if (w.pos < 0) return;
    const uint16_t* in = a.in + w.r * a.in_stride;
    uint16_t* out = a.out + w.r * a.out_stride;
    const int half = a.rope.rot / 2, units = half / V, lanes = w.T / units, u = w.t % units;
    typedef Unit<DT, LAYOUT, V> U;
    if (w.t < lanes * units)
        for (int h = w.t / units; h < a.heads; h += lanes) {
            const int at = h * a.D + U::first(u);
            U x;
            x.load(in + at, half);
            x.rotate(w.cs + u * V);
            x.x.store(out + at);
            if constexpr (LAYOUT == TKM_ROPE_HALVES) x.y.store(out + at + half);
        }
    if (in == out) return;
    // what is not rotated: the heads' other dims, and whole heads
    const int rest = a.D - a.rope.rot, from = a.heads * a.D;
    auto copy = [&](auto Nc) {
        constexpr int N = decltype(Nc)::value;
        const int each = rest / N, n = a.heads * each;
        for (int i = w.t; i < n; i += w.T) {
            const int at = i / each * a.D + a.rope.rot + i % each * N;
            Part<N> p;
            p.load(in + at);
            p.store(out + at);
        }
    };
    if (rest) {
        if (a.rope.rot % 8 == 0) copy(std::integral_constant<int, 8>{});
        else copy(std::integral_constant<int, 2>{});
    }
    for (int i = w.t * 8; i < (a.all - a.heads) * a.D; i += w.T * 8) {
        Part<8> p;
        p.load(in + from + i);
        p.store(out + from + i);
    }
}

// ---- rows to the cache ------------------------------------------------------------------------------

struct StoreK {
    tkm_attn_kv kv;
    tkm_attn_rope rope;        // rot 0: none
    const uint16_t* qkv;
    uint16_t* q;               // or NULL
    const int32_t *seq, *pos;
    const int64_t* slot;
    long long stride, q_stride;
    int rows, Hq, T, row_blocks;     // row_blocks: the blocks that have rows; those behind them have tiles of V
};

// Elements before the 32-token tile that holds a slot in its page's kv head.
__device__ __forceinline__ long long tile_of(const tkm_attn_kv& kv, int64_t slot, int h) {
    const int shift = __ffs(kv.page) - 1;
    return ((((slot >> shift) * kv.Hkv + h) << (shift - 5)) + ((slot & (kv.page - 1)) >> 5)) * (32 * kv.D);
}
__device__ __forceinline__ bool in_pool(const tkm_attn_kv& kv, int64_t slot) {
    return slot >= 0 && slot < (int64_t)kv.num_pages * kv.page;
}

// V of 32 rows of one kv head: through LDS, so that a wave's stores have neighbouring tokens.
__device__ __forceinline__ void store_v_tile(const StoreK& a, int tile, int h) {
    __shared__ __attribute__((aligned(16))) uint16_t vt[32][136];      // rows 272 bytes apart
    __shared__ int64_t slots[32];
    const tkm_attn_kv& kv = a.kv;
    const int r0 = tile * 32, chunks = kv.D / 8;
    if (threadIdx.x < 32) {
        const int r = r0 + threadIdx.x;
        const int64_t s = r < a.rows && a.pos[r] >= 0 ? a.slot[r] : -1;
        slots[threadIdx.x] = in_pool(kv, s) ? s : -1;
    }
    for (int i = threadIdx.x; i < 32 * chunks; i += kThreads) {
        const int t = i / chunks, c = i % chunks;
        if (r0 + t < a.rows)
            *(u32x4*)&vt[t][c * 8] = ld_global16(a.qkv + (r0 + t) * a.stride + (long long)(a.Hq + kv.Hkv + h) * kv.D + c * 8);
    }
    __syncthreads();
    const int t = threadIdx.x % 32;
    const int64_t s = slots[t];
    if (s < 0) return;
    uint16_t* v = (uint16_t*)kv.v + tile_of(kv, s, h) + s % 32;
    for (int d = threadIdx.x / 32; d < kv.D; d += kThreads / 32) v[d * 32] = vt[t][d];
}

template <int DT, int LAYOUT, int V>
__global__ __launch_bounds__(kThreads) void store_rows_kernel(StoreK a) {
    const tkm_attn_kv& kv = a.kv;
    if ((int)blockIdx.x >= a.row_blocks) {
        const int i = (int)blockIdx.x - a.row_blocks;
        store_v_tile(a, i / kv.Hkv, i % kv.Hkv);
        return;
    }
    __shared__ float2 cs[kThreads / 64][64];
    const Row w = begin_row(cs, a.T, a.rows, a.pos, 1, a.rope, 1.0f);
    if (w.pos < 0) return;
    const int64_t slot = a.slot[w.r];
    const bool kept = in_pool(kv, slot);
    const int tok = (int)(slot & 31), rot = a.rope.rot, D = kv.D;
    const uint16_t* in = a.qkv + w.r * a.stride;
    uint16_t* q = a.q ? a.q + w.r * a.q_stride : nullptr;
    // where dim d of head h (Q heads, then K heads) goes
    auto to = [&](int h, int d) {
        if (h < a.Hq) return q + h * D + d;
        return (uint16_t*)kv.k + tile_of(kv, slot, h - a.Hq) + (d >> 5) * 1024 + tok * 32 + (d & 31);
    };
    const int h0 = a.q ? 0 : a.Hq, h1 = a.Hq + (kept ? kv.Hkv : 0);
    if (rot) {
        const int half = rot / 2, units = half / V, lanes = w.T / units, u = w.t % units;
        typedef Unit<DT, LAYOUT, V> U;
        if (w.t < lanes * units)
            for (int h = h0 + w.t / units; h < h1; h += lanes) {
                U x;
                x.load(in + h * D + U::first(u), half);
                x.rotate(w.cs + u * V);
                x.x.store(to(h, U::first(u)));
                if constexpr (LAYOUT == TKM_ROPE_HALVES) x.y.store(to(h, U::first(u) + half));
            }
    }
    const int rest = D - rot, c0 = q == in ? a.Hq : h0;        // Q's other dims are in place already
    auto copy = [&](auto Nc) {
        constexpr int N = decltype(Nc)::value;
        const int each = rest / N;
        for (int i = w.t; i < (h1 - c0) * each; i += w.T) {
            const int h = c0 + i / each, d = rot + i % each * N;
            Part<N> p;
            p.load(in + h * D + d);
            p.store(to(h, d));
        }
    };
    if (rest) {
        if (rot % 8 == 0) copy(std::integral_constant<int, 8>{});
        else copy(std::integral_constant<int, 2>{});
    }
    if (!kept) return;
    if (a.T == kThreads) {             // few rows: V here too, its values to 64-byte rows of their own
        const int chunks = D / 8;
        for (int i = w.t; i < kv.Hkv * chunks; i += w.T) {
            const int h = i / chunks, c = i % chunks;
            const u32x4 x = ld_global16(in + (long long)(a.Hq + kv.Hkv + h) * D + c * 8);
            uint16_t* v = (uint16_t*)kv.v + tile_of(kv, slot, h) + c * 8 * 32 + tok;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                v[2 * j * 32] = (uint16_t)x[j];
                v[(2 * j + 1) * 32] = (uint16_t)(x[j] >> 16);
            }
        }
    }
    if (kv.weight) {
        const int b = a.seq[w.r], cap = kv.max_pages * kv.page;
        if ((unsigned)b < (unsigned)kv.B && w.pos < cap)
            for (int h = w.t; h < kv.Hkv; h += w.T) kv.weight[((long long)b * kv.Hkv + h) * cap + w.pos] = 0.f;
    }
}

// Rows up to which one has a whole workgroup.
constexpr int kFewRows = 1024;
int threads_a_row(int rows) { return rows <= kFewRows ? kThreads : 64; }
unsigned row_blocks(int rows) {
    const unsigned each = kThreads / threads_a_row(rows);
    return ((unsigned)rows + each - 1) / each;
}

// Pairs of a unit: as many as keep its parts aligned, of up to 16 bytes.
int unit_pairs(const tkm_attn_rope& r) {
    const int n = r.layout == TKM_ROPE_HALVES ? r.rot / 2 : r.rot;
    int v = n % 8 == 0 ? 8 : n % 4 == 0 ? 4 : n % 2 == 0 ? 2 : 1;
    return r.layout == TKM_ROPE_HALVES ? v : v / 2;
}

template <class A, class F>
void pick(int dtype, const tkm_attn_rope& r, const A& a, F launch) {
    const int v = unit_pairs(r);
    auto with = [&](auto DT) {
        auto go = [&](auto L, auto V) { launch(DT, L, V); };
        using H = std::integral_constant<int, TKM_ROPE_HALVES>;
        using Pr = std::integral_constant<int, TKM_ROPE_PAIRS>;
        if (r.layout == TKM_ROPE_HALVES) {
            if (v == 8) go(H{}, std::integral_constant<int, 8>{});
            else if (v == 4) go(H{}, std::integral_constant<int, 4>{});
            else if (v == 2) go(H{}, std::integral_constant<int, 2>{});
            else go(H{}, std::integral_constant<int, 1>{});
        } else {
            if (v == 4) go(Pr{}, std::integral_constant<int, 4>{});
            else if (v == 2) go(Pr{}, std::integral_constant<int, 2>{});
            else go(Pr{}, std::integral_constant<int, 1>{});
        }
    };
    if (dtype == TKM_ATTN_F16) with(std::integral_constant<int, DT_F16>{});
    else with(std::integral_constant<int, DT_BF16>{});
}

}  // namespace

bool rows_fit(const tkm_attn_kv* kv, int rows) {
    double blocks = row_blocks(rows);
    if (kv) blocks += (rows + 31.0) / 32.0 * kv->Hkv;
    return launch_fits(blocks, kThreads);
}

int launch_rope(const RopeArgs& a) {
    RopeK k{a.rope, (const uint16_t*)a.in, (uint16_t*)a.out, a.pos, a.in_stride, a.out_stride, a.S, a.rows, a.Hq + a.Hkv,
            a.Hq + 2 * a.Hkv, a.D, threads_a_row(a.rows), a.inverse ? -1.0f : 1.0f};
    note_kernels(kRope);
    pick(a.dtype, a.rope, k, [&](auto DT, auto L, auto V) {
        hipLaunchKernelGGL((rope_kernel<decltype(DT)::value, decltype(L)::value, decltype(V)::value>), dim3(row_blocks(a.rows)),
                           dim3(kThreads), 0, (hipStream_t)a.stream, k);
    });
    return hipGetLastError() == hipSuccess ? 0 : -1;
}

int launch_store(const StoreArgs& a) {
    StoreK k{a.kv, {}, (const uint16_t*)a.qkv, (uint16_t*)a.q, a.seq, a.pos, a.slot, a.stride, a.q_stride, a.rows, a.Hq,
             threads_a_row(a.rows), (int)row_blocks(a.rows)};
    if (a.rope) k.rope = *a.rope;
    else if (a.q == a.qkv) k.q = nullptr;       // Q stays as it is
    const int tiles = k.T == kThreads ? 0 : (a.rows + 31) / 32 * a.kv.Hkv;
    note_kernels(kAppend);
    pick(a.kv.dtype, k.rope, k, [&](auto DT, auto L, auto V) {
        hipLaunchKernelGGL((store_rows_kernel<decltype(DT)::value, decltype(L)::value, decltype(V)::value>), dim3(k.row_blocks + tiles),
                           dim3(kThreads), 0, (hipStream_t)a.stream, k);
    });
    return hipGetLastError() == hipSuccess ? 0 : -1;
}

}  // namespace tkm
