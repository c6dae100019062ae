// attn_rope.hip -- rotary positions, and packed rows of Q, K and V into the paged cache (gfx950).
//
//   (x0, x1) -> factor (x0 cos a - x1 sin a, x0 sin a + x1 cos a),  a = pos * turns_i * 2^-64 of a circle
//
// An angle is the low 64 bits of pos * turns_i, of which the upper 32 are kept (two 32-bit products) and rounded to fp32:
// cut by less than 2^-32 of a circle and rounded by 2^-26 at most, whatever the position is.  A row's rot/2 sines and
// cosines are formed once, in fp32, and shared by its heads through LDS; products and sums are fp32, rounded once on the
// way out.
//
// Both kernels move data and are bound by HBM, or by the launch where rows are few.  A thread has a chunk of 8 dims, 16
// bytes, of one head at a time, and forms its side of the pairs; a head's chunks are one wave's, at one time, which
// reads the other sides before it writes, so that rows may be rotated in place.  (With a pair's sides in one thread, stores
// were as wide as the largest power of two in rot / 2: 16384 rows of 40 heads of 64 with 40 dims rotated took 41 us for
// 27.)  A training batch of 8192 rows of 48 heads of 128: 45 us of operands from HBM, 4.4 TB/s; 15011 prompt rows of 28 heads
// of 128 into the cache: 51.5 us, 4.2 TB/s.
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
struct Chunk {
    uint16_t e[8];
    template <int N>
    __device__ __forceinline__ void load(int i, const uint16_t* p) {
        const typename Vec<N>::T v = *(const typename Vec<N>::T*)p;
        __builtin_memcpy(e + i, &v, 2 * N);
    }
    __device__ __forceinline__ void store(uint16_t* p) const {
        u32x4 v;
        __builtin_memcpy(&v, e, 16);
        *(u32x4*)p = v;
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

// Dims d .. d + 7 of a rotated head at p.  HALVES: pairs (i, i + rot / 2), whose other sides come V at a time, the
// largest power of two that divides rot / 2 (of up to 8), so that all V have the same place in their pairs.
template <int DT, int LAYOUT, int V>
__device__ __forceinline__ Chunk rotated(const uint16_t* p, int d, int rot, const float2* cs) {
    Chunk x, y;
    x.load<8>(0, p + d);
    if constexpr (LAYOUT == TKM_ROPE_HALVES) {
        const int half = rot / 2;
#pragma unroll
        for (int i = 0; i < 8; i += V)
            if (d + i < rot) y.load<V>(i, p + (d + i < half ? d + i + half : d + i - half));
#pragma unroll
        for (int i = 0; i < 8; i += V) {
            if (d + i >= rot) continue;
            const bool low = d + i < half;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float2 t = cs[d + i + j - (low ? 0 : half)];
                x.e[i + j] = to_16<DT>(to_f32<DT>(x.e[i + j]) * t.x + to_f32<DT>(y.e[i + j]) * (low ? -t.y : t.y));
            }
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
            if (d + j >= rot) continue;
            const float2 t = cs[(d + j) / 2];
            const float a = to_f32<DT>(x.e[j]), b = to_f32<DT>(x.e[j + 1]);
            x.e[j] = to_16<DT>(a * t.x - b * t.y);
            x.e[j + 1] = to_16<DT>(a * t.y + b * t.x);
        }
    }
    return x;
}

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
    int clear;
};

template <int DT, int LAYOUT, int V>
__global__ __launch_bounds__(kThreads) void rope_kernel(RopeK a) {
    __shared__ float2 cs[kThreads / 64][64];
    const Row w = begin_row(cs, a.T, a.rows, a.pos, a.S, a.rope, a.sign);
    const uint16_t* in = a.in + w.r * a.in_stride;
    uint16_t* out = a.out + w.r * a.out_stride;
    if (w.pos < 0) {
        if (a.clear && w.r < a.rows)
            for (int i = w.t; i < a.all * (a.D / 8); i += w.T) *(u32x4*)(out + i * 8) = u32x4{0u, 0u, 0u, 0u};
        return;
    }
    const int chunks = a.D / 8, rotate = a.heads * chunks, all = in == out ? rotate : a.all * chunks;
    for (int i = w.t; i < all; i += w.T) {
        Chunk x;
        if (i < rotate) {
            const int d = i % chunks * 8;
            x = rotated<DT, LAYOUT, V>(in + i * 8 - d, d, a.rope.rot, w.cs);
        } else {
            x.load<8>(0, in + i * 8);
        }
        __builtin_amdgcn_wave_barrier();      // all lanes have read before one writes
        x.store(out + i * 8);
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
    const int tok = (int)(slot & 31), rot = a.rope.rot, D = kv.D, chunks = D / 8;
    const uint16_t* in = a.qkv + w.r * a.stride;
    uint16_t* q = a.q ? a.q + w.r * a.q_stride : nullptr;
    for (int i = (a.q ? 0 : a.Hq * chunks) + w.t; i < (a.Hq + (kept ? kv.Hkv : 0)) * chunks; i += w.T) {
        const int h = i / chunks, d = i % chunks * 8;
        const Chunk x = rotated<DT, LAYOUT, V>(in + h * D, d, rot, w.cs);
        __builtin_amdgcn_wave_barrier();      // all lanes have read before one writes
        if (h < a.Hq) x.store(q + h * D + d);
        else x.store((uint16_t*)kv.k + tile_of(kv, slot, h - a.Hq) + (d >> 5) * 1024 + tok * 32 + (d & 31));
    }
    if (!kept) return;
    if (a.T == kThreads) {             // few rows: V here too, its values to 64-byte rows of their own
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

// Rows up to which one has a whole workgroup, else a wave (32 + 2 * 8 heads of 128, kernels, workgroup and wave: rotation of
// 64 rows 4.7 and 8.0 us, 1024 7.5 and 9.3, 2048 10.4 and 12.6, 4096 17 and 17; into the cache, where the many have V in
// tiles of 32 rows, 64 rows 6.7 and 9.6, 256 8.9 and 11.8, 450 10.8 and 10.1, 900 15.5 and 11.4).
constexpr int kFewTurned = 4096, kFewStored = 400;
int threads_a_row(int rows, int few) { return rows <= few ? kThreads : 64; }
unsigned row_blocks(int rows, int few) {
    const unsigned each = kThreads / threads_a_row(rows, few);
    return ((unsigned)rows + each - 1) / each;
}

// Other sides of pairs that are one access.
int sides(const tkm_attn_rope& r) {
    const int n = r.layout == TKM_ROPE_HALVES ? r.rot / 2 : 8;
    return n % 8 == 0 ? 8 : n % 4 == 0 ? 4 : n % 2 == 0 ? 2 : 1;
}

template <class A, class F>
void pick(int dtype, const tkm_attn_rope& r, const A& a, F launch) {
    const int v = sides(r);
    auto with = [&](auto DT) {
        using H = std::integral_constant<int, TKM_ROPE_HALVES>;
        if (r.layout != TKM_ROPE_HALVES) launch(DT, std::integral_constant<int, TKM_ROPE_PAIRS>{}, std::integral_constant<int, 8>{});
        else if (v == 8) launch(DT, H{}, std::integral_constant<int, 8>{});
        else if (v == 4) launch(DT, H{}, std::integral_constant<int, 4>{});
        else if (v == 2) launch(DT, H{}, std::integral_constant<int, 2>{});
        else launch(DT, H{}, std::integral_constant<int, 1>{});
    };
    if (dtype == TKM_ATTN_F16) with(std::integral_constant<int, DT_F16>{});
    else with(std::integral_constant<int, DT_BF16>{});
}

}  // namespace

bool rows_fit(const tkm_attn_kv* kv, int rows) {
    double blocks = row_blocks(rows, kv ? kFewStored : kFewTurned);
    if (kv) blocks += (rows + 31.0) / 32.0 * kv->Hkv;
    return launch_fits(blocks, kThreads);
}

int launch_rope(const RopeArgs& a) {
    RopeK k{a.rope, (const uint16_t*)a.in, (uint16_t*)a.out, a.pos, a.in_stride, a.out_stride, a.S, a.rows, a.Hq + a.Hkv,
            a.Hq + 2 * a.Hkv, a.D, threads_a_row(a.rows, kFewTurned), a.inverse ? -1.0f : 1.0f, a.clear};
    note_kernels(kRope);
    pick(a.dtype, a.rope, k, [&](auto DT, auto L, auto V) {
        hipLaunchKernelGGL((rope_kernel<decltype(DT)::value, decltype(L)::value, decltype(V)::value>), dim3(row_blocks(a.rows, kFewTurned)),
                           dim3(kThreads), 0, (hipStream_t)a.stream, k);
    });
    return hipGetLastError() == hipSuccess ? 0 : -1;
}

int launch_store(const StoreArgs& a) {
    StoreK k{a.kv, {}, (const uint16_t*)a.qkv, (uint16_t*)a.q, a.seq, a.pos, a.slot, a.stride, a.q_stride, a.rows, a.Hq,
             threads_a_row(a.rows, kFewStored), (int)row_blocks(a.rows, kFewStored)};
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
