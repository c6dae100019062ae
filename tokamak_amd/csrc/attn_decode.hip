// attn_decode.hip -- attention of one new token a sequence over a paged key-value cache (gfx950).
//
//   s_j = scale <q, k_j>, j < len[b];  o = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m);  lse = m + ln sum_j exp(s_j - m)
//
// Bound by HBM: every K and V value is read once for 4 * Hq/Hkv operations. A tile of 32 tokens goes from HBM
// into MFMA operand registers (the cache's layout, attn_kv.h), per wave and tile:
//   S^T = K Q^T    two 16x16 blocks: rows = tokens, columns = 16 of the kv head's query heads (a kv head with
//                  more has them in up to 4 waves, which read the same tiles at the same time)
//   P^T            stays where it is: a lane holds 8 consecutive tokens of one head, which is the B operand of
//   O^T += V^T P^T D/16 blocks of 16 dims x 16 heads, contracted over the tile's 32 tokens
// K's rows are dealt to the two blocks so that the 8 tokens a lane ends up with are consecutive: row r of block
// t is token 8 (r/4) + 4 t + r%4.  P goes to the second product as two 16-bit halves (hi + lo), which leaves
// only the output's own rounding: the MFMAs have 20 times the rate that HBM can feed, so it costs no time.
//
// The running maximum m moves only when a score exceeds it by more than 8 (log2 units), so that a tile needs no
// exchange between lanes; P = exp2(s - m + 6) then stays below 2^14, and what fp16's smallest value loses of a
// P is below 2^-31 of the row's largest.
//
// Split over the length: all tiles of all rows (row = sequence, kv head, group of query heads) are numbered
// row after row, and every workgroup takes the same count T of consecutive ones, whatever the lengths are:
// the lengths are read on the device, so a captured launch fits any. T is the least that 512 (two to a CU)
// workgroups cover. A workgroup whose tiles lie in one row deals them to its 4 waves in turn and merges
// them through LDS; otherwise each wave takes a quarter of the range by itself. Rows that no one worker has
// whole are merged from the pieces in a second launch, in the order of the tokens: results do not depend on
// timing.
#include <hip/hip_runtime.h>

#include "attn_common.h"
#include "attn_kv.h"
#include "attn_launch.h"

namespace tkm {
namespace {

constexpr float kSlack = 8.0f;   // m moves when a score exceeds it by more than this (log2)
constexpr float kLift = 6.0f;    // P = 2^(s - m + kLift)
constexpr int kWaves = 4;        // waves of a workgroup
constexpr int kGroups = 512;     // workgroups of a split launch: two on each of 256 compute units
constexpr float kLn2 = 0.69314718055994531f;

typedef float f32x2 __attribute__((ext_vector_type(2)));

template <int DT>
__device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c) {
    if constexpr (DT == DT_F16)
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// Two fp32 as 16-bit hi and lo = 16-bit(x - hi): the words {hi, lo}.
template <int DT>
__device__ __forceinline__ u32x2 split2(float x, float y) {
    if constexpr (DT == DT_BF16) return pack_split_bf16(x, y);
    const uint32_t hi = pack2<DT_F16>(x, y);
    const f16x2 h = as_f16x2(hi);
    return u32x2{hi, pack2<DT_F16>(x - (float)h[0], y - (float)h[1])};
}

__device__ __forceinline__ float quad_max(float v) {   // over lanes l, l^16, l^32, l^48
    v = fmaxf(v, __shfl_xor(v, 16, 64));
    return fmaxf(v, __shfl_xor(v, 32, 64));
}
__device__ __forceinline__ float quad_sum(float v) {
    v += __shfl_xor(v, 16, 64);
    return v + __shfl_xor(v, 32, 64);
}
__device__ __forceinline__ int uni(int v) { return __builtin_amdgcn_readfirstlane(v); }

// Tiles of a sequence; a length outside the table's capacity has none (its rows become NaN).
__device__ __forceinline__ int tiles_of(int len, int cap) { return (unsigned)len > (unsigned)cap ? 0 : (len + 31) >> 5; }

struct P {   // kernel arguments
    const uint16_t* k;
    const uint16_t* v;
    const int32_t* table;
    const int32_t* len;
    const uint16_t* q;
    uint16_t* o;
    float* lse;
    float* part;      // pieces: [slot][cols][D] unnormalised O, then [slot][cols] (m, l)
    f32x2* part_ml;
    float* scores;    // [B][Hq][cap] log2 units, or NULL
    float* lse2;      // [B][Hq] log2 units, or NULL (with scores)
    float* weight;
    long long q_stride;
    int B, Hkv, G, HG, num_pages, page_shift, max_pages, cap;
    int cols;         // query heads of a group: min(G, 16 * NH)
    int groups;       // workgroups of a split launch; 0: one workgroup a row
    float sl2;        // scale * log2(e)
};

// Tiles of the whole call and of the sequences before b.
__device__ __forceinline__ void count_tiles(const P& a, int b, int lane, int& all, int& before) {
    all = before = 0;
    for (int c = 0; c < a.B; c += 64) {
        const int n = c + lane < a.B ? tiles_of(a.len[c + lane], a.cap) : 0;
        const int s = wave_scan(n);
        if (b >= c && b < c + 64) before = all + lane_value(s - n, b - c);
        all += lane_value(s, 63);
    }
}
// Tiles of each worker of a call of n: the least that covers them.
__device__ __forceinline__ int tiles_each(int n, int workers) { return (n + workers - 1) / workers; }

// Adds a piece's sums, of maximum ml[0], to those of maximum mm >= ml[0]. A piece without a finite score
// has nothing but perhaps a NaN in ml[1].
__device__ __forceinline__ void add_piece(f32x2 ml, f32x4 x, float mm, f32x4& o, float& l) {
    const bool none = ml[0] == -INFINITY;
    const float f = none ? 0.f : fast_exp2(ml[0] - mm);
    l += none ? ml[1] : f * ml[1];
    o += f * x;
}

// Where a wave stands: tile `tile` of the `nt` of row `rh` (kv head and query head group) of sequence b.
struct At {
    int b, rh, tile, nt, len;
};

// NH waves hold 16 query heads each of the group, and TW = 4 / NH such sets walk tiles of their own.
template <int D, int DT, int NH, bool SC>
__global__ __launch_bounds__(64 * kWaves, 2) void decode_kernel(P a) {
    constexpr int KS = D / 32, DB = D / 16, TW = kWaves / NH;
    constexpr uint32_t TILE = D * 64;   // bytes of a tile of K or V
    __shared__ float red_o[kWaves][16][D + 4];   // padded: 16 heads' rows start in other banks
    __shared__ f32x2 red_ml[kWaves][16];

    const int lane = threadIdx.x & 63, wave = uni(threadIdx.x >> 6);
    const int hs = wave / TW, tw = wave % TW;
    const int n16 = lane & 15, quad = lane >> 4;
    const int RH = a.Hkv * a.HG;

    // ---- this wave's tiles
    At it;
    int count, stride;     // tiles to do, and the step between them
    bool shared;           // the workgroup's tiles are all of one row
    bool whole;            // ... and all of the row's
    int slot = 0;
    if (a.groups == 0) {
        it.b = blockIdx.x / RH;
        it.rh = blockIdx.x % RH;
        it.len = a.len[it.b];
        it.nt = tiles_of(it.len, a.cap);
        it.tile = tw;
        count = (it.nt - tw + TW - 1) / TW;
        stride = TW;
        shared = whole = true;
    } else {
        // the first 64 sequences' tiles, their running sum, and the call's
        const int n0 = lane < a.B ? tiles_of(a.len[lane], a.cap) : 0, s0 = wave_scan(n0);
        int all = lane_value(s0, 63);
        for (int c = 64; c < a.B; c += 64) all += lane_value(wave_scan(c + lane < a.B ? tiles_of(a.len[c + lane], a.cap) : 0), 63);
        all *= RH;
        const int t = tiles_each(all, a.groups * TW);
        const int first = blockIdx.x * TW * t, last = min(first + TW * t, all);
        if (first >= last) return;
        auto find = [&](int at) {     // the row that holds tile `at`
            int before = 0, n = n0, s = s0;
            for (int c = 0;; c += 64) {
                const uint64_t m = __ballot((before + s) * RH > at);
                if (m) {
                    const int w = __ffsll((unsigned long long)m) - 1;
                    it.b = uni(c + w);
                    it.nt = lane_value(n, w);
                    it.len = a.len[it.b];
                    const int r = at - (before + lane_value(s, w) - it.nt) * RH;
                    it.rh = r / it.nt;
                    it.tile = r % it.nt;
                    return;
                }
                before += lane_value(s, 63);
                n = c + 64 + lane < a.B ? tiles_of(a.len[c + 64 + lane], a.cap) : 0;
                s = wave_scan(n);
            }
        };
        find(first);
        shared = last - first <= it.nt - it.tile;
        whole = shared && it.tile == 0 && last - first == it.nt;
        if (shared) {
            slot = blockIdx.x * TW * 2 + (it.tile == 0 ? 1 : 0);
            it.tile += tw;
            count = max(0, (last - first - tw + TW - 1) / TW);
            stride = TW;
        } else {
            const int mine = first + tw * t;
            if (mine >= last) return;
            if (tw) find(mine);
            count = min(t, last - mine);
            stride = 1;
        }
    }

    // ---- the walk
    const uint32_t koff = (uint32_t)(8 * (n16 >> 2) + (n16 & 3)) * 64 + quad * 16;   // + t * 256 + ks * 2048
    const uint32_t voff = (uint32_t)n16 * 64 + quad * 16;                            // + db * 1024
    const int sub_mask = (1 << (a.page_shift - 5)) - 1;
    u32x4 kf[2][2][KS], vf[2][DB], qf[KS], qn[KS];
    f32x4 acc[DB];
    float m, l;
    bool bad = false;

    auto load = [&](int buf, const At& x) {
        const int page = a.table[(long long)x.b * a.max_pages + (x.tile >> (a.page_shift - 5))];
        const bool ok = (unsigned)page < (unsigned)a.num_pages;
        bad |= !ok;      // page 0 is read in its place, and the row becomes NaN
        const long long tile = (((long long)(ok ? page : 0) * a.Hkv + x.rh / a.HG) << (a.page_shift - 5)) + (x.tile & sub_mask);
        const char* kb = (const char*)a.k + tile * TILE;
        const char* vb = (const char*)a.v + tile * TILE;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int t = 0; t < 2; ++t) kf[buf][t][ks] = *(const u32x4*)(kb + koff + t * 256 + ks * 2048);
#pragma unroll
        for (int db = 0; db < DB; ++db) vf[buf][db] = *(const u32x4*)(vb + voff + db * 1024);
    };
    // this lane's query head within the kv head, of row x
    auto head_of = [&](const At& x) { return (x.rh % a.HG * NH + hs) * 16 + n16; };
    auto load_q = [&](const At& x) {
        const int h = head_of(x);
        const uint16_t* qp = a.q + (long long)x.b * a.q_stride + (x.rh / a.HG * a.G + h) * D + quad * 8;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) qn[ks] = h < a.G ? ld_global16(qp + ks * 32) : u32x4{0u, 0u, 0u, 0u};
    };
    auto reset = [&]() {
        m = -INFINITY;
        l = 0.f;
#pragma unroll
        for (int db = 0; db < DB; ++db) acc[db] = f32x4{0.f, 0.f, 0.f, 0.f};
        bad = false;
    };
    auto tile = [&](int buf, const At& x) {
        const int left = x.len - x.tile * 32;         // visible tokens of the tile
        f32x4 s0 = {0.f, 0.f, 0.f, 0.f}, s1 = s0;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            s0 = mfma16<DT>(kf[buf][0][ks], qf[ks], s0);
            s1 = mfma16<DT>(kf[buf][1][ks], qf[ks], s1);
        }
        float s[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            s[i] = s0[i] * a.sl2;
            s[4 + i] = s1[i] * a.sl2;
        }
        if (left < 32) {
            // what lies behind the last token may be anything: its scores are replaced, and as 0 * NaN is not 0
            // its values become 0 too
#pragma unroll
            for (int i = 0; i < 8; ++i) s[i] = quad * 8 + i < left ? s[i] : -INFINITY;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int at = quad * 8 + 2 * i;
                const uint32_t keep = (at < left ? 0xffffu : 0u) | (at + 1 < left ? 0xffff0000u : 0u);
#pragma unroll
                for (int db = 0; db < DB; ++db) vf[buf][db][i] &= keep;
            }
        }
        if (SC && head_of(x) < a.G) {
            float* sp = a.scores + (((long long)x.b * a.Hkv + x.rh / a.HG) * a.G + head_of(x)) * a.cap + x.tile * 32 + quad * 8;
            *(f32x4*)sp = f32x4{s[0], s[1], s[2], s[3]};
            *(f32x4*)(sp + 4) = f32x4{s[4], s[5], s[6], s[7]};
        }
        const float top = fmaxf(fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3])), fmaxf(fmaxf(s[4], s[5]), fmaxf(s[6], s[7])));
        if (__any(top > m + kSlack)) {
            const float mn = fmaxf(m, quad_max(top));
            const float f = mn == -INFINITY ? 1.0f : fast_exp2(m - mn);
            m = mn;
            l *= f;
#pragma unroll
            for (int db = 0; db < DB; ++db) acc[db] *= f;
        }
        const float ref = m == -INFINITY ? 0.f : m - kLift;
        float p[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) p[i] = fast_exp2(s[i] - ref);
        l += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
        u32x4 hi, lo;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const u32x2 w = split2<DT>(p[2 * i], p[2 * i + 1]);
            hi[i] = w[0];
            lo[i] = w[1];
        }
#pragma unroll
        for (int db = 0; db < DB; ++db) acc[db] = mfma16<DT>(vf[buf][db], hi, acc[db]);
#pragma unroll
        for (int db = 0; db < DB; ++db) acc[db] = mfma16<DT>(vf[buf][db], lo, acc[db]);
    };
    // output row of a head of the kv head of x
    auto out_row = [&](const At& x, int h) { return ((long long)x.b * a.Hkv + x.rh / a.HG) * a.G + h; };
    auto put_lse = [&](long long row, float mm, float ll) {
        const float l2 = ll > 0.f ? mm - kLift + __log2f(ll) : ll == 0.f ? -INFINITY : NAN;
        if (a.lse) a.lse[row] = ll > 0.f ? (mm - kLift) * kLn2 + logf(ll) : l2;
        if (SC) a.lse2[row] = l2;
    };
    auto finish = [&](const At& x, bool all, int at) {   // private mode: this wave's sums of a row's piece
        float ll = quad_sum(l);
        if (bad) ll = NAN;
        const int h = head_of(x), c = hs * 16 + n16;
        if (h >= a.G) return;
        if (all) {
            const long long row = out_row(x, h);
            const float inv = ll == 0.f ? 0.f : 1.0f / ll;
#pragma unroll
            for (int db = 0; db < DB; ++db) {
                const f32x4 v = acc[db] * inv;
                *(u32x2*)(a.o + row * D + db * 16 + quad * 4) = u32x2{pack2<DT>(v[0], v[1]), pack2<DT>(v[2], v[3])};
            }
            if (quad == 0) put_lse(row, m, ll);
        } else {
            float* pp = a.part + ((long long)at * a.cols + c) * D + quad * 4;
#pragma unroll
            for (int db = 0; db < DB; ++db) *(f32x4*)(pp + db * 16) = acc[db];
            if (quad == 0) a.part_ml[(long long)at * a.cols + c] = f32x2{m, ll};
        }
    };
    auto advance = [&](At& x) {
        x.tile += stride;
        if (!shared && x.tile == x.nt) {
            x.tile = 0;
            if (++x.rh == RH) {
                x.rh = 0;
                do {
                    ++x.b;
                    x.len = a.len[x.b];
                    x.nt = tiles_of(x.len, a.cap);
                } while (x.nt == 0);
            }
        }
    };

    reset();
    if (count > 0) {
        At nx = it;
        int from = it.tile;      // first tile of the row's piece (private mode)
        load_q(it);
        load(0, it);
        bool bad_next = bad;
        bad = false;
        auto step = [&](int buf, int i) {
            const bool more = i + 1 < count;
            if (i == 0 || (!shared && it.tile == 0)) {
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) qf[ks] = qn[ks];
            }
            const bool was = bad | bad_next;
            bad = false;
            if (more) {
                advance(nx);
                load(buf ^ 1, nx);
                if (!shared && nx.tile == 0) load_q(nx);
            }
            bad_next = bad;
            bad = was;
            tile(buf, it);
            if (!shared && (!more || nx.tile == 0)) {
                const int n = it.tile + 1 - from;
                const int w = blockIdx.x * TW + tw;
                finish(it, n == it.nt, w * 2 + (from == 0 ? 1 : 0));
                reset();
                from = 0;
            }
            it = nx;
        };
        for (int i = 0; i < count; i += 2) {
            step(0, i);
            if (i + 1 < count) step(1, i + 1);
        }
        if (shared) bad |= bad_next;
    }
    if (!shared) return;

    // ---- shared mode: the waves' sums of one row
    {
        float ll = quad_sum(l);
        if (bad) ll = NAN;
        if (quad == 0) red_ml[wave][n16] = f32x2{m, ll};
#pragma unroll
        for (int db = 0; db < DB; ++db) *(f32x4*)&red_o[wave][n16][db * 16 + quad * 4] = acc[db];
    }
    __syncthreads();
    it.len = a.len[it.b];
    const bool lost = (unsigned)it.len > (unsigned)a.cap;     // no length of this table
    const int h0 = it.rh % a.HG * NH * 16, have = min(a.cols, a.G - h0);
    for (int i = threadIdx.x; i < have * (D / 4); i += 64 * kWaves) {
        const int c = i / (D / 4), d = i % (D / 4) * 4, w0 = c / 16 * TW;
        float mm = -INFINITY;
#pragma unroll
        for (int w = 0; w < TW; ++w) mm = fmaxf(mm, red_ml[w0 + w][c % 16][0]);
        f32x4 o = {0.f, 0.f, 0.f, 0.f};
        float ll = 0.f;
#pragma unroll
        for (int w = 0; w < TW; ++w) add_piece(red_ml[w0 + w][c % 16], *(const f32x4*)&red_o[w0 + w][c % 16][d], mm, o, ll);
        if (whole) {
            if (lost) ll = NAN;
            const float inv = ll == 0.f ? 0.f : 1.0f / ll;
            o *= inv;
            const long long row = out_row(it, h0 + c);
            *(u32x2*)(a.o + row * D + d) = u32x2{pack2<DT>(o[0], o[1]), pack2<DT>(o[2], o[3])};
            if (d == 0) put_lse(row, mm, ll);
        } else {
            *(f32x4*)(a.part + ((long long)slot * a.cols + c) * D + d) = o;
            if (d == 0) a.part_ml[(long long)slot * a.cols + c] = f32x2{mm, ll};
        }
    }
}

// The rows that the split launch left in pieces, and those without a tile. One workgroup a query head: D/4
// threads have 4 dims each of a piece, and the workgroup's groups of them take pieces in turn, 8 in flight.
template <int D, int DT, int NH>
__global__ __launch_bounds__(256) void join_kernel(P a) {
    constexpr int TW = kWaves / NH, DV = D / 4, PAR = 256 / DV, FLY = 8;
    __shared__ f32x4 red_o[PAR][DV];
    __shared__ f32x2 red_ml[PAR];
    const int tid = threadIdx.x, lane = tid & 63;
    const int h = blockIdx.x % (a.Hkv * a.G), b = blockIdx.x / (a.Hkv * a.G);
    const int kvh = h / a.G, hg = h % a.G / (16 * NH), c = h % a.G % (16 * NH);
    const int RH = a.Hkv * a.HG;
    const long long row = blockIdx.x;
    const int len = a.len[b], nt = tiles_of(len, a.cap);
    if (nt == 0) {
        const bool lost = len != 0;
        for (int d = tid; d < D; d += 256) a.o[row * D + d] = (uint16_t)(lost ? (DT == DT_F16 ? 0x7e00 : 0x7fc0) : 0);
        if (tid == 0 && a.lse) a.lse[row] = lost ? NAN : -INFINITY;
        if (tid == 0 && a.lse2) a.lse2[row] = lost ? NAN : -INFINITY;
        return;
    }
    int all, before;
    count_tiles(a, b, lane, all, before);
    all *= RH;
    const int t = tiles_each(all, a.groups * TW), T = t * TW;
    const int r0 = before * RH + (kvh * a.HG + hg) * nt, r1 = r0 + nt;
    const int w0 = r0 / t, w1 = (r1 - 1) / t;
    const int ga = (r0 + T - 1) / T, gb = r1 == all ? (r1 + T - 1) / T : r1 / T;   // workgroups [ga, gb) lie in the row
    if (w0 == w1 && ga >= gb) return;                  // one worker had all of it
    if (gb - ga == 1 && ga * T == r0 && r1 <= gb * T) return;   // one workgroup had
    const int head = ga < gb ? ga * TW - w0 : w1 - w0 + 1;      // pieces of single workers before those
    const int tail = ga < gb ? max(0, w1 + 1 - gb * TW) : 0;
    const int n = head + max(0, gb - ga) + tail;
    auto slot = [&](int i) {
        const int w = i < head ? w0 + i : i < head + (gb - ga) || tail == 0 ? (ga + i - head) * TW : gb * TW + i - head - (gb - ga);
        return ((long long)w * 2 + (w * t <= r0 ? 1 : 0)) * a.cols + c;
    };
    const int d = tid % DV, g = tid / DV;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    float mm = -INFINITY, ll = 0.f;
    for (int i0 = g; i0 < n; i0 += PAR * FLY) {
        f32x2 ml[FLY];
        f32x4 x[FLY];
        float top = mm;
#pragma unroll
        for (int j = 0; j < FLY; ++j) {
            const int i = i0 + j * PAR;
            ml[j] = f32x2{-INFINITY, 0.f};
            if (i < n) {
                const long long s = slot(i);
                ml[j] = a.part_ml[s];
                x[j] = *(const f32x4*)(a.part + s * D + d * 4);
            } else {
                x[j] = f32x4{0.f, 0.f, 0.f, 0.f};
            }
        }
#pragma unroll
        for (int j = 0; j < FLY; ++j) top = fmaxf(top, ml[j][0]);
        const float f = mm == -INFINITY ? 0.f : fast_exp2(mm - top);
        o *= f;
        ll = mm == -INFINITY ? ll : ll * f;
        mm = top;
#pragma unroll
        for (int j = 0; j < FLY; ++j) add_piece(ml[j], x[j], mm, o, ll);
    }
    red_o[g][d] = o;
    if (d == 0) red_ml[g] = f32x2{mm, ll};
    __syncthreads();
    if (tid >= DV) return;
    mm = -INFINITY;
#pragma unroll
    for (int i = 0; i < PAR; ++i) mm = fmaxf(mm, red_ml[i][0]);
    o = f32x4{0.f, 0.f, 0.f, 0.f};
    ll = 0.f;
#pragma unroll
    for (int i = 0; i < PAR; ++i) add_piece(red_ml[i], red_o[i][tid], mm, o, ll);
    o *= ll == 0.f ? 0.f : 1.0f / ll;
    *(u32x2*)(a.o + row * D + tid * 4) = u32x2{pack2<DT>(o[0], o[1]), pack2<DT>(o[2], o[3])};
    if (tid == 0) {
        const float l2 = ll > 0.f ? mm - kLift + __log2f(ll) : ll == 0.f ? -INFINITY : NAN;
        if (a.lse) a.lse[row] = ll > 0.f ? (mm - kLift) * kLn2 + logf(ll) : l2;
        if (a.lse2) a.lse2[row] = l2;
    }
}

// weight[b][kvh][j] += sum over the kv head's query heads of exp2(score - lse), 4 tokens a thread.
__global__ __launch_bounds__(256) void weights_kernel(P a) {
    const unsigned chunks = (unsigned)(a.cap + 1023) / 1024;
    const long long row = blockIdx.x / chunks;     // sequence and kv head
    const int j = (int)(blockIdx.x % chunks * 1024 + threadIdx.x * 4), len = a.len[row / a.Hkv];
    if ((unsigned)len > (unsigned)a.cap || j >= len) return;
    f32x4 w = {0.f, 0.f, 0.f, 0.f};
    for (int g = 0; g < a.G; ++g) {
        const float l2 = a.lse2[row * a.G + g];
        const f32x4 s = *(const f32x4*)(a.scores + (row * a.G + g) * a.cap + j);
        if (l2 == -INFINITY) continue;    // every score is -inf: no key has a weight
        if (l2 != l2) return;             // a page outside the pool: the weights stay
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] += fast_exp2(s[i] - l2);
    }
    float* wp = a.weight + row * a.cap + j;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (j + i < len) wp[i] += w[i];
}

// Waves that share a kv head's query heads, 16 each, and the groups of so many heads.
int head_waves(int G) { return G <= 16 ? 1 : G <= 32 ? 2 : 4; }
int head_groups(int G) { return (G + 63) / 64; }
int head_cols(int G) { return G < 64 ? G : 64; }
size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }

// Whether a call runs as one workgroup a row, without pieces.
bool by_row(int cap) { return cap <= 512; }

int groups_of(const tkm_attn_kv& kv, int Hq) {
    const double most = decode_tiles_most(kv, Hq) * head_waves(Hq / kv.Hkv) / kWaves + 1;
    return most < kGroups ? (int)most : kGroups;
}

template <int D, int DT, int NH>
int run(const P& a, int B, hipStream_t st) {
    const unsigned grid = a.groups ? (unsigned)a.groups : (unsigned)(B * a.Hkv * a.HG);
    if (a.scores)
        hipLaunchKernelGGL((decode_kernel<D, DT, NH, true>), dim3(grid), dim3(64 * kWaves), 0, st, a);
    else
        hipLaunchKernelGGL((decode_kernel<D, DT, NH, false>), dim3(grid), dim3(64 * kWaves), 0, st, a);
    if (a.groups)
        hipLaunchKernelGGL((join_kernel<D, DT, NH>), dim3((unsigned)(B * a.Hkv * a.G)), dim3(256), 0, st, a);
    if (a.scores)
        hipLaunchKernelGGL(weights_kernel, dim3((unsigned)(a.cap + 1023) / 1024 * (unsigned)(B * a.Hkv)), dim3(256), 0, st, a);
    return hipGetLastError() == hipSuccess ? 0 : -1;
}

template <int D, int DT>
int run_heads(const P& a, int B, hipStream_t st) {
    const int n = head_waves(a.G);
    return n == 1 ? run<D, DT, 1>(a, B, st) : n == 2 ? run<D, DT, 2>(a, B, st) : run<D, DT, 4>(a, B, st);
}

}  // namespace

double decode_tiles_most(const tkm_attn_kv& kv, int Hq) {
    return (double)kv.B * kv.Hkv * head_groups(Hq / kv.Hkv) * kv.max_pages * (kv.page / 32);
}

size_t decode_workspace(const tkm_attn_kv& kv, int Hq, int add_weights) {
    const int G = Hq / kv.Hkv;
    const long long cap = (long long)kv.max_pages * kv.page;
    size_t n = 0;
    if (!by_row((int)cap)) {
        const size_t slots = (size_t)groups_of(kv, Hq) * (kWaves / head_waves(G)) * 2 * head_cols(G);
        n += up256(slots * kv.D * 4) + up256(slots * 8);
    }
    if (add_weights) n += up256((size_t)kv.B * Hq * 4) + (size_t)kv.B * Hq * cap * 4;
    return n;
}

int launch_decode(const DecodeArgs& d) {
    const tkm_attn_kv& kv = d.kv;
    P a = {};
    a.k = (const uint16_t*)kv.k;
    a.v = (const uint16_t*)kv.v;
    a.table = kv.table;
    a.len = kv.len;
    a.q = (const uint16_t*)d.q;
    a.o = (uint16_t*)d.o;
    a.lse = d.lse;
    a.q_stride = d.q_stride;
    a.B = kv.B;
    a.Hkv = kv.Hkv;
    a.G = d.Hq / kv.Hkv;
    a.HG = head_groups(a.G);
    a.cols = head_cols(a.G);
    a.num_pages = kv.num_pages;
    a.page_shift = __builtin_ctz((unsigned)kv.page);
    a.max_pages = kv.max_pages;
    a.cap = kv.max_pages * kv.page;
    a.sl2 = d.scale * 1.4426950408889634f;
    a.groups = by_row(a.cap) ? 0 : groups_of(kv, d.Hq);
    char* ws = (char*)d.ws;
    if (a.groups) {
        const size_t slots = (size_t)a.groups * (kWaves / head_waves(a.G)) * 2 * a.cols;
        a.part = (float*)ws;
        ws += up256(slots * kv.D * 4);
        a.part_ml = (f32x2*)ws;
        ws += up256(slots * 8);
    }
    if (d.add_weights) {
        a.weight = kv.weight;
        a.lse2 = (float*)ws;
        ws += up256((size_t)kv.B * d.Hq * 4);
        a.scores = (float*)ws;
    }
    hipStream_t st = (hipStream_t)d.stream;
    note_kernels(kDecode | (a.groups ? kJoin : 0u) | (a.scores ? kWeights : 0u));
    return kv.D == 64 ? (kv.dtype == TKM_ATTN_BF16 ? run_heads<64, DT_BF16>(a, kv.B, st) : run_heads<64, DT_F16>(a, kv.B, st))
                      : (kv.dtype == TKM_ATTN_BF16 ? run_heads<128, DT_BF16>(a, kv.B, st) : run_heads<128, DT_F16>(a, kv.B, st));
}

}  // namespace tkm
