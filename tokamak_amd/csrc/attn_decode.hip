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
// t is token 8 (r/4) + 4 t + r%4.  P goes to the second product in 16-bit parts, two in
// fp16 and three in bf16, which leaves what fp32 leaves (bf16's first two lose up to 2^-17 of a P): the MFMAs have 13
// to 20 times the rate that HBM can feed, so it costs no time.
//
// The running maximum m moves only when a score exceeds it by more than 8 (log2 units), so that a tile needs no
// exchange between lanes; P = exp2(s - m + 6) then stays below 2^14, and what fp16's smallest value loses of a
// P is below 2^-31 of the row's largest.
//
// Split over the length: all tiles of all rows (row = sequence, kv head, group of query heads) are numbered
// row after row, and every workgroup takes the same count T of consecutive ones, whatever the lengths are:
// the lengths are read on the device, so a captured launch fits any. T is the least that 256 workgroups
// cover, one on each compute unit (us a call at 131035 tokens, 8 kv heads of D 128 / 64 sequences of up to 4096 / 16 of up
// to 8192 on one kv head: 256 97.8 / 125.8 / 15.5, 512 99.6 / 127.1 / 18.4, 1024 99.9 / 130.3 / 19.8: more
// leave more pieces). A workgroup whose tiles lie in one row deals them to its 4 waves in turn and merges
// them through LDS; otherwise each wave takes a quarter of the range by itself. Rows that no one worker has
// whole are merged from the pieces in a second launch, in the order of the tokens: results do not depend on
// timing.
//
// us of the kernels: 131035 tokens, 8 kv heads of D 128 (537 MB of K and V): 93, and 5 for the join: 5.5 TB/s (a loop that
// only reads takes 84 to 88 for as much; the XCDs read at different rates, 72 to 88 us for equal shares); 64 sequences
// of up to 4096 (671 MB on average): 117 + 5, 5.5 TB/s; 16 of up to 8192 on one kv head of 32 query heads (42 MB):
// 12.6 + 4.4; 200 tokens in one launch: 4.8.  With weights the second launch has a workgroup for each 1024 positions
// that the tables can hold: 16 sequences of 500 on 8 kv heads, 8.2 + 36 in tables of 32768 (10.6 in one launch where
// the tables hold 512).
#include <hip/hip_runtime.h>

#include <type_traits>

#include "attn_common.h"
#include "attn_kv.h"
#include "attn_launch.h"

namespace tkm {
namespace {

constexpr float kSlack = 8.0f;   // m moves when a score exceeds it by more than this (log2)
constexpr float kLift = 6.0f;    // P = 2^(s - m + kLift)
constexpr int kWaves = 4;        // waves of a workgroup of a split launch
constexpr int kRowWaves = 8;     // and where a workgroup has a row
constexpr int kGroups = 256;     // workgroups of a split launch: one on each compute unit
constexpr float kLn2 = 0.69314718055994531f;

typedef float f32x2 __attribute__((ext_vector_type(2)));

template <int DT>
__device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c) {
    if constexpr (DT == DT_F16)
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// Two fp32 P as 16-bit parts, each what the ones before leave, rounded: the words w[0], w[1], ..  Two parts in fp16
// hold 22 bits, three in bf16 the 24 of fp32.
template <int DT>
constexpr int kParts = DT == DT_BF16 ? 3 : 2;
template <int DT>
__device__ __forceinline__ void split_p(float x, float y, uint32_t (&w)[kParts<DT>]) {
#pragma unroll
    for (int i = 0; i < kParts<DT>; ++i) {
        w[i] = pack2<DT>(x, y);
        if constexpr (DT == DT_BF16) {
            x -= __uint_as_float(w[i] << 16);
            y -= __uint_as_float(w[i] & 0xffff0000u);
        } else {
            const f16x2 h = as_f16x2(w[i]);
            x -= (float)h[0];
            y -= (float)h[1];
        }
    }
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

// An element of an array that no kernel here writes, at a wave-uniform index: a scalar load also behind stores
// (which the compiler must otherwise take for possible writes to it, and wait for all vector loads with the page's).
__device__ __forceinline__ int fixed(const int32_t* p, long long i) {
    return *((const __attribute__((address_space(4))) int32_t*)(uintptr_t)p + i);
}

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

// LSE from a row's maximum and sum, in log2 units and natural.
__device__ __forceinline__ float lse2_of(float m, float l) { return l > 0.f ? m - kLift + __log2f(l) : l == 0.f ? -INFINITY : NAN; }
__device__ __forceinline__ float lse_of(float m, float l) { return l > 0.f ? (m - kLift) * kLn2 + logf(l) : l == 0.f ? -INFINITY : NAN; }

// Four positions' weights of `row` (sequence and kv head), j .. j + 3: loaded ahead of what is added to them.  The query
// heads' are summed first and added once: alone they may be below half a step of what a position has gathered.
struct Weights {
    f32x4 w, sum;
    float* at;
    int left;      // of the four, those of the sequence
    __device__ __forceinline__ void load(const P& a, long long row, int j, int len) {
        at = a.weight + row * a.cap + j;
        left = len - j;
        if (left > 0) __builtin_memcpy(&w, at, 16);      // a row ends at a multiple of 32
    }
    // adds exp2(score - LSE), l2 the LSE; a head whose LSE is NaN, or -inf (all its scores are), adds nothing
    __device__ __forceinline__ void add(f32x4 score, float l2) {
        if (!(l2 > -INFINITY)) return;
#pragma unroll
        for (int i = 0; i < 4; ++i) sum[i] += fast_exp2(score[i] - l2);
    }
    __device__ __forceinline__ void store() const {
        const f32x4 x = w + sum;
        if (left >= 4) __builtin_memcpy(at, &x, 16);
        else
            for (int i = 0; i < left; ++i) at[i] = x[i];
    }
};

// Where a wave stands: tile `tile` of the `nt` of row `rh` (kv head and query head group) of sequence b.
struct At {
    int b, rh, tile, nt, len;
};

// NH waves hold 16 query heads each of the group, and TW = NW / NH such sets walk tiles of their own.  ROW: a
// workgroup has a row, else its share of all tiles.  SC: the scores are kept, and with ROW and one group of query
// heads the row's weights are added here too.
template <int D, int DT, int NH, bool SC, bool ROW>
__global__ __launch_bounds__(64 * (ROW ? kRowWaves : kWaves), 2) void decode_kernel(P a) {
    constexpr int NW = ROW ? kRowWaves : kWaves, KS = D / 32, DB = D / 16, TW = NW / NH;
    constexpr uint32_t TILE = D * 64;   // bytes of a tile of K or V
    __shared__ float red_o[NW][16][D + 4];   // padded: 16 heads' rows start in other banks
    __shared__ f32x2 red_ml[NW][16];
    __shared__ float red_lse[16 * NH];

    const int lane = threadIdx.x & 63, wave = uni(threadIdx.x >> 6);
    const int hs = wave / TW, tw = wave % TW;
    const int n16 = lane & 15, quad = lane >> 4;
    const int RH = a.Hkv * a.HG;

    // ---- this wave's tiles
    At it;
    int count;             // tiles to do
    bool shared;           // the workgroup's tiles are all of one row
    bool whole;            // ... and all of the row's
    int slot = 0;
    if constexpr (ROW) {
        it.b = blockIdx.x / RH;
        it.rh = blockIdx.x % RH;
        it.len = fixed(a.len, it.b);
        it.nt = tiles_of(it.len, a.cap);
        it.tile = tw;
        count = (it.nt - tw + TW - 1) / TW;
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
        auto find = [&](int at) {     // the row that holds tile `at`; none, if the lengths have changed meanwhile
            int before = 0, n = n0, s = s0;
            for (int c = 0; c < a.B; c += 64) {
                const uint64_t m = __ballot((before + s) * RH > at);
                if (m) {
                    const int w = __ffsll((unsigned long long)m) - 1;
                    it.b = uni(c + w);
                    it.nt = lane_value(n, w);
                    it.len = fixed(a.len, it.b);
                    const int r = at - (before + lane_value(s, w) - it.nt) * RH;
                    it.rh = r / it.nt;
                    it.tile = r % it.nt;
                    return true;
                }
                before += lane_value(s, 63);
                n = c + 64 + lane < a.B ? tiles_of(a.len[c + 64 + lane], a.cap) : 0;
                s = wave_scan(n);
            }
            return false;
        };
        if (!find(first)) return;
        shared = last - first <= it.nt - it.tile;
        whole = shared && it.tile == 0 && last - first == it.nt;
        if (shared) {
            slot = blockIdx.x * TW * 2 + (it.tile == 0 ? 1 : 0);
            it.tile += tw;
            count = max(0, (last - first - tw + TW - 1) / TW);
        } else {
            const int mine = first + tw * t;
            if (mine >= last) return;
            if (tw && !find(mine)) return;
            count = min(t, last - mine);
        }
    }

    // ---- the walk
    const uint32_t koff = (uint32_t)(8 * (n16 >> 2) + (n16 & 3)) * 64 + quad * 16;   // + t * 256 + ks * 2048
    const uint32_t voff = (uint32_t)n16 * 64 + quad * 16;                            // + db * 1024
    const int tile_bits = a.page_shift - 5, sub_mask = (1 << tile_bits) - 1;
    u32x4 kf[2][2][KS], vf[2][DB], qf[KS];
    f32x4 acc[DB];
    float m, l;
    bool bad;

    // (of a tile behind the row's last, the table's last or whatever it says: it is not used)
    auto page_of = [&](const At& x, int tile) { return fixed(a.table, (long long)x.b * a.max_pages + min(tile >> tile_bits, a.max_pages - 1)); };
    auto load = [&](int buf, const At& x, int tile, int page) {
        const bool ok = (unsigned)page < (unsigned)a.num_pages;
        bad |= !ok;      // page 0 is read in its place, and the row becomes NaN
        const long long at = (((long long)(ok ? page : 0) * a.Hkv + x.rh / a.HG) << tile_bits) + (tile & sub_mask);
        const char* kb = (const char*)a.k + at * TILE;
        const char* vb = (const char*)a.v + at * TILE;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int t = 0; t < 2; ++t) kf[buf][t][ks] = *(const u32x4*)(kb + koff + t * 256 + ks * 2048);
#pragma unroll
        for (int db = 0; db < DB; ++db) vf[buf][db] = *(const u32x4*)(vb + voff + db * 1024);
    };
    // this lane's query head within the kv head, of row x
    auto head_of = [&](const At& x) { return (x.rh % a.HG * NH + hs) * 16 + n16; };
    auto reset = [&]() {
        m = -INFINITY;
        l = 0.f;
#pragma unroll
        for (int db = 0; db < DB; ++db) acc[db] = f32x4{0.f, 0.f, 0.f, 0.f};
        bad = false;
    };
    // a tile's scores, log2 units: of tokens quad * 8 .. + 7
    auto scores = [&](int buf, float (&s)[8]) {
        f32x4 s0 = {0.f, 0.f, 0.f, 0.f}, s1 = s0;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            s0 = mfma16<DT>(kf[buf][0][ks], qf[ks], s0);
            s1 = mfma16<DT>(kf[buf][1][ks], qf[ks], s1);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            s[i] = s0[i] * a.sl2;
            s[4 + i] = s1[i] * a.sl2;
        }
    };
    auto tile = [&](int buf, const At& x, int tile, auto last) {
        const int left = decltype(last)::value ? x.len - tile * 32 : 32;         // visible tokens of the tile
        float s[8];
        scores(buf, s);
        if (decltype(last)::value && left < 32) {
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
            float* sp = a.scores + (((long long)x.b * a.Hkv + x.rh / a.HG) * a.G + head_of(x)) * a.cap + tile * 32 + quad * 8;
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
        u32x4 pw[kParts<DT>];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t w[kParts<DT>];
            split_p<DT>(p[2 * i], p[2 * i + 1], w);
#pragma unroll
            for (int j = 0; j < kParts<DT>; ++j) pw[j][i] = w[j];
        }
#pragma unroll
        for (int j = 0; j < kParts<DT>; ++j)
#pragma unroll
            for (int db = 0; db < DB; ++db) acc[db] = mfma16<DT>(vf[buf][db], pw[j], acc[db]);
    };
    // An infinite value times a part of P that is 0 or negative makes NaN of a sum, where exp(s - m) > 0 makes it
    // infinite.  So sums that are NaN are looked at again, over the same tiles: which of their values are infinite, in
    // which direction (a NaN counts as both), and whether a token's exp is 0, which leaves NaN.
    auto recount = [&](const At& x, int n, int stride) {
        constexpr uint32_t inf16 = DT == DT_F16 ? 0x7c00u : 0x7f80u, one = DT == DT_F16 ? 0x3c00u : 0x3f80u;
        f32x4 up[DB], down[DB];
#pragma unroll
        for (int db = 0; db < DB; ++db) up[db] = down[db] = f32x4{0.f, 0.f, 0.f, 0.f};
        const float ref = m == -INFINITY ? 0.f : m - kLift;
        for (int at = x.tile; n > 0; --n, at += stride) {
            load(0, x, at, page_of(x, at));
            const int left = x.len - at * 32;
            float s[8];
            scores(0, s);
            u32x4 some, none, keep;      // tokens whose exp is positive, or 0; those of the sequence
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                some[i] = none[i] = keep[i] = 0;
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const float p = fast_exp2(s[2 * i + j] - ref);
                    some[i] |= p > 0.f ? one << 16 * j : 0u;
                    none[i] |= p == 0.f ? one << 16 * j : 0u;
                    keep[i] |= quad * 8 + 2 * i + j < left ? 0xffffu << 16 * j : 0u;
                }
            }
#pragma unroll
            for (int db = 0; db < DB; ++db) {
                u32x4 pos, neg, any;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t w = vf[0][db][i] & keep[i];
                    pos[i] = neg[i] = any[i] = 0;
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const uint32_t h = w >> 16 * j & 0xffffu, size = h & 0x7fffu;
                        pos[i] |= size > inf16 || h == inf16 ? one << 16 * j : 0u;
                        neg[i] |= size > inf16 || h == (inf16 | 0x8000u) ? one << 16 * j : 0u;
                        any[i] |= size >= inf16 ? one << 16 * j : 0u;
                    }
                }
                up[db] = mfma16<DT>(any, none, mfma16<DT>(pos, some, up[db]));
                down[db] = mfma16<DT>(any, none, mfma16<DT>(neg, some, down[db]));
            }
        }
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const bool u = up[db][i] > 0.f, d = down[db][i] > 0.f;
                if (acc[db][i] != acc[db][i] && u != d) acc[db][i] = u ? INFINITY : -INFINITY;
            }
    };
    // output row of a head of the kv head of x
    auto out_row = [&](const At& x, int h) { return ((long long)x.b * a.Hkv + x.rh / a.HG) * a.G + h; };
    auto put_lse = [&](long long row, float mm, float ll) {
        const float l2 = lse2_of(mm, ll);
        if (a.lse) a.lse[row] = lse_of(mm, ll);
        if (SC) a.lse2[row] = l2;
        return l2;
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
    // The sums of n tiles of row x from x.tile on, `stride` apart: the next tile's loads, and the page of the one
    // after it, are under way while a tile is computed.  Straight code for all but the last two, so that the
    // compiler can count what is in flight (a load under a condition, and it waits for all of them).
    auto walk = [&](const At& x, int n, int stride) {
        const int all = n;
        reset();
        const int h = head_of(x);
        const uint16_t* qp = a.q + (long long)x.b * a.q_stride + (x.rh / a.HG * a.G + min(h, a.G - 1)) * D + quad * 8;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            const u32x4 w = ld_global16(qp + ks * 32);
            qf[ks] = h < a.G ? w : u32x4{0u, 0u, 0u, 0u};
        }
        int at = x.tile, page = page_of(x, at + stride);
        load(0, x, at, page_of(x, at));
        auto go = [&](int buf) {          // computes tile `at`, with two more to come
            const int next = at + stride, p = page;
            page = page_of(x, next + stride);
            load(buf ^ 1, x, next, p);
            tile(buf, x, at, std::false_type());
            at = next;
        };
        for (; n > 2; n -= 2) {
            go(0);
            go(1);
        }
        if (n == 2) {
            go(0);
            tile(1, x, at, std::true_type());
        } else {
            tile(0, x, at, std::true_type());
        }
        bool nan = false;
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
            for (int i = 0; i < 4; ++i) nan |= acc[db][i] != acc[db][i];
        if (__builtin_expect(__any(nan), 0)) recount(x, all, stride);
    };

    if (shared) {
        if (count > 0) walk(it, count, TW);
        else reset();
    } else {
        while (true) {
            const int n = min(count, it.nt - it.tile);
            walk(it, n, 1);
            finish(it, n == it.nt, (blockIdx.x * TW + tw) * 2 + (it.tile == 0 ? 1 : 0));
            count -= n;
            if (count == 0) return;
            it.tile = 0;                 // of the next row with tiles
            if (++it.rh == RH) {
                it.rh = 0;
                do {
                    if (++it.b == a.B) return;
                    it.len = fixed(a.len, it.b);
                    it.nt = tiles_of(it.len, a.cap);
                } while (it.nt == 0);
            }
        }
    }

    // ---- shared mode: the waves' sums of one row
    {
        float ll = quad_sum(l);
        if (bad) ll = NAN;
        if (quad == 0) red_ml[wave][n16] = f32x2{m, ll};
#pragma unroll
        for (int db = 0; db < DB; ++db) *(f32x4*)&red_o[wave][n16][db * 16 + quad * 4] = acc[db];
    }
    it.len = fixed(a.len, it.b);
    Weights ws = {};
    const long long kvrow = (long long)it.b * a.Hkv + it.rh / a.HG;
    if constexpr (SC && ROW)
        if ((unsigned)it.len <= (unsigned)a.cap) ws.load(a, kvrow, threadIdx.x * 4, it.len);
    __syncthreads();
    const bool lost = (unsigned)it.len > (unsigned)a.cap;     // no length of this table
    const int h0 = it.rh % a.HG * NH * 16, have = min(a.cols, a.G - h0);
    for (int i = threadIdx.x; i < have * (D / 4); i += 64 * NW) {
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
            if (d == 0) red_lse[c] = put_lse(row, mm, ll);
        } else {
            *(f32x4*)(a.part + ((long long)slot * a.cols + c) * D + d) = o;
            if (d == 0) a.part_ml[(long long)slot * a.cols + c] = f32x2{mm, ll};
        }
    }
    if constexpr (SC && ROW) {
        if (lost) return;
        __syncthreads();      // the scores of all waves too
        for (int j = threadIdx.x * 4; j < it.len; j += 64 * NW * 4) {
            Weights next = {};
            next.load(a, kvrow, j + 64 * NW * 4, it.len);
            const float* sp = a.scores + kvrow * a.G * a.cap + j;
#pragma unroll 4
            for (int c = 0; c < a.G; ++c) ws.add(*(const f32x4*)(sp + (long long)c * a.cap), red_lse[c]);
            ws.store();
            ws = next;
        }
    }
}

// The pieces in which a split launch of TW workers a workgroup left a row: `head` of single workers, those of the
// workgroups [ga, gb) that lie in the row, and `tail` of single workers.  none: one worker or workgroup had it all.
struct Pieces {
    int n, head, tail, w0, ga, gb, t, r0, tw, cols, most;
    __device__ __forceinline__ long long slot(int i, int c) const {
        const int mid = gb - ga;
        const int w = min(i < head ? w0 + i : i < head + mid || tail == 0 ? (ga + i - head) * tw : gb * tw + i - head - mid, most);
        return ((long long)w * 2 + (w * t <= r0 ? 1 : 0)) * cols + c;
    }
};
template <int TW>
__device__ __forceinline__ bool pieces_of(const P& a, int b, int rh, int nt, int lane, Pieces& p) {
    int all, before;
    count_tiles(a, b, lane, all, before);
    const int RH = a.Hkv * a.HG;
    all *= RH;
    p.tw = TW;
    p.cols = a.cols;
    p.most = a.groups * TW - 1;      // the last worker: no slot lies behind, if the lengths have changed meanwhile
    p.t = tiles_each(all, a.groups * TW);
    const int T = p.t * TW, r1 = before * RH + rh * nt + nt;
    p.r0 = r1 - nt;
    p.w0 = p.r0 / p.t;
    const int w1 = (r1 - 1) / p.t;
    p.ga = (p.r0 + T - 1) / T;
    p.gb = r1 == all ? (r1 + T - 1) / T : r1 / T;
    if (p.w0 == w1 && p.ga >= p.gb) return false;
    if (p.gb - p.ga == 1 && p.ga * T == p.r0 && r1 <= p.gb * T) return false;
    p.head = p.ga < p.gb ? p.ga * TW - p.w0 : w1 - p.w0 + 1;
    p.tail = p.ga < p.gb ? max(0, w1 + 1 - p.gb * TW) : 0;
    p.n = p.head + max(0, p.gb - p.ga) + p.tail;
    return true;
}

// A row without a tile: zeros, or NaN where the length is none of this table.
template <int D, int DT>
__device__ __forceinline__ void put_empty(const P& a, long long row, bool lost, int t, int threads) {
    for (int d = t; d < D; d += threads) a.o[row * D + d] = (uint16_t)(lost ? (DT == DT_F16 ? 0x7e00 : 0x7fc0) : 0);
    if (t == 0 && a.lse) a.lse[row] = lost ? NAN : -INFINITY;
}

// Joins the pieces of column c of a row by the TEAM threads t: D/4 of them have 4 dims each of a piece, and the
// groups of so many take pieces in turn, 8 in flight.  A team is a wave, or a workgroup (then `red` is LDS for it).
template <int D, int DT, int TEAM>
__device__ __forceinline__ void join_row(const P& a, const Pieces& p, int c, long long row, int t, f32x4* red_o, f32x2* red_ml) {
    constexpr int DV = D / 4, PAR = TEAM / DV, FLY = 8;
    const int d = t % DV, g = t / DV;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    float mm = -INFINITY, ll = 0.f;
    auto lift = [&](float top) {       // the sums so far, relative to top
        const float f = mm == -INFINITY ? 0.f : fast_exp2(mm - top);
        o *= f;
        ll = mm == -INFINITY ? ll : ll * f;
        mm = top;
    };
    for (int i0 = g; i0 < p.n; i0 += PAR * FLY) {
        f32x2 ml[FLY];
        f32x4 x[FLY];
        float top = mm;
#pragma unroll
        for (int j = 0; j < FLY; ++j) {
            const int i = i0 + j * PAR;
            ml[j] = f32x2{-INFINITY, 0.f};
            x[j] = f32x4{0.f, 0.f, 0.f, 0.f};
            if (i < p.n) {
                const long long s = p.slot(i, c);
                ml[j] = a.part_ml[s];
                x[j] = *(const f32x4*)(a.part + s * D + d * 4);
            }
        }
#pragma unroll
        for (int j = 0; j < FLY; ++j) top = fmaxf(top, ml[j][0]);
        lift(top);
#pragma unroll
        for (int j = 0; j < FLY; ++j) add_piece(ml[j], x[j], mm, o, ll);
    }
    if constexpr (TEAM == 64) {
#pragma unroll
        for (int k = DV; k < 64; k <<= 1) {
            const f32x2 ml = {__shfl_xor(mm, k, 64), __shfl_xor(ll, k, 64)};
            f32x4 x;
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = __shfl_xor(o[i], k, 64);
            lift(fmaxf(mm, ml[0]));
            add_piece(ml, x, mm, o, ll);
        }
    } else {
        red_o[t] = o;
        if (d == 0) red_ml[g] = f32x2{mm, ll};
        __syncthreads();
        mm = -INFINITY;
#pragma unroll
        for (int i = 0; i < PAR; ++i) mm = fmaxf(mm, red_ml[i][0]);
        o = f32x4{0.f, 0.f, 0.f, 0.f};
        ll = 0.f;
#pragma unroll
        for (int i = 0; i < PAR; ++i) add_piece(red_ml[i], red_o[i * DV + d], mm, o, ll);
    }
    if (g != 0) return;
    o *= ll == 0.f ? 0.f : 1.0f / ll;
    *(u32x2*)(a.o + row * D + d * 4) = u32x2{pack2<DT>(o[0], o[1]), pack2<DT>(o[2], o[3])};
    if (d == 0 && a.lse) a.lse[row] = lse_of(mm, ll);
}

// The rows that a split launch left in pieces, and those without a tile. A team of TEAM threads a query head.
template <int D, int DT, int NH, int TEAM>
__global__ __launch_bounds__(256) void join_kernel(P a) {
    __shared__ f32x4 red_o[TEAM == 64 ? 1 : 256];
    __shared__ f32x2 red_ml[TEAM == 64 ? 1 : 1024 / D];
    const int lane = threadIdx.x & 63, t = threadIdx.x % TEAM;
    const long long row = (long long)blockIdx.x * (256 / TEAM) + uni(threadIdx.x / TEAM);
    if (row >= (long long)a.B * a.Hkv * a.G) return;
    const int h = (int)(row % (a.Hkv * a.G)), b = (int)(row / (a.Hkv * a.G)), kvh = h / a.G, hg = h % a.G / (16 * NH), c = h % a.G % (16 * NH);
    const int len = a.len[b], nt = tiles_of(len, a.cap);
    Pieces p;
    if (nt == 0) put_empty<D, DT>(a, row, len != 0, t, TEAM);
    else if (pieces_of<kWaves / NH>(a, b, kvh * a.HG + hg, nt, lane, p)) join_row<D, DT, TEAM>(a, p, c, row, t, red_o, red_ml);
}

__host__ __device__ constexpr int weight_chunks(int cap) { return (cap + 1023) / 1024; }

// With weights: the same, and 1024 positions' weights of a kv head a workgroup.  Each workgroup takes the LSE of
// the head's query heads from their pieces itself, and joins the O of every n-th of them, n the workgroups of the
// row, so that one launch does both.
template <int D, int DT, int NH, int TEAM>
__global__ __launch_bounds__(256) void join_weights_kernel(P a) {
    __shared__ f32x4 red_o[TEAM == 64 ? 1 : 256];
    __shared__ f32x2 red_ml[TEAM == 64 ? 1 : 1024 / D];
    __shared__ float l2[64];
    const int tid = threadIdx.x, lane = tid & 63, wave = uni(tid >> 6);
    const unsigned chunks = (unsigned)weight_chunks(a.cap);
    const long long kvrow = blockIdx.x / chunks;     // sequence and kv head
    const int chunk = (int)(blockIdx.x % chunks), b = (int)(kvrow / a.Hkv), kvh = (int)(kvrow % a.Hkv);
    const int len = a.len[b], nt = tiles_of(len, a.cap);
    if (nt == 0) {
        for (int g = chunk; g < a.G; g += (int)chunks) put_empty<D, DT>(a, kvrow * a.G + g, len != 0, tid, 256);
        return;
    }
    const int mine = (len + 1023) / 1024, j = chunk * 1024 + tid * 4;
    if (chunk >= mine) return;
    // the weights and the first heads' scores are on their way while the LSE are joined
    constexpr int AHEAD = 4;
    Weights ws = {};
    ws.load(a, kvrow, j, len);
    const float* sp = a.scores + kvrow * a.G * a.cap + j;
    f32x4 sc[AHEAD];
#pragma unroll
    for (int c = 0; c < AHEAD; ++c)
        if (c < a.G && j < len) sc[c] = *(const f32x4*)(sp + (long long)c * a.cap);
    for (int hg = 0; hg < a.HG; ++hg) {              // up to 64 query heads at a time
        const int g0 = hg * 16 * NH, n = min(a.cols, a.G - g0);
        Pieces p;
        const bool some = pieces_of<kWaves / NH>(a, b, kvh * a.HG + hg, nt, lane, p);
        if (hg) __syncthreads();
        if (some) {
            for (int c = wave; c < n; c += 4) {
                float m = -INFINITY, l = 0.f;
                for (int i = lane; i < p.n; i += 64) {
                    const f32x2 ml = a.part_ml[p.slot(i, c)];
                    const float top = fmaxf(m, ml[0]);
                    if (top == -INFINITY) {
                        l += ml[1];
                    } else {
                        l = (m == -INFINITY ? l : l * fast_exp2(m - top)) + (ml[0] == -INFINITY ? ml[1] : ml[1] * fast_exp2(ml[0] - top));
                        m = top;
                    }
                }
                float top = m;
#pragma unroll
                for (int k = 32; k > 0; k >>= 1) top = fmaxf(top, __shfl_xor(top, k, 64));
                if (m != -INFINITY) l *= fast_exp2(m - top);
#pragma unroll
                for (int k = 32; k > 0; k >>= 1) l += __shfl_xor(l, k, 64);
                if (lane == 0) l2[c] = lse2_of(top, l);
            }
        } else if (tid < n) {
            l2[tid] = a.lse2[kvrow * a.G + g0 + tid];
        }
        __syncthreads();
        if (j < len) {
            if (hg == 0)
#pragma unroll
                for (int c = 0; c < AHEAD; ++c)
                    if (c < n) ws.add(sc[c], l2[c]);
#pragma unroll 4
            for (int c = hg ? 0 : AHEAD; c < n; ++c) ws.add(*(const f32x4*)(sp + (long long)(g0 + c) * a.cap), l2[c]);
        }
        if (!some) continue;
        constexpr int TEAMS = 256 / TEAM;
        for (int c = chunk * TEAMS + uni(tid / TEAM); c < n; c += mine * TEAMS) {
            join_row<D, DT, TEAM>(a, p, c, kvrow * a.G + g0 + c, tid % TEAM, red_o, red_ml);
            if (TEAM > 64) __syncthreads();
        }
    }
    ws.store();
}

// Waves that share a kv head's query heads, 16 each, and the groups of so many heads.
int head_waves(int G) { return G <= 16 ? 1 : G <= 32 ? 2 : 4; }
int head_groups(int G) { return (G + 63) / 64; }
int head_cols(int G) { return G < 64 ? G : 64; }
size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }

// Whether a call runs as one workgroup (of 8 waves) a row, in one launch without pieces: where the longest row that
// the tables can hold is short, and longer where there are rows enough to keep HBM busy, or where the weights
// would need the second launch anyway.  Measured, us of one workgroup a row / split and joined (B, tokens, Hkv, D;
// ragged where B > 1):
//   1, 200, 8, 64: 4.2 / 7.4        1, 500, 8, 128: 6.8 / 7.9         1, 1000, 8, 128: 10.7 / 8.8    1, 2000, 8, 64: 10.4 / 8.4
//   16, 500, 8, 128: 7.6 / 12.0     16, 1000, 8, 128: 14.4 / 16.9     16, 2000, 8, 128: 25.0 / 22.3
//   64, 1000, 8, 128: 33.1 / 37.3   64, 2000, 8, 128: 67.0 / 69.4     128, 1000, 8, 64: 31.1 / 36.9
//   with weights  12, 1000, 4, 64: 9.5 / 16.3     4, 1000, 8, 128: 12.6 / 16.2    12, 2500, 4, 64: 16.4 / 17.7
//                 16, 2000, 8, 128: 28.9 / 28.5   4, 8000, 4, 64: 39 / 14.9
bool by_row(const tkm_attn_kv& kv, int Hq, int add_weights) {
    const double kb = (double)kv.max_pages * kv.page * kv.D * 4 / 1024, rows = (double)kv.B * kv.Hkv;   // K and V of a row
    return Hq / kv.Hkv <= 64 && kb <= (rows >= 512 ? 1280 : add_weights || rows >= 96 ? 704 : 320);
}

int groups_of(const tkm_attn_kv& kv, int Hq) {
    const double most = decode_tiles_most(kv, Hq) * head_waves(Hq / kv.Hkv) / kWaves + 1;
    return most < kGroups ? (int)most : kGroups;
}

int status() { return hipGetLastError() == hipSuccess ? 0 : -1; }

template <int D, int DT, int NH, bool SC>
int run(const P& a, hipStream_t st) {
    const unsigned rows = (unsigned)(a.B * a.Hkv);
    if (!a.groups) {
        hipLaunchKernelGGL((decode_kernel<D, DT, NH, SC, true>), dim3(rows * a.HG), dim3(64 * kRowWaves), 0, st, a);
        return status();
    }
    hipLaunchKernelGGL((decode_kernel<D, DT, NH, SC, false>), dim3((unsigned)a.groups), dim3(64 * kWaves), 0, st, a);
    if (status()) return -1;      // there are no pieces to join
    const unsigned heads = rows * a.G, chunks = (unsigned)weight_chunks(a.cap) * rows;
    const bool waves = heads > 512;      // a wave a query head, or a workgroup
    if (SC && waves)
        hipLaunchKernelGGL((join_weights_kernel<D, DT, NH, 64>), dim3(chunks), dim3(256), 0, st, a);
    else if (SC)
        hipLaunchKernelGGL((join_weights_kernel<D, DT, NH, 256>), dim3(chunks), dim3(256), 0, st, a);
    else if (waves)
        hipLaunchKernelGGL((join_kernel<D, DT, NH, 64>), dim3((heads + 3) / 4), dim3(256), 0, st, a);
    else
        hipLaunchKernelGGL((join_kernel<D, DT, NH, 256>), dim3(heads), dim3(256), 0, st, a);
    return status();
}

template <int D, int DT, int NH>
int run_scores(const P& a, hipStream_t st) {
    return a.scores ? run<D, DT, NH, true>(a, st) : run<D, DT, NH, false>(a, st);
}

template <int D, int DT>
int run_heads(const P& a, hipStream_t st) {
    const int n = head_waves(a.G);
    return n == 1 ? run_scores<D, DT, 1>(a, st) : n == 2 ? run_scores<D, DT, 2>(a, st) : run_scores<D, DT, 4>(a, st);
}

}  // namespace

double decode_tiles_most(const tkm_attn_kv& kv, int Hq) {
    return (double)kv.B * kv.Hkv * head_groups(Hq / kv.Hkv) * kv.max_pages * (kv.page / 32);
}

// (The join's launch without weights has at most 64 threads a query head where these are many, and B * Hq * D at most
// 2^30: it always fits.)
bool decode_fits(const tkm_attn_kv& kv, int Hq, int add_weights) {
    const double rows = (double)kv.B * kv.Hkv;
    if (by_row(kv, Hq, add_weights)) return launch_fits(rows * head_groups(Hq / kv.Hkv), 64 * kRowWaves);
    return !add_weights || launch_fits(rows * weight_chunks(kv.max_pages * kv.page), 256);
}

size_t decode_workspace(const tkm_attn_kv& kv, int Hq, int add_weights) {
    const int G = Hq / kv.Hkv;
    const long long cap = (long long)kv.max_pages * kv.page;
    size_t n = 0;
    if (!by_row(kv, Hq, add_weights)) {
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
    a.groups = by_row(kv, d.Hq, d.add_weights) ? 0 : groups_of(kv, d.Hq);
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
    note_kernels(kDecode | (!a.groups ? 0u : a.scores ? kJoin | kWeights : kJoin));
    return kv.D == 64 ? (kv.dtype == TKM_ATTN_BF16 ? run_heads<64, DT_BF16>(a, st) : run_heads<64, DT_F16>(a, st))
                      : (kv.dtype == TKM_ATTN_BF16 ? run_heads<128, DT_BF16>(a, st) : run_heads<128, DT_F16>(a, st));
}

}  // namespace tkm
