// attn_chunk.hip -- attention of several new tokens a sequence over a paged key-value cache (gfx950).
//
//   row i of sequence b stands at p = len[b] - n[b] + i and sees lo <= j < hi:  s_j = scale <q, k_j>
//   o = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m);  lse = m + ln sum_j exp(s_j - m)
//
// A kv head's query heads share its keys, so that the rows of a tile are (token, query head of the kv head) pairs:
// row r is token r / G, head r % G.  An item is (kv head, sequence, tile of 128 such rows), 32 rows a wave; it walks
// the tiles of 64 tokens that any of its rows sees.  Keys and values move HBM -> LDS by DMA, double-buffered, in the
// cache's own 32 x 32 blocks (attn_kv.h), 64-byte rows whose 16-byte chunks are stored at c ^ (row / 4 % 4): operand
// reads of 16 rows then meet all banks once.  Per tile and wave:
//   S^T = K Q^T        32 tokens x 32 rows an MFMA block; lane = row.  K's tokens are dealt to the block's rows with
//                      bits 2 and 3 swapped, so that the 8 registers of a k-step are 8 consecutive tokens:
//   P^T                takes its place, and goes in 16-bit parts, k-step by k-step, as the B operand to
//   O^T += V^T P^T     whose A operand is 8 consecutive tokens of a dim, one 16-byte read of a V block.
//
// P = 2^(s - m + 8): m moves only when a lane's sum of a tile reaches fp16's largest value (the tile's scores are then
// formed once more), and the 8 keep weights of down to 2^-22 of the row's largest in fp16's normal range.  P goes to the
// second product in parts that hold what decoding (attn_decode.hip) keeps of it, two in fp16 (22 bits) and three in bf16
// (24), so that a row has the same precision in either.  One part in fp16 and two in bf16 lost 2^-11 and 2^-16 of a P, and
// took, on one card, 957 us for 1310 (prompts in fp16, limited by the products' power), and in bf16 321 for 392 (a mixed
// step), 117 for 131 (13 rows over 131000 tokens), 61.5 for 71 (windows, 64 dims).
//
// Splitting: all items' tiles are numbered in one line, kv head after kv head, and every workgroup takes an equal
// share, whatever the lengths are, which are read on the device: a first launch of one workgroup lists the items of a
// kv head, the place where each share begins, and the items that no one workgroup has whole.  These leave pieces in
// the workspace, which a third launch joins in the order of the tokens: results do not depend on timing.  Where items
// are short, or fill the card, a workgroup has one, and there is one launch.  (Shares weighted by what a tile has of
// rows were slower: on a full card a tile took 2 us, with fewer parts of P, be it one row's, from HBM, or 128 rows', whose
// keys are in L2.)
//
// What bounds it: for few rows HBM and, between two tiles, the products of the one or two waves that have rows (13 tokens,
// 32 heads of 128 on 8, about 131000: 116 us for 537 MB, 4.6 TB/s; listing and joining 15 more); for prompts of 128 dims
// products and vector instructions one after the other (52 and 39% of the clocks at 1.84 GHz; 849 GFLOP, 1281 with the second
// product's parts, in 1270 to 1310 us); at 64 dims the issue of exponentials, sums and parts, three waves a SIMD, and a
// part's beginning and end.
//
// 0 times an infinity or NaN is NaN, also where P is 0 because its row does not see the token, and an infinity times a part
// of P that is 0 or negative is NaN where the whole of P makes it infinite.  So a tile that an item's rows do not see alike
// is searched for such values in LDS, where they become 0.  If there were any, or sums have become NaN, the workgroup
// goes through its tiles once more, searches all of them, and adds what it finds, kept as a bit each, to the sums of
// the rows that see them: an infinity, or NaN where P is 0, as in attn_decode.hip.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "attn_common.h"
#include "attn_kv.h"
#include "attn_launch.h"
#include "attn_scan.h"

namespace tkm {
namespace {

constexpr int BM = 128;           // rows of an item
constexpr int BN = 64;            // tokens of a tile
constexpr int kWaves = 4;
// Three or two workgroups on each compute unit (5 prompts in windows of 1024, 12 heads of 64: 71 and 89 us).
constexpr int workers_at(int D) { return D == 64 ? 768 : 512; }
constexpr float kLift = 8.0f;
constexpr float kSumMax = 65504.0f;
constexpr float kLn2 = 0.69314718055994531f;

// An item of a kv head: rows [r0, rows) of sequence b, up to BM of them, which begins at row row0 of the call and at
// position pos of len; the tiles [x, y) of tokens that they see, of which all see [alike, alike_end) whole; and its
// place in the head's line.
struct Item {
    int b, r0, row0, rows, pos, len, x, y, alike, alike_end;
    int64_t at;
};
// Where a worker's share begins: tile `tile` of item e of kv head h, and the tiles that are its; a kv head has `items`.
struct Start {
    int h, e, tile, items;
    int64_t tiles;
};
// An item of which n workers have pieces, from worker w on: `rows` rows of kv head h, the first of them row r0 of a
// sequence whose first token is row `row0` of the call.
struct Joint {
    int h, row0, r0, rows, w, n, pad[2];
};

struct C {   // kernel arguments
    const uint16_t *k, *v;
    const int32_t *table, *len;
    const uint16_t* q;
    const int32_t *row_start, *n_new;
    uint16_t* o;
    float* lse;
    Start* starts;     // of the workers
    Joint* joints;     // n is 0 behind the last
    Item* items;       // of a kv head, up to `most`
    float* part;       // pieces: [slot][BM][D] unnormalised O, then [slot][BM] (m, l)
    float2* part_ml;
    long long q_stride;
    int B, Hkv, G, num_pages, page_shift, max_pages, cap, rows, causal, window;
    uint32_t per_g;    // a number is divided by G by this and a shift
    int g_shift;
    int each;          // rows of a sequence where n_new is NULL
    int workers;       // 0: a workgroup an item
    int most;          // items that the rows can make, if no two sequences have one of them; more are passed over
    float sl2;         // scale * log2(e)
};

__device__ __forceinline__ int uni(int v) { return __builtin_amdgcn_readfirstlane(v); }
// An element of an array that no kernel of the launch writes, at a wave-uniform index: a scalar load.
__device__ __forceinline__ int fixed(const int32_t* p, long long i) {
    return *((const __attribute__((address_space(4))) int32_t*)(uintptr_t)p + i);
}
__device__ __forceinline__ Item fixed_item(const Item* p) {
    const auto* q = (const __attribute__((address_space(4))) int32_t*)(uintptr_t)p;
    return Item{q[0], q[1], q[2], q[3], q[4], q[5], q[6], q[7], q[8], q[9], 0};
}
__device__ __forceinline__ Start fixed_start(const Start* p) {
    const auto* q = (const __attribute__((address_space(4))) int32_t*)(uintptr_t)p;
    return Start{q[0], q[1], q[2], q[3], *(const __attribute__((address_space(4))) int64_t*)(uintptr_t)&p->tiles};
}
__device__ __forceinline__ Joint fixed_joint(const Joint* p) {
    const auto* q = (const __attribute__((address_space(4))) int32_t*)(uintptr_t)p;
    return Joint{q[0], q[1], q[2], q[3], q[4], q[5], {}};
}
template <int DT>
constexpr uint32_t kInf = DT == DT_BF16 ? 0x7f80u : 0x7c00u;
// Two P as 16-bit parts, each what the ones before leave, rounded: the words w[0], w[1], ..  Two parts in fp16 hold 22
// bits, three in bf16 the 24 of fp32 (as in attn_decode.hip).  What a part leaves is exact: by a mixed-precision fma in
// fp16, which also rounds the last part, by a dot product with (-1, 0) or (0, -1) in bf16: 3 and 7 instructions a pair (8
// and 13 where the compiler converts the parts back).
template <int DT>
constexpr int kParts = DT == DT_BF16 ? 3 : 2;
template <int DT>
__device__ __forceinline__ void split_p(float x, float y, uint32_t (&w)[kParts<DT>]) {
    // constants that the compiler does not know: it would make a subtraction of -1, and in bf16 has the wrong half
    float minus = -1.0f;
    uint32_t of_x = 0xbf80u, of_y = 0xbf800000u;
    if constexpr (DT == DT_BF16) asm("" : "+s"(of_x), "+s"(of_y));
    else asm("" : "+s"(minus));
#pragma unroll
    for (int i = 0; i < kParts<DT>; ++i) {
        w[i] = pack2<DT>(x, y);
        if (i + 1 == kParts<DT>) break;
        asm("" : "+v"(w[i]));      // both from the one word
        if constexpr (DT == DT_BF16) {
            const bf16x2 h = __builtin_bit_cast(bf16x2, w[i]);
            x = __builtin_amdgcn_fdot2_f32_bf16(h, __builtin_bit_cast(bf16x2, of_x), x, false);
            y = __builtin_amdgcn_fdot2_f32_bf16(h, __builtin_bit_cast(bf16x2, of_y), y, false);
        } else {
            const f16x2 h = as_f16x2(w[i]);
            x = __builtin_fmaf((float)h[0], minus, x);
            y = __builtin_fmaf((float)h[1], minus, y);
        }
    }
}
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));

// A sequence's rows: `n` of them from row `row0` on, the first at position `pos`; len -1 if it lies outside the table.
struct Seq {
    int n, row0, pos, len;
};
template <bool FIXED = false>
__device__ __forceinline__ Seq seq_of(const C& a, int b) {
    auto get = [&](const int32_t* p) {
        if constexpr (FIXED) return fixed(p, b);
        else return p[b];
    };
    Seq s;
    s.row0 = a.row_start ? get(a.row_start) : b * a.each;
    int n = a.n_new ? get(a.n_new) : a.each;
    if (!a.row_start) n = min(n, a.each);      // the next sequence's rows begin there
    s.len = get(a.len);
    if ((unsigned)s.len > (unsigned)a.cap) s.len = -1;
    s.n = s.row0 < 0 || s.row0 >= a.rows ? 0 : max(0, min(n, a.rows - s.row0));
    s.pos = s.len - max(n, 0);       // above -2^31: neither is below -1, nor n above 2^31 - 1
    return s;
}
// r / G of r in [0, 2^31): per_g is ceil(2^(31 + g_shift) / G) with 2^g_shift >= G, so G per_g exceeds the power by less
// than G, and r per_g / 2^(31 + g_shift) exceeds r / G by less than 1 / G.
__device__ __forceinline__ int over_g(const C& a, int r) { return (int)(__umulhi(2u * (uint32_t)r, a.per_g) >> a.g_shift); }

// The positions that the row of token i sees, of a sequence whose first is at pos of len: [lo, hi).
__device__ __forceinline__ int2 seen_by(const C& a, int pos, int len, int i) {
    if (!a.causal) return int2{0, max(len, 0)};
    const int p = pos + i;
    // windows reach up to 2^31 - 1, and p below 0 where a sequence has more rows than tokens
    return int2{a.window && p >= a.window ? p - a.window + 1 : 0, max(0, min(p + 1, len))};
}
// Item t of a sequence.
__device__ __forceinline__ Item item_of(const C& a, const Seq& s, int b, int t) {
    Item e{b, t * BM, s.row0, s.n * a.G, s.pos, s.len, 0, 0, 0, 0, 0};
    const int2 first = seen_by(a, s.pos, s.len, over_g(a, e.r0)), last = seen_by(a, s.pos, s.len, over_g(a, max(min(e.r0 + BM, e.rows) - 1, 0)));
    if (first.x < last.y) {
        e.x = first.x / BN;
        e.y = (last.y + BN - 1) / BN;
    }
    e.alike = (last.x + BN - 1) / BN;
    e.alike_end = first.y / BN;
    return e;
}

constexpr int TL = 1024;

__device__ __forceinline__ int64_t div_up(int64_t x, int64_t y) { return (x + y - 1) / y; }

// Lists the items of a kv head, sequence after sequence, and their places in its line; then the workers' shares.  One
// workgroup.
__global__ __launch_bounds__(TL) void chunk_items_kernel(C a) {
    __shared__ Scan<TL> lds;
    __shared__ int64_t place[TL];      // of the first items
    int64_t before = 0, items = 0;
    for (int c = 0; c < a.B; c += TL) {
        const int b = c + threadIdx.x;
        const int rows = b < a.B ? seq_of(a, b).n * a.G : 0;
        int64_t all, sum;
        lds.end[threadIdx.x] = (int)min(lds.sum(0, (rows + BM - 1) / BM, all), (int64_t)INT_MAX);
        all = min(all, a.most - items);
        __syncthreads();
        for (int64_t k0 = 0; k0 < all; k0 += TL) {
            const int k = (int)k0 + threadIdx.x;
            Item e{};
            int tiles = 0;
            if (k < all) {
                const int i = first_above(lds.end, TL, k);
                const int b = c + i;
                e = item_of(a, seq_of(a, b), b, k - (i ? lds.end[i - 1] : 0));
                tiles = max(1, e.y - e.x);       // an item that sees nothing still has outputs
            }
            e.at = before + lds.sum(1, tiles, sum) - tiles;
            if (k < all) {
                a.items[items + k] = e;
                if (items + k < TL) place[items + k] = e.at;
            }
            before += sum;
            __syncthreads();
        }
        items += all;
        __syncthreads();
    }
    const int64_t all = before * a.Hkv, each = div_up(all, a.workers);
    auto begin = [&](int64_t e) { return e < TL ? place[e] : a.items[e].at; };
    int64_t joints = 0;
    for (int w0 = 0; w0 < a.workers; w0 += TL) {
        const int w = w0 + threadIdx.x;
        Start st{0, 0, 0, (int)items, 0};
        Joint j{0, 0, 0, 0, w - 1, 0, {}};
        if (w < a.workers && w * each < all) {
            const int64_t at = w * each % before;
            st.h = (int)(w * each / before);
            st.tiles = min(each, all - w * each);
            int lo = 0, hi = (int)items - 1;          // the last item that begins at or before `at`
            while (lo < hi) {
                const int mid = (lo + hi + 1) >> 1;
                if (begin(mid) <= at) lo = mid;
                else hi = mid - 1;
            }
            st.e = lo;
            st.tile = (int)(at - begin(lo));
            if (st.tile > 0 && st.tile <= each) {     // the first share that begins inside the item
                const Item it = a.items[lo];
                const int64_t left = (lo + 1 < items ? begin(lo + 1) : before) - at;
                j.h = st.h;
                j.row0 = it.row0;
                j.r0 = it.r0;
                j.rows = min(it.rows - it.r0, BM);
                j.n = 1 + (int)div_up(left, each);
            }
        }
        int64_t sum;
        const int64_t to = joints + lds.sum(w0 / TL % 2, j.n > 0, sum);
        if (w < a.workers) a.starts[w] = st;
        if (j.n > 0) a.joints[to - 1] = j;
        joints += sum;
    }
    for (int64_t i = joints + threadIdx.x; i < a.workers; i += TL) a.joints[i].n = 0;
}

// Row r of an item: its row of o and lse, and its head.
__device__ __forceinline__ long long out_row(const C& a, int row0, int h, int r) {
    const int i = over_g(a, r);
    return ((long long)(row0 + i) * a.Hkv + h) * a.G + (r - i * a.G);
}

// The arguments of the kernel that runs, read where they are used: those of its whole life would not fit into the scalar
// registers, and every tile would move some of them from and to vector registers.
__device__ __forceinline__ const C& arguments() {
    auto p = (const __attribute__((address_space(4))) C*)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(p));
    return *(const C*)p;
}

template <int D, int DT>
__global__ __launch_bounds__(64 * kWaves) __attribute__((amdgpu_waves_per_eu(D == 64 ? 3 : 2, D == 64 ? 3 : 2))) void chunk_kernel(C args) {
    constexpr int KS = D / 16, NDB = D / 32, PKS = BN / 16;
    constexpr int HALF = D * 64;               // bytes of 32 tokens of K or V
    constexpr int TILE = 2 * HALF;
    constexpr int NI = TILE / 1024 / kWaves;   // DMA requests of a wave, a tile of K or V
    __shared__ __attribute__((aligned(1024))) char smem[2][2][TILE];    // [K, V][buffer]
    __shared__ uint2 odds[2][D];               // [half][dim]: bits of the tokens whose value is inf or NaN, -inf or NaN
    __shared__ int votes[kWaves];

    const int lane = threadIdx.x & 63, wave = uni(threadIdx.x >> 6), l32 = lane & 31, hi = lane >> 5;
    // consecutive shares on one XCD, whose L2 their keys and values then share
    const int workers = args.workers;
    const int place = workers % 8 || !workers ? blockIdx.x : (int)(blockIdx.x % 8 * (workers / 8) + blockIdx.x / 8);
    Start st{(int)blockIdx.z, 0, 0, 0, 0};
    if (workers) {
        st = fixed_start(&args.starts[place]);
        if (st.tiles == 0) return;
    }
    int h = st.h, e = st.e, from = st.tile;
    int64_t left = st.tiles;

    const uint32_t lds0 = lds_addr(smem);
    // DMA: this wave's requests of a tile are 1024 bytes each, all of one half of 32 tokens
    const int my_half = wave / (kWaves / 2);
    uint32_t dma_v[NI];
#pragma unroll
    for (int i = 0; i < NI; ++i) {
        const int c = ((wave % (kWaves / 2)) * NI + i) * 64 + lane;      // chunk of the half
        dma_v[i] = (uint32_t)(c / 4 * 64 + (((c % 4) ^ (c / 16 % 4)) << 4));
    }
    const uint32_t dma_at = lds0 + (uint32_t)(wave * NI * 1024);
    // operand reads: chunks (ks % 2) * 2 + hi of a 64-byte row
    const int tok = (l32 & 19) | (l32 & 4) << 1 | (l32 & 8) >> 1;        // bits 2 and 3 swapped
    int koff[2], voff[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        koff[j] = tok * 64 + (((j * 2 + hi) ^ (tok / 4 % 4)) << 4);
        voff[j] = l32 * 64 + (((j * 2 + hi) ^ (l32 / 4 % 4)) << 4);
    }

    do {
        // ---- the item, and this workgroup's share of its tiles
        const C& a = arguments();
        const Item it = workers ? fixed_item(&a.items[e]) : item_of(a, seq_of<true>(a, blockIdx.y), blockIdx.y, blockIdx.x);
        const int R = it.rows, r0 = it.r0;
        if (r0 >= R) return;              // a workgroup an item: the sequence has fewer
        const int all = max(1, it.y - it.x);
        if (!workers) left = all;
        const int mine = (int)min(left, (int64_t)(all - from)), ta = it.x + from, te = min(ta + mine, it.y);
        const bool whole = mine == all;

        // this lane's row; those behind the sequence's rows act as its last
        const int r = r0 + wave * 32 + l32;
        const bool valid = r < R;
        const int first = r0 + wave * 32, final = min(first + 31, R - 1);
        const bool active = first < R;
        const int2 seen = seen_by(a, it.pos, it.len, over_g(a, min(r, R - 1)));
        // tiles in [p0, p1) need no mask in this wave, those in [n0, n1) hold a token that one of its rows sees
        int p0 = 0, p1 = 0, n0 = 0, n1 = 0;
        if (active) {
            const int2 x = seen_by(a, it.pos, it.len, over_g(a, first)), y = seen_by(a, it.pos, it.len, over_g(a, final));
            p0 = (y.x + BN - 1) / BN;
            p1 = x.y / BN;
            n0 = x.x / BN;
            n1 = (y.y + BN - 1) / BN;
        }
        u32x4 qf[KS];
        {
            const int i = over_g(a, r);
            const uint16_t* qp = a.q + (it.row0 + i) * a.q_stride + (long long)(h * a.G + (r - i * a.G)) * D + hi * 8;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) qf[ks] = valid ? ld_global16(qp + ks * 16) : u32x4{0u, 0u, 0u, 0u};
        }
        f32x16 o[NDB];
#pragma unroll
        for (int db = 0; db < NDB; ++db) o[db] = f32x16{};
        float m = -INFINITY, lsum = 0.f;     // m less the lift, log2 units
        bool bad = it.len < 0;

        // pages of a tile's halves, fetched a tile ahead
        const int half_bits = a.page_shift - 5, last_page = a.max_pages - 1, num_pages = a.num_pages, Hkv = a.Hkv;
        const int32_t* pages = a.table + (long long)it.b * a.max_pages;
        const char *keys = (const char*)a.k, *values = (const char*)a.v;
        const float sl2 = a.sl2;
        auto page_of = [&](int t, int x) { return fixed(pages, min((t * 2 + x) >> half_bits, last_page)); };
        int pg[2];
        auto fetch = [&](int t) {
            pg[0] = page_of(t, 0);
            pg[1] = page_of(t, 1);
        };
        auto issue = [&](int t, int buf) __attribute__((always_inline)) {
            int page[2];
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                page[x] = pg[x];
                const int from = t * BN + x * 32;
                if ((unsigned)page[x] >= (unsigned)num_pages) {      // page 0 in its place; rows that see it become NaN
                    page[x] = 0;
                    bad |= from < seen.y && from + 32 > seen.x;
                }
            }
            if (t * BN + my_half * 32 < it.len) {
                const int half = t * 2 + my_half;
                const long long sub = (((long long)(my_half ? page[1] : page[0]) * Hkv + h) << half_bits) + (half & ((1 << half_bits) - 1));
                dma16_rows(make_rsrc(keys + sub * HALF, HALF), dma_at + (uint32_t)(buf * TILE), dma_v);
                dma16_rows(make_rsrc(values + sub * HALF, HALF), dma_at + (uint32_t)((2 + buf) * TILE), dma_v);
            }
        };
        // Whether a thread of the workgroup has it.  The next question comes behind a barrier.
        auto any_of = [&](bool mine) {
            mine = __any(mine);
            if (lane == 0) votes[wave] = mine;
            __syncthreads();
            int all = 0;
#pragma unroll
            for (int w = 0; w < kWaves; ++w) all |= votes[w];
            return uni(all) != 0;
        };
        // Values of tokens behind the sequence's last become 0, for what is there may be anything, and infinities and
        // NaN, whose bits are left in `odds`.  True if there were any of these.  `me`: this thread.
        auto search = [&](int t, int buf, int me) __attribute__((always_inline)) {
            const int left = it.len - t * BN;
            bool any = false;
            for (int i = me; i < 2 * D; i += 64 * kWaves) {         // rows of 32 tokens of one dim
                char* row = smem[1][buf] + i * 64;
                const int from = i < D ? 0 : 32;
                u16x2 most = {0, 0};
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    u32x4* p = (u32x4*)(row + ((c ^ (i / 4 % 4)) << 4));
                    u32x4 x = *p;
                    if (left < BN) {
#pragma unroll
                        for (int w = 0; w < 4; ++w) {
                            const int j = from + c * 8 + 2 * w;
                            x[w] &= (j < left ? 0xffffu : 0u) | (j + 1 < left ? 0xffff0000u : 0u);
                        }
                        *p = x;
                    }
#pragma unroll
                    for (int w = 0; w < 4; ++w) most = __builtin_elementwise_max(most, __builtin_bit_cast(u16x2, x[w] & 0x7fff7fffu));
                }
                uint2 bits = {0u, 0u};
                if (max(most[0], most[1]) >= kInf<DT>) {
                    any = true;
#pragma unroll 1
                    for (int j = 0; j < 32; ++j) {
                        uint16_t* p = (uint16_t*)(row + ((j / 8 ^ (i / 4 % 4)) << 4)) + j % 8;
                        const uint32_t x = *p, e = x & 0x7fffu;
                        if (e < kInf<DT>) continue;
                        if (x != (kInf<DT> | 0x8000u)) bits.x |= 1u << j;
                        if (x != kInf<DT>) bits.y |= 1u << j;
                        *p = 0;
                    }
                }
                odds[i / D][i % D] = bits;
            }
            return any_of(any);
        };
        f32x16 sr[2];
        // In the second walk: the values that `search` took out, for the rows that see them; NaN where P is 0.  Of numbers
        // of its own, as that walk's search: what is formed of a thread's place would keep registers in the first walk (at
        // 64 dims the products' operands were then read one by one, 1.14 us a tile for 1.01).
        auto add_odd = [&](int t) __attribute__((always_inline)) {
            uint32_t sees[2], none[2];
            int hi = lane >> 5;
            asm volatile("" : "+v"(hi));
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const int to = min(max(seen.y - t * BN - x * 32, 0), 32), from = min(max(seen.x - t * BN - x * 32, 0), 32);
                sees[x] = (uint32_t)((1ull << to) - 1) & ~(uint32_t)((1ull << from) - 1);
                none[x] = 0;
#pragma unroll
                for (int i = 0; i < 16; ++i) none[x] |= sr[x][i] == 0.f ? 1u << ((i >> 3) * 16 + (i & 7)) : 0u;
                none[x] <<= hi * 8;
                none[x] = sees[x] & (none[x] | (uint32_t)__shfl_xor((int)none[x], 32, 64));      // the other half's tokens
            }
#pragma unroll
            for (int db = 0; db < NDB; ++db)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int d = db * 32 + i / 4 * 8 + hi * 4 + i % 4;
                    const uint2 a0 = odds[0][d], a1 = odds[1][d];
                    const uint32_t lost = ((a0.x | a0.y) & none[0]) | ((a1.x | a1.y) & none[1]);
                    if (lost | (a0.x & sees[0]) | (a1.x & sees[1])) o[db][i] += INFINITY;
                    if (lost | (a0.y & sees[0]) | (a1.y & sees[1])) o[db][i] -= INFINITY;
                    __builtin_amdgcn_sched_barrier(0);       // it is seldom run, and is to take few registers
                }
        };

        auto scores = [&](int buf) __attribute__((always_inline)) {
#pragma unroll
            for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                for (int kb = 0; kb < 2; ++kb) {
                    const u32x4 x = ld_lds16((const uint16_t*)(smem[0][buf] + kb * HALF + ks / 2 * 2048 + koff[ks & 1]));
                    sr[kb] = mfma32<DT>(x, qf[ks], ks == 0 ? f32x16{} : sr[kb]);
                }
            if constexpr (DT == DT_F16) sched_reads_mfma<2 * KS, 1, 4>();      // drafts of 64 dims 13.85 -> 13.67 us; in bf16 slower
        };
        // register x of block kb is token kb * 32 + x / 8 * 16 + hi * 8 + x % 8
        auto mask = [&](int t) __attribute__((always_inline)) {
            const int up = seen.y - t * BN - hi * 8, down = seen.x - t * BN - hi * 8;
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                for (int x = 0; x < 16; ++x) {
                    const int j = kb * 32 + (x >> 3) * 16 + (x & 7);
                    if (j >= up || j < down) sr[kb][x] = -INFINITY;
                }
        };
        // P in the scores' place
        auto expo = [&](float ref) __attribute__((always_inline)) {
            float sum = 0.f;
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                for (int x = 0; x < 16; ++x) {
                    sr[kb][x] = fast_exp2(__builtin_fmaf(sr[kb][x], sl2, -ref));
                    sum += sr[kb][x];
                }
            return sum;
        };
        // the parts of P of a k-step
        constexpr int NP = kParts<DT>;
        auto parts = [&](int ks, u32x4 (&pr)[NP]) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int x = (ks & 1) * 8 + 2 * i;
                uint32_t w[NP];
                split_p<DT>(sr[ks >> 1][x], sr[ks >> 1][x + 1], w);
#pragma unroll
                for (int j = 0; j < NP; ++j) pr[j][i] = w[j];
            }
        };
        auto tile = [&](int t, int buf) __attribute__((always_inline)) {
            auto masked = [&](int t, int buf) __attribute__((always_inline)) {
                scores(buf);
                if (t < p0 || t >= p1) mask(t);
            };
            masked(t, buf);
            float sum = INFINITY;
            bool move = __any(m == -INFINITY);                         // m is not set yet in an item's first tile
            if (!move) {
                sum = expo(m);
                if (__builtin_expect(__any(!(sum < kSumMax)), 0)) {    // the scores once more, P having taken their place
                    int again = t, from = buf;
                    asm volatile("" : "+s"(again), "+s"(from));        // and not what the compiler would keep of the first ones
                    masked(again, from);
                    move = true;
                }
            }
            if (__builtin_expect(move, 0)) {
                float v = sr[0][0];
#pragma unroll
                for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                    for (int x = kb ? 0 : 1; x < 16; ++x) v = fmaxf(v, sr[kb][x]);
                const float mn = fmaxf(m, half_max(v) * sl2 - kLift);
                const float f = m == -INFINITY ? 0.f : fast_exp2(m - mn);      // nothing is there to be scaled if m is not set
                lsum *= f;
#pragma unroll
                for (int db = 0; db < NDB; ++db) o[db] *= f;
                m = mn;
                sum = expo(m == -INFINITY ? 0.f : m);
            }
            lsum += sum;
            u32x4 pr[2][NP];
            parts(0, pr[0]);
#pragma unroll
            for (int ks = 0; ks < PKS; ++ks) {
                if (ks + 1 < PKS) parts(ks + 1, pr[(ks + 1) & 1]);
#pragma unroll
                for (int db = 0; db < NDB; ++db) {
                    const u32x4 x = ld_lds16((const uint16_t*)(smem[1][buf] + ks / 2 * HALF + db * 2048 + voff[ks & 1]));
#pragma unroll
                    for (int j = 0; j < NP; ++j) o[db] = mfma32<DT>(x, pr[ks & 1][j], o[db]);
                }
            }
        };

        // ---- the walk: tile t + 1 comes while t is worked on.  True if infinities or NaN were found (and, but for ODD,
        // left out).
        auto walk = [&](auto Odd) __attribute__((always_inline)) {
            constexpr bool ODD = decltype(Odd)::value;
            bool odd = false;
            if (ta < te) {
                fetch(ta);
                issue(ta, 0);
                if (ta + 1 < te) fetch(ta + 1);
            }
            wait_dma();
            __syncthreads();
            for (int t = ta; t < te; ++t) {
                const int buf = (t - ta) & 1;
                int me = threadIdx.x;
                if constexpr (ODD) asm volatile("" : "+v"(me));
                if (ODD || t < it.alike || t >= it.alike_end) odd |= search(t, buf, me);
                if (t + 1 < te) {
                    issue(t + 1, buf ^ 1);
                    if (t + 2 < te) fetch(t + 2);
                }
                if (t >= n0 && t < n1) {
                    tile(t, buf);
                    if constexpr (ODD) add_odd(t);
                }
                wait_dma();
                __syncthreads();
            }
            return odd;
        };
        bool odd = walk(std::false_type{}), lost = false;
#pragma unroll
        for (int db = 0; db < NDB; ++db)
#pragma unroll
            for (int i = 0; i < 16; i += 2) lost |= __builtin_isunordered(o[db][i], o[db][i + 1]);
        if (__builtin_expect(any_of(odd || (lost && valid && lsum == lsum)), 0)) {
#pragma unroll
            for (int db = 0; db < NDB; ++db) o[db] = f32x16{};
            m = -INFINITY;
            lsum = 0.f;
            walk(std::true_type{});
        }

        // ---- out
        const C& z = arguments();
        float l = half_sum(lsum);
        if (bad) l = NAN;
        if (whole) {
            if (valid) {
                const long long row = out_row(z, it.row0, h, r);
                const float inv = l == 0.f ? 0.f : 1.0f / l;
                uint16_t* orow = z.o + row * D;
#pragma unroll
                for (int db = 0; db < NDB; ++db)
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        const u32x2 w = {pack2<DT>(o[db][g * 4] * inv, o[db][g * 4 + 1] * inv), pack2<DT>(o[db][g * 4 + 2] * inv, o[db][g * 4 + 3] * inv)};
                        *(u32x2*)(orow + db * 32 + g * 8 + hi * 4) = w;
                    }
                if (z.lse && hi == 0) z.lse[row] = l > 0.f ? m * kLn2 + logf(l) : l == 0.f ? -INFINITY : NAN;
            }
        } else if (valid) {
            const long long slot = (long long)place * 2 + (from == 0 ? 1 : 0);
            float* p = z.part + (slot * BM + (r - r0)) * D;
#pragma unroll
            for (int db = 0; db < NDB; ++db)
#pragma unroll
                for (int g = 0; g < 4; ++g)
                    *(f32x4*)(p + db * 32 + g * 8 + hi * 4) = f32x4{o[db][g * 4], o[db][g * 4 + 1], o[db][g * 4 + 2], o[db][g * 4 + 3]};
            if (hi == 0) z.part_ml[slot * BM + (r - r0)] = float2{m, l};
        }
        left -= mine;
        from = 0;
        if (++e == st.items) {
            e = 0;
            ++h;
        }
    } while (left > 0);
}

template <int D, int DT>
__device__ __forceinline__ void put_joined(const C& a, const Joint& it, int r, int d, f32x4 o, float m, float l) {
    const float inv = l == 0.f ? 0.f : 1.0f / l;
    const long long row = out_row(a, it.row0, it.h, it.r0 + r);
    *(u32x2*)(a.o + row * D + d) = u32x2{pack2<DT>(o[0] * inv, o[1] * inv), pack2<DT>(o[2] * inv, o[3] * inv)};
    if (a.lse && d == 0) a.lse[row] = l > 0.f ? m * kLn2 + logf(l) : l == 0.f ? -INFINITY : NAN;
}

// Joins the pieces of the items that several workers shared, `each` rows a workgroup.  Few pieces: a row for each D / 4
// lanes, whose loads are all under way at once.  Else a wave has a row: each lane weighs a piece, of 64 at a time, and
// has four dims of every (256 / D)th.
template <int D, int DT>
__global__ __launch_bounds__(256) void chunk_join_kernel(C a, int each) {
    constexpr int LANES = D / 4, EACH = 64 / LANES, FEW = 4;
    const Joint it = fixed_joint(&a.joints[blockIdx.x]);
    const int first = (int)blockIdx.y * each, end = min(first + each, it.rows);
    if (it.n == 0 || first >= end) return;
    const int lane = threadIdx.x & 63, wave = uni(threadIdx.x >> 6), d = lane % LANES * 4;
    // the first worker's piece is of the item that its share ends with, the others' of the one that theirs begin with
    auto slot = [&](int i, int r) { return ((long long)(it.w + i) * 2 + (i ? 0 : 1)) * BM + r; };
    // a piece without a finite score has nothing but perhaps a NaN in its sum
    auto weight = [](float2 ml, float m) { return ml.x == -INFINITY ? 0.f : fast_exp2(ml.x - m); };
    if (it.n <= FEW) {
        for (int r = first + wave * EACH + lane / LANES; r < end; r += 4 * EACH) {
            float2 ml[FEW];
            f32x4 x[FEW], o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < FEW; ++i) {
                const long long from = slot(min(i, it.n - 1), r);
                ml[i] = a.part_ml[from];
                x[i] = *(const f32x4*)(a.part + from * D + d);
            }
            float m = ml[0].x, l = 0.f;
#pragma unroll
            for (int i = 1; i < FEW; ++i) m = fmaxf(m, ml[i].x);
#pragma unroll
            for (int i = 0; i < FEW; ++i) {
                if (i >= it.n) break;
                const float f = weight(ml[i], m);
                l += ml[i].x == -INFINITY ? ml[i].y : f * ml[i].y;
                o += f * x[i];
            }
            put_joined<D, DT>(a, it, r, d, o, m, l);
        }
        return;
    }
    for (int r = first + wave; r < end; r += 4) {
        float m = -INFINITY;
        for (int i = lane; i < it.n; i += 64) m = fmaxf(m, a.part_ml[slot(i, r)].x);
#pragma unroll
        for (int x = 32; x; x >>= 1) m = fmaxf(m, __shfl_xor(m, x, 64));
        f32x4 o = {0.f, 0.f, 0.f, 0.f};
        float l = 0.f;
        for (int i0 = 0; i0 < it.n; i0 += 64) {
            float f = 0.f;
            if (i0 + lane < it.n) {
                const float2 ml = a.part_ml[slot(i0 + lane, r)];
                f = weight(ml, m);
                l += ml.x == -INFINITY ? ml.y : f * ml.y;
            }
            const int n = min(64, it.n - i0);
            for (int i = 0; i < n; i += 4 * EACH) {
                f32x4 x[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) x[k] = *(const f32x4*)(a.part + slot(i0 + min(i + k * EACH + lane / LANES, n - 1), r) * D + d);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float w = __shfl(f, i + k * EACH + lane / LANES, 64);      // 0 behind the last
                    if (i + k * EACH + lane / LANES < n) o += w * x[k];
                }
            }
        }
#pragma unroll
        for (int x = 32; x; x >>= 1) l += __shfl_xor(l, x, 64);
#pragma unroll
        for (int x = 32; x >= LANES; x >>= 1)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[i] += __shfl_xor(o[i], x, 64);
        if (lane < LANES) put_joined<D, DT>(a, it, r, d, o, m, l);
    }
}

// The most items that a sequence and that a kv head can have.
long long items_each(const tkm_attn_kv& kv, int rows, int Hq) { return ((long long)rows * (Hq / kv.Hkv) + BM - 1) / BM; }
long long items_most(const tkm_attn_kv& kv, int rows, int Hq) { return items_each(kv, rows, Hq) + std::min<long long>(kv.B, rows); }

// A workgroup an item, in one launch, of a grid laid out for all rows being one sequence's:
//   where no item has more than 10 tiles, which take a lone workgroup about 1.1 us each (kernels, one launch or three: 4
//     times 5 rows over up to 300 tokens 12 and 16 us, 500 14 and 16, 900 21 and 16);
//   where full items are workgroups enough for the card and the longest, by the table or the window, has a 16th as
//     many tiles, and at most 32 (32 heads of 128, fp16, 4 prompts of up to 500 tokens 35 and 56 us, 1000 80 and 99, 1900
//     214 and 236; 12 heads of 64, bf16, 5 prompts in windows of 256 38 and 54, 1024 75 and 81, 2048 126 and 124; but 64 rows
//     over 990, 33 and 29).
// What sequences hold is known to the device alone: the same 4 prompts of 500 take the three launches, 55 us for 33 a call,
// where the tables could hold 131072 tokens.
constexpr long long kFewTiles = 10, kFewItems = 1024, kMoreTiles = 32, kMoreItems = 16384, kFill = 16;

bool item_each(const tkm_attn_kv& kv, int rows, int Hq, int window) {
    const long long G = Hq / kv.Hkv, table = (long long)kv.max_pages * kv.page, seen = window + (BM + G - 1) / G + BN;
    const long long tiles = (std::min(table, window ? seen : table) + BN - 1) / BN, grid = items_each(kv, rows, Hq) * kv.B;
    return (tiles <= kFewTiles && grid <= kFewItems / kv.Hkv) ||
           (tiles <= kMoreTiles && grid <= kMoreItems / kv.Hkv && tiles * kFill <= (long long)rows * Hq / BM);
}

// The workers of a split call.
int workers_of(const tkm_attn_kv& kv, int rows, int Hq) {
    const double tiles = (double)items_most(kv, rows, Hq) * kv.Hkv * (kv.max_pages * (double)kv.page / BN + 1);
    return (int)std::max(std::min(tiles, (double)workers_at(kv.D)), 1.0);
}
// Items that several workers can share: each holds a place where a share begins.
int joints_of(const tkm_attn_kv& kv, int rows, int Hq) {
    return (int)std::min<long long>(workers_of(kv, rows, Hq) - 1, items_most(kv, rows, Hq) * kv.Hkv);
}
size_t align_up(size_t n) { return (n + 255) & ~(size_t)255; }
struct Place {      // of the workspace's parts
    size_t joints, items, part, ml, end;
};
Place places(const tkm_attn_kv& kv, int rows, int Hq) {
    const size_t workers = workers_of(kv, rows, Hq), rows_of = workers * 2 * BM;
    Place p;
    p.joints = align_up(workers * sizeof(Start));
    p.items = p.joints + align_up(workers * sizeof(Joint));
    p.part = p.items + align_up((size_t)items_most(kv, rows, Hq) * sizeof(Item));
    p.ml = p.part + rows_of * kv.D * sizeof(float);
    p.end = p.ml + rows_of * sizeof(float2);
    return p;
}

template <int D, int DT>
int launch_t(const C& a, dim3 grid, int joints, hipStream_t stream) {
    if (a.workers) {
        hipLaunchKernelGGL(chunk_items_kernel, dim3(1), dim3(TL), 0, stream, a);
        if (hipGetLastError() != hipSuccess) return -1;
    }
    hipLaunchKernelGGL((chunk_kernel<D, DT>), grid, dim3(64 * kWaves), 0, stream, a);
    if (hipGetLastError() != hipSuccess) return -1;
    if (joints > 0) {
        // few items in many pieces: a wave a row; else workgroups enough without it
        const int each = joints * (BM / 4) <= 4096 ? 4 : 32;
        hipLaunchKernelGGL((chunk_join_kernel<D, DT>), dim3(joints, BM / each), dim3(256), 0, stream, a, each);
        if (hipGetLastError() != hipSuccess) return -1;
    }
    return 0;
}

}  // namespace

bool chunk_fits(const tkm_attn_kv& kv, int rows, int Hq) {
    // the rows of a kv head, and a head's line, in the integers that hold them
    return (double)rows * (Hq / kv.Hkv) <= 1073741824.0;
}

size_t chunk_workspace(const tkm_attn_kv& kv, int rows, int Hq) {
    return item_each(kv, rows, Hq, 0) ? 0 : places(kv, rows, Hq).end;      // a window only ever saves it
}

int launch_chunk(const ChunkArgs& x) {
    const tkm_attn_kv& kv = x.kv;
    const bool split = !item_each(kv, x.rows, x.Hq, x.window);
    const int workers = split ? workers_of(kv, x.rows, x.Hq) : 0, joints = split ? joints_of(kv, x.rows, x.Hq) : 0;
    char* ws = (char*)x.ws;
    const Place p = places(kv, x.rows, x.Hq);
    const int G = x.Hq / kv.Hkv;
    int shift = 0;
    while (1u << shift < (unsigned)G) ++shift;
    const uint32_t per_g = (uint32_t)(((1ull << (31 + shift)) + G - 1) / G);
    const C a{(const uint16_t*)kv.k, (const uint16_t*)kv.v, kv.table, kv.len, (const uint16_t*)x.q, x.row_start, x.n_new,
              (uint16_t*)x.o, x.lse, (Start*)ws, (Joint*)(ws + p.joints), (Item*)(ws + p.items), (float*)(ws + p.part),
              (float2*)(ws + p.ml), x.q_stride, kv.B, kv.Hkv, x.Hq / kv.Hkv, kv.num_pages, __builtin_ctz(kv.page), kv.max_pages,
              kv.max_pages * kv.page, x.rows, x.causal, x.window, per_g, shift, x.rows / kv.B, workers, (int)items_most(kv, x.rows, x.Hq), x.scale * 1.4426950408889634f};
    note_kernels(kChunk | (joints > 0 ? kJoin : 0));
    const dim3 grid = workers ? dim3(workers) : dim3(items_each(kv, x.rows, x.Hq), kv.B, kv.Hkv);
    const hipStream_t stream = (hipStream_t)x.stream;
    if (kv.D == 128) return kv.dtype == DT_F16 ? launch_t<128, DT_F16>(a, grid, joints, stream) : launch_t<128, DT_BF16>(a, grid, joints, stream);
    return kv.dtype == DT_F16 ? launch_t<64, DT_F16>(a, grid, joints, stream) : launch_t<64, DT_BF16>(a, grid, joints, stream);
}

}  // namespace tkm
