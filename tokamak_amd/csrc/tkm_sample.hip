// tkm_sample.hip -- one token a row of logits, drawn with temperature, top-k, top-p and min-p from a given
// random number (gfx950), and its entry point tkm_hip_sample (include/tkm_hip.h).
//
//   w_i = exp((l_i - max) / T); order: larger l first, equal ones by index
//   top-k: the first k; top-p: of these the shortest head whose sum reaches p of theirs; min-p: of these w >= min_p
//   token: the first i, in the vocabulary's order, at which the running sum of the kept w exceeds u * their sum
//
// Weights are summed as integers, w * 2^shift rounded to nearest (shift 45 at 131072 words, 43 at the most words, 50 at
// few): integer sums are the same in any order, so a draw does not depend on timing, and a border is off by half of
// 2^-shift a word at most, 2^-46 at 131072 words.  (fp32 weights, off by 2^-24 of themselves, move the borders between
// 131072 words so far that about one draw in 10^4 meets another word.)
//
// One workgroup of 16 waves has a row and goes over it two to four times, 8 words a thread a turn:
//   1  the largest logit (where T <= 0, then its first index, and that is all), and for top-k a histogram of the
//      logits' order-preserving bits, the upper 13.  If the bin of top-k's border and those above it have at most
//      2048 words, these go to a list in LDS, and the rest needs no more of the row
//   2  otherwise, and for top-p alone, such a histogram of the weights' sums
//   3  the sums of segments of 512 words over all words in the bins above the border's, and a list in LDS of the
//      border's bin.  The list (a histogram of 10 bits more first, if it is long) gives the border's own bits and
//      how many of the words that equal it are in; its kept words are then added to their segments.  A bin that
//      does not fit the list is gone through in memory instead, and the segments after that.  (Once for each of
//      top-k and top-p; a row without either has all words in 3.)
//   4  the running sum of the segments finds the one that holds the token, and one wave finds the word in it.
// Few words are kept of most rows, so 3 packs those a wave meets and takes 64 exponentials at a time.
// Bound by the passes over the row (from L2 or the Infinity Cache after the first), by the fp64 operations of 2,
// and with few rows by the chain of barriers.  us on one card: 1 x 8192 fp16 with top-k and top-p 14.5; 64 x 32003
// bf16 with all three 24; 256 x 131072 fp32 with top-p and min-p 97, of which reading the rows once is 26, and half
// of the SIMDs' issue is taken.
#include <hip/hip_runtime.h>
#include <hip/hip_fp16.h>
#include <stdarg.h>
#include <stddef.h>
#include <stdint.h>

#include <type_traits>

#include "attn_common.h"
#include "tkm_hip.h"
#include "tkm_prep_internal.h"

namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64, kPer = 8;    // words a thread a turn
constexpr int kTurn = kThreads * kPer;
constexpr int kMostVocab = 1 << 19;
constexpr int kMostDraws = (1 << 22) - 1;      // HIP takes launches of fewer than 2^32 threads
constexpr int kSeg = 64 * kPer, kSegs = kMostVocab / kSeg;           // words of a segment
constexpr int kBits0 = 13, kBits1 = 10, kBits2 = 9, kLow0 = kBits1 + kBits2;
constexpr int kList = 2048, kTable = 32, kQueue = 128;
enum { DT_F32 = 2 };

struct Args {
    const void* logits;
    size_t stride;
    int vocab;
    const int32_t* index;       // row of draw r, or NULL: r
    const float* temperature;
    const int32_t* top_k;
    const float* top_p;
    const float* min_p;
    const float* u;
    int32_t* token;
    int rows;                   // of logits: an index outside them draws -1
    int shift;
};

// The one workgroup of a compute unit's 1024 threads may have most of its 160 KB.
struct __attribute__((aligned(16))) Lds {
    uint64_t s0[1 << kBits0];   // the histograms; those of levels 1 and 2 are zero between their uses
    uint32_t n0[1 << kBits0];
    uint64_t s1[1 << kBits1], s2[1 << kBits2];
    uint32_t n1[1 << kBits1], n2[1 << kBits2];
    uint64_t seg[kSegs];        // sums of segments
    uint32_t ties[kSegs];       // and their words that equal the border
    uint32_t list[kList];       // keys of the border's bin, and their segments
    uint16_t list_seg[kList];
    uint32_t queue[kWaves][kQueue];
    uint32_t few[64];           // what is left of the list, and for each: larger ones, equal ones, the larger ones' sum
    uint32_t few_larger[64], few_same[64];
    uint64_t few_sum[64];
    double pow2[kTable];
    uint64_t tot[2][kWaves];
    uint64_t found64, above64;
    uint32_t found32, found_bin, found_key, list_n, few_n;
};

// Order-preserving bits of a logit, -0 as +0 (not for NaN).
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);
    return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float logit_of(uint32_t k) { return __uint_as_float((k & 0x80000000u) ? k & 0x7fffffffu : ~k); }
constexpr float kLeast = -3.4028234663852886e38f;
constexpr uint32_t kNoBin = ~0u;

// Eight words from i on, as they lie in memory; behind the vocabulary's end -inf.
template <int DT>
struct Raw {
    uint32_t w[DT == DT_F32 ? 8 : 4];
    __device__ __forceinline__ void load(const void* row, int i, int vocab) {
        if (i + kPer <= vocab) {
            __builtin_memcpy(w, (const char*)row + (size_t)i * (DT == DT_F32 ? 4 : 2), sizeof w);
        } else if constexpr (DT == DT_F32) {
#pragma unroll
            for (int j = 0; j < kPer; ++j) {
                const uint32_t x = ((const uint32_t*)row)[min(i + j, vocab - 1)];
                w[j] = i + j < vocab ? x : 0xff800000u;
            }
        } else {
            constexpr uint32_t none = DT == tkm::DT_F16 ? 0xfc00u : 0xff80u;
#pragma unroll
            for (int j = 0; j < kPer; j += 2) {
                const uint32_t x = ((const uint16_t*)row)[min(i + j, vocab - 1)], y = ((const uint16_t*)row)[min(i + j + 1, vocab - 1)];
                w[j / 2] = (i + j < vocab ? x : none) | (i + j + 1 < vocab ? y : none) << 16;
            }
        }
    }
    __device__ __forceinline__ void logits(float (&x)[kPer]) const {
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            if constexpr (DT == DT_F32) {
                x[j] = __uint_as_float(w[j]);
            } else {
                const uint32_t h = w[j / 2];
                x[j] = tkm::to_f32<DT>((uint16_t)(j % 2 ? h >> 16 : h));
            }
        }
    }
};

// exp((x - max) / T) as an integer multiple of 2^-shift, by 2^t = 2^(j/32) 2^(f/32), |f| <= 1/2: the first factor's
// fraction from a table of 32 (64 banks wide: lanes meet in one only where they read the same), the second by its
// Taylor series to f^5 (the next term is below 2^-48).  Adding 1.5 * 2^52 leaves j in the low word; adding
// 2^(52 - shift) leaves the result, rounded to nearest, in the low 52 bits.
struct Weight {
    double max, scale, low, bias;   // scale = 32 log2(e) / T; low: what is further below max counts as this far, 2^-60
    const double* pow2;
    __device__ __forceinline__ uint64_t of(float x) const {     // 0 for -inf and NaN
        constexpr double c = 0.69314718055994530942 / kTable, magic = 6755399441055744.0;
        const double d = fmax((double)x - max, low);
        const double u = fma(d, scale, magic), f = fma(d, scale, magic - u);
        const int j = (int)(uint32_t)(uint64_t)__double_as_longlong(u);
        const double p = fma(fma(fma(fma(fma(f, c * c * c * c * c / 120, c * c * c * c / 24), f, c * c * c / 6), f, c * c / 2), f, c), f, 1.0);
        const uint64_t t = (uint64_t)__double_as_longlong(pow2[j & (kTable - 1)]);
        const double e = __longlong_as_double((long long)(t + ((uint64_t)(uint32_t)((j >> 5) << 20) << 32)));
        return (uint64_t)__double_as_longlong(fma(p, e, bias)) & 0xfffffffffffffull;
    }
};

__device__ __forceinline__ int uni(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ uint64_t lane_value64(uint64_t v, int lane) {
    return ((uint64_t)(uint32_t)tkm::lane_value((int)(v >> 32), lane) << 32) | (uint32_t)tkm::lane_value((int)(uint32_t)v, lane);
}
__device__ __forceinline__ int rank_in(uint64_t mask) {      // lanes of the mask below this one
    return __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
}

// The sum of v over the threads before this one, and over all. One barrier; two calls in a row use two arrays.
__device__ __forceinline__ uint64_t before_me(Lds& lds, int& flip, uint64_t v, uint64_t& total) {
    const int lane = threadIdx.x & 63, wave = uni(threadIdx.x >> 6);
    const uint64_t s = tkm::wave_scan(v);
    if (lane == 63) lds.tot[flip][wave] = s;
    __syncthreads();
    const uint64_t t = tkm::wave_scan(lane < kWaves ? lds.tot[flip][lane] : (uint64_t)0);
    flip ^= 1;
    total = lane_value64(t, 63);
    return (wave ? lane_value64(t, wave - 1) : 0) + s - v;
}

// Where the border lies in a histogram of 2^BITS bins, read from the largest, with `before` already passed: the
// first bin at which the running count n (or sum s) reaches goal_of(the total of the bins), kNoBin if that is 0.
// `before` becomes what lies before that bin, and `above` (where it is asked for) grows by the sums of the bins above.
template <int BITS, class F>
__device__ __forceinline__ uint32_t find_bin(Lds& lds, int& flip, const uint32_t* n, const uint64_t* s, bool by_count, F goal_of,
                                             uint64_t& before, bool want_above, uint64_t& above) {
    constexpr int BINS = 1 << BITS, PER = BINS > kThreads ? BINS / kThreads : 1;
    const int tid = threadIdx.x, last = BINS - 1 - tid * PER, first = last - PER + 1;      // this thread's bins
    uint64_t x[PER] = {}, sum = 0, all;
    if (tid * PER < BINS) {
        if (by_count) {
            uint32_t y[PER];
            __builtin_memcpy(y, n + first, sizeof y);
#pragma unroll
            for (int i = 0; i < PER; ++i) x[i] = y[i];
        } else {
            __builtin_memcpy(x, s + first, sizeof x);
        }
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) sum += x[i];
    uint64_t at = before + before_me(lds, flip, sum, all);
    const uint64_t goal = goal_of(all);
    if (goal == 0) return kNoBin;
    if (at < goal && at + sum >= goal) {      // one thread's
        int bin = last;
#pragma unroll
        for (int i = PER - 1; i > 0; --i)
            if (bin == first + i && at + x[i] < goal) {
                at += x[i];
                --bin;
            }
        lds.found_bin = (uint32_t)bin;
        lds.found64 = at;
    }
    __syncthreads();
    before = lds.found64;
    const uint32_t bin = lds.found_bin;
    if (want_above) {
        sum = 0;
        if (tid * PER < BINS)
#pragma unroll
            for (int i = 0; i < PER; ++i) sum += (uint32_t)(first + i) > bin ? s[first + i] : 0;
        before_me(lds, flip, sum, all);
        above += all;
    }
    return bin;
}

// HELD: the row has one turn, whose keys stay in registers.
template <int DT, bool HELD>
__global__ __launch_bounds__(kThreads) void sample_kernel(Args a) {
    __shared__ Lds lds;
    const int tid = threadIdx.x, lane = tid & 63, wave = uni(tid >> 6), r = blockIdx.x;
    int flip = 0;
    const int at_row = a.index ? a.index[r] : r;
    if (a.index && (unsigned)at_row >= (unsigned)a.rows) {
        if (tid == 0) a.token[r] = -1;
        return;
    }
    const void* row = (const char*)a.logits + (size_t)at_row * a.stride * (DT == DT_F32 ? 4 : 2);
    const int V = a.vocab, turns = HELD ? 1 : (V + kTurn - 1) / kTurn;
    bool only_inf = false;      // the largest is +inf: those words become 0, all others -inf
    auto words_of = [&](const Raw<DT>& raw, float (&x)[kPer]) {
        raw.logits(x);
        if (only_inf)
#pragma unroll
            for (int j = 0; j < kPer; ++j) x[j] = x[j] == INFINITY ? 0.f : -INFINITY;
    };
    Raw<DT> held;
    if (HELD) held.load(row, tid * kPer, V);
    auto each = [&](auto f) {          // f(turn, 8 words), the next turn's words under way
        if constexpr (HELD) {
            // opaque, or the compiler keeps what it made of each word for the next pass, in 60 spilled registers
#pragma unroll
            for (auto& w : held.w) asm volatile("" : "+v"(w));
            float w[kPer];
            words_of(held, w);
            f(0, w);
        } else {
            Raw<DT> x, y;
            const int i0 = tid * kPer;
            x.load(row, i0, V);
            for (int t = 0; t < turns; ++t) {
                float w[kPer];
                words_of(x, w);
                if (t + 1 < turns) y.load(row, i0 + (t + 1) * kTurn, V);
                f(t, w);
                x = y;
            }
        }
    };
    const float T = a.temperature ? a.temperature[r] : 1.0f;
    const int top_k = a.top_k ? a.top_k[r] : 0;
    const float top_p = a.top_p ? a.top_p[r] : 1.0f;
    const float min_p = a.min_p ? a.min_p[r] : 0.f;
    const bool by_p = T > 0.f && top_p < 1.0f;
    bool by_k = T > 0.f && top_k > 0 && top_k < V;

    // 1: the largest, and for top-k the histogram of counts.  If it is +inf, once more with only those words.
    float top;
    for (;; only_inf = true) {
        if (by_k || by_p) {
            const uint4 zero = make_uint4(0, 0, 0, 0);
            for (int i = tid; i < (int)(offsetof(Lds, seg) / 16); i += kThreads) ((uint4*)&lds)[i] = zero;
        }
        if (tid < kTable) lds.pow2[tid] = exp2(tid * (1.0 / kTable));
        if (tid < 64) lds.few_larger[tid] = lds.few_same[tid] = 0, lds.few_sum[tid] = 0;
        if (tid == 0) lds.list_n = lds.few_n = 0;
        if (by_k) __syncthreads();
        top = -INFINITY;
        each([&](int, const float (&x)[kPer]) {
#pragma unroll
            for (int j = 0; j < kPer; ++j) {
                top = fmaxf(top, x[j]);
                if (by_k && x[j] >= kLeast) atomicAdd(&lds.n0[key_of(x[j]) >> kLow0], 1u);
            }
        });
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
        if (lane == 0) lds.tot[0][wave] = __float_as_uint(top);
        __syncthreads();
        top = __uint_as_float((uint32_t)lds.tot[0][lane & (kWaves - 1)]);
#pragma unroll
        for (int o = kWaves / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
        flip = 1;
        if (top < INFINITY) break;
        __syncthreads();
    }
    if (top == -INFINITY) {
        if (tid == 0) a.token[r] = -1;
        return;
    }
    if (!(T > 0.f)) {                // the first of the largest
        uint32_t first = ~0u;
        each([&](int t, const float (&x)[kPer]) {
#pragma unroll
            for (int j = kPer - 1; j >= 0; --j)
                if (x[j] == top) first = min(first, (uint32_t)(t * kTurn + tid * kPer + j));
        });
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) first = min(first, (uint32_t)__shfl_xor((int)first, o, 64));
        if (lane == 0) lds.tot[1][wave] = first;
        __syncthreads();
        if (tid == 0) {
            for (int w = 1; w < kWaves; ++w) first = min(first, (uint32_t)lds.tot[1][w]);
            a.token[r] = (int32_t)first;
        }
        return;
    }
    Weight wt;
    wt.max = (double)top;
    wt.scale = fmax(kTable * 1.4426950408889634074 / (double)T, 1e-60);   // T = inf: any difference of two fp32 is nothing
    wt.low = -60.0 * kTable / wt.scale;
    wt.bias = ldexp(1.0, 52 - a.shift);
    wt.pow2 = lds.pow2;
    // min-p as the least logit that stays: w >= min_p is x >= max + T ln(min_p).  The largest always stays.
    float least = kLeast;
    if (min_p >= 1.0f) {
        least = top;
    } else if (min_p > 0.f) {
        const double x = wt.max + (double)T * log((double)min_p);
        float f = (float)x;
        if ((double)f < x) f = logit_of(key_of(f) + 1);
        least = fmaxf(least, fminf(top, f));
    }

    // 2: the counts give the bin of top-k's border; if the list takes that bin and all above it, it is all that
    // matters of the row.  Otherwise the histogram of sums, if top-p asks for it.
    uint32_t bin_k = kNoBin;
    uint64_t before_k = 0, none = 0;
    bool full = false;
    if (by_k) {
        bin_k = find_bin<kBits0>(lds, flip, lds.n0, lds.s0, true, [&](uint64_t all) { return (uint64_t)top_k < all ? (uint64_t)top_k : 0; },
                                 before_k, false, none);
        by_k = bin_k != kNoBin;            // else all words are in
        full = by_k && before_k + lds.n0[bin_k] <= kList;
    }
    if (by_p && !full) {
        each([&](int, const float (&x)[kPer]) {
            uint64_t q[kPer];
#pragma unroll
            for (int j = 0; j < kPer; ++j) q[j] = wt.of(x[j]);
#pragma unroll
            for (int j = 0; j < kPer; ++j)
                if (q[j]) atomicAdd((unsigned long long*)&lds.s0[key_of(x[j]) >> kLow0], (unsigned long long)q[j]);
        });
        __syncthreads();
    }

    // 3: the border: kept are the words above `border`, and the first `in` of those equal to it.  Step 0 finds
    // top-k's, step 1 top-p's, step 2 has the sums where no list gave them.
    float border = -INFINITY;
    uint32_t in = 0, many = 0;      // many: words that the list has, or should have if there are too many
    bool some = false;                             // only some of the words equal to the border are in
    uint64_t kept_sum = ~0ull;                     // of what top-k keeps; ~0: everything
    for (int step = 0; step < 3; ++step) {
        const bool by_count = step == 0;
        uint64_t goal = (uint64_t)top_k, before = 0, above = 0;
        uint32_t b0 = kNoBin;
        float low = -INFINITY, cut = least;        // words of [low, cut) go to the list, those from cut on to the sums
        if (step < 2) {
            if (by_count ? !by_k : !by_p) continue;
            if (by_count) {
                b0 = bin_k;
                before = before_k;
                if (by_p && !full) {
                    uint64_t m = 0;
                    for (int i = tid; i < 1 << kBits0; i += kThreads) m += (uint32_t)i > b0 ? lds.s0[i] : 0;
                    before_me(lds, flip, m, above);
                }
            } else {
                if (full) {
                    for (uint32_t i = tid; i < many; i += kThreads) {
                        const float x = logit_of(lds.list[i]);
                        if (x >= border) atomicAdd((unsigned long long*)&lds.s0[lds.list[i] >> kLow0], (unsigned long long)wt.of(x));
                    }
                    __syncthreads();
                }
                b0 = find_bin<kBits0>(lds, flip, lds.n0, lds.s0, false, [&](uint64_t all) {
                    kept_sum = min(kept_sum, all);
                    const double x = ceil((double)top_p * (double)kept_sum);
                    return goal = x < 1.0 ? 1 : x < (double)kept_sum ? (uint64_t)x : kept_sum;
                }, before, false, none);
            }
            low = logit_of(b0 << kLow0);
            cut = logit_of((b0 + 1) << kLow0);     // behind +inf's bin a NaN: no word is from there on
        } else {
            if ((by_k || by_p) && many <= kList) break;      // (the list is not empty)
            cut = some ? logit_of(key_of(border) + 1) : border;
        }
        const bool list_only = full || (by_count && by_p);   // the sums are top-p's affair, or the list's
        if (!full || by_count) {
            if (tid == 0) lds.list_n = 0;
            __syncthreads();
            const float from = cut < least ? least : cut;
            uint32_t* queue = lds.queue[wave];
            each([&](int t, const float (&x)[kPer]) {
                const int seg = t * kWaves + wave;
                if (!list_only) {
                    uint64_t m = 0, mask[kPer];
                    int n = 0, ties = 0;
#pragma unroll
                    for (int j = 0; j < kPer; ++j) {
                        mask[j] = __ballot(x[j] >= from);
                        n += __popcll(mask[j]);
                    }
                    if (n > kQueue) {
#pragma unroll
                        for (int j = 0; j < kPer; ++j) {
                            const uint64_t q = wt.of(x[j]);
                            m += x[j] >= from ? q : 0;
                        }
                    } else if (n) {
                        int at = 0;
#pragma unroll
                        for (int j = 0; j < kPer; ++j) {
                            if (x[j] >= from) queue[at + rank_in(mask[j])] = __float_as_uint(x[j]);
                            at += __popcll(mask[j]);
                        }
                        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                        for (int i = lane; i < n; i += 64) m += wt.of(__uint_as_float(queue[i]));
                        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                    }
                    if (step == 2 && some)
#pragma unroll
                        for (int j = 0; j < kPer; ++j) ties += __popcll(__ballot(x[j] == border));
                    m = n ? tkm::wave_scan(m) : 0;
                    if (lane == 63) {
                        lds.seg[seg] = m;
                        lds.ties[seg] = (uint32_t)ties;
                    }
                }
                if (step < 2) {
                    uint32_t here = 0;
#pragma unroll
                    for (int j = 0; j < kPer; ++j) here |= x[j] >= low && (full || !(x[j] >= cut)) ? 1u << j : 0u;
                    if (__any(here)) {
                        const uint32_t c = (uint32_t)__popc(here), s = tkm::wave_scan(c);
                        uint32_t at = 0;
                        if (lane == 63) at = atomicAdd(&lds.list_n, s);
                        at = (uint32_t)tkm::lane_value((int)at, 63) + s - c;
#pragma unroll
                        for (int j = 0; j < kPer; ++j)
                            if (here >> j & 1) {
                                if (at < kList) {
                                    lds.list[at] = key_of(x[j]);
                                    lds.list_seg[at] = (uint16_t)seg;
                                }
                                ++at;
                            }
                    }
                }
            });
            __syncthreads();
            many = lds.list_n;
        }
        if (step == 2) break;

        // the border's own bits: of a long list (or bin) first 10 more, and if that leaves many words the last 9
        const uint32_t* few = lds.list;
        uint32_t n = full ? lds.n0[b0] : many, equal = 0, prefix = b0;
        auto pick = [&](int below) {             // the list's words with that prefix
            for (uint32_t i = tid; i < many; i += kThreads)
                if (lds.list[i] >> below == prefix) lds.few[atomicAdd(&lds.few_n, 1u)] = lds.list[i];
            few = lds.few;
        };
        const bool want_above = by_count && by_p && !full;
        if (full && n <= 64) {
            pick(kLow0);
            __syncthreads();
            if (tid == 0) lds.few_n = 0;
        }
        for (int level = 1; level < 3 && n > 64; ++level) {
            uint32_t* nh = level == 1 ? lds.n1 : lds.n2;
            uint64_t* sh = level == 1 ? lds.s1 : lds.s2;
            const int below = level == 1 ? kBits2 : 0, bits = level == 1 ? kBits1 : kBits2;
            auto one = [&](uint32_t k) {
                if (k >> (below + bits) != prefix) return;
                const uint32_t b = k >> below & ((1u << bits) - 1);
                atomicAdd(&nh[b], 1u);
                if (by_p) atomicAdd((unsigned long long*)&sh[b], (unsigned long long)wt.of(logit_of(k)));
            };
            if (many <= kList) {
                for (uint32_t i = tid; i < many; i += kThreads) one(lds.list[i]);
            } else {
                each([&](int, const float (&x)[kPer]) {
#pragma unroll
                    for (int j = 0; j < kPer; ++j)
                        if (x[j] >= low && !(x[j] >= cut)) one(key_of(x[j]));
                });
            }
            __syncthreads();
            const auto same_goal = [&](uint64_t) { return goal; };
            const uint32_t b1 = level == 1 ? find_bin<kBits1>(lds, flip, nh, sh, by_count, same_goal, before, want_above, above)
                                           : find_bin<kBits2>(lds, flip, nh, sh, by_count, same_goal, before, want_above, above);
            prefix = prefix << bits | b1;
            equal = nh[b1];
            __syncthreads();
            if (tid < 1 << bits) {
                nh[tid] = 0;
                sh[tid] = 0;
            }
            if (level == 2) {
                border = logit_of(prefix);
                n = 0;
            } else if (many <= kList && equal <= 64) {
                pick(kBits2);
                n = equal;
            }
            __syncthreads();
            if (tid == 0) lds.few_n = 0;
        }
        if (n) {        // at most 64 words: each with all, 4 a wave
            const uint32_t x = lane < (int)n ? few[lane] : 0;
            const uint64_t q = by_p ? wt.of(logit_of(x)) : 0;
            if (wave * 4 < (int)n) {
                uint32_t larger = 0, same = 0;
                uint64_t sum = 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int j = wave * 4 + i;
                    const uint32_t y = (uint32_t)tkm::lane_value((int)x, j);      // 0 from n on: neither larger nor equal
                    larger += y > x;
                    same += y == x;
                    sum += y > x ? lane_value64(q, j) : 0;
                }
                if (lane < (int)n) {
                    atomicAdd(&lds.few_larger[lane], larger);
                    atomicAdd(&lds.few_same[lane], same);
                    if (by_p) atomicAdd((unsigned long long*)&lds.few_sum[lane], (unsigned long long)sum);
                }
            }
            __syncthreads();
            if (wave == 0) {
                const uint32_t larger = lds.few_larger[lane], same = lds.few_same[lane];
                const uint64_t sum = lds.few_sum[lane], at = before + (by_count ? larger : sum);
                lds.few_larger[lane] = lds.few_same[lane] = 0;
                lds.few_sum[lane] = 0;
                if (lane < (int)n && at < goal && at + (by_count ? same : same * q) >= goal) {   // equal words agree
                    lds.found_key = x;
                    lds.found32 = same;
                    lds.found64 = at;
                    lds.above64 = above + sum;
                }
            }
            __syncthreads();
            border = logit_of(lds.found_key);
            equal = lds.found32;
            before = lds.found64;
            above = lds.above64;
        }
        if (by_count) {
            in = (uint32_t)(goal - before);
            if (full && by_p) {
                uint64_t m = 0;
                for (uint32_t i = tid; i < many; i += kThreads) {
                    const float x = logit_of(lds.list[i]);
                    m += x > border ? wt.of(x) : 0;
                }
                before_me(lds, flip, m, above);
            }
            kept_sum = above + in * wt.of(border);
        } else {
            const uint64_t q = wt.of(border);
            in = (uint32_t)((goal - before + q - 1) / q);      // q > 0: the border's bin has a sum
        }
        some = in < equal;
    }
    if ((by_k || by_p) && many <= kList) {          // the list's kept words to their segments
        if (full) {
            if (tid < kSegs) {
                lds.seg[tid] = 0;
                lds.ties[tid] = 0;
            }
            __syncthreads();
        }
        for (uint32_t i = tid; i < many; i += kThreads) {
            const float x = logit_of(lds.list[i]);
            if (x == border && some) atomicAdd(&lds.ties[lds.list_seg[i]], 1u);
            else if (x >= border && x >= least)
                atomicAdd((unsigned long long*)&lds.seg[lds.list_seg[i]], (unsigned long long)wt.of(x));
        }
        __syncthreads();
    }

    // 4: the segment, then the word in it
    const uint64_t qb = some && border >= least ? wt.of(border) : 0;     // a word equal to the border, where only some are in
    const int segs = turns * kWaves;     // at most kThreads: one a thread
    uint64_t m = tid < segs ? lds.seg[tid] : 0, before_ties = 0, total;
    if (some) {
        const uint64_t ties = tid < segs ? lds.ties[tid] : 0;
        before_ties = before_me(lds, flip, ties, total);
        m += (before_ties >= in ? 0 : min(ties, in - before_ties)) * qb;
    }
    const uint64_t up = before_me(lds, flip, m, total);
    const double goal = (double)a.u[r] * (double)total;
    uint64_t g = goal > 0.0 ? (uint64_t)fmin(goal, 9.0e18) : 0;    // the running sum has to exceed it
    if (g >= total) g = total - 1;                                 // the largest logit is kept: total > 0
    if (up <= g && g < up + m) {
        lds.found_bin = (uint32_t)tid;
        lds.found64 = up;
        lds.found32 = (uint32_t)before_ties;
    }
    __syncthreads();
    const int s = (int)lds.found_bin;
    if (HELD ? wave != s : wave != 0) return;
    float x[kPer];
    const int i = s * kSeg + lane * kPer;
    if (!HELD) held.load(row, i, V);
    words_of(held, x);
    uint32_t e = 0;
#pragma unroll
    for (int j = 0; j < kPer; ++j) e += some && x[j] == border ? 1u : 0u;
    uint32_t rank = lds.found32 + tkm::wave_scan(e) - e;
    uint64_t q[kPer], mine = 0;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        q[j] = x[j] >= border && x[j] >= least ? wt.of(x[j]) : 0;
        if (some && x[j] == border) q[j] = rank++ < in ? qb : 0;
        mine += q[j];
    }
    uint64_t run = lds.found64 + tkm::wave_scan(mine) - mine;
    if (run <= g && g < run + mine) {
        int at = 0;
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            if (run <= g && g < run + q[j]) at = i + j;
            run += q[j];
        }
        a.token[r] = at;
    }
}

int fail(int status, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
int fail(int status, const char* fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    tkm_vset_error(status, fmt, ap);
    va_end(ap);
    return status;
}

}  // namespace

extern "C" TKM_API int tkm_hip_sample(const tkm_sample_args* s, void* stream) {
    if (!s || !s->logits || !s->u || !s->token) return fail(TKM_ATTN_EINVAL, "logits, u and token must be non-null");
    if (s->rows < 1 || s->draws < 1 || s->vocab < 1)
        return fail(TKM_ATTN_EINVAL, "sizes must be positive (rows=%d draws=%d vocab=%d)", s->rows, s->draws, s->vocab);
    if (!s->row_index && s->draws > s->rows)
        return fail(TKM_ATTN_EINVAL, "%d draws of %d rows need a row_index", s->draws, s->rows);
    if (s->draws > kMostDraws) return fail(TKM_ATTN_EUNSUPPORTED, "%d draws (at most %d)", s->draws, kMostDraws);
    if (s->dtype != TKM_ATTN_F16 && s->dtype != TKM_ATTN_BF16 && s->dtype != TKM_SAMPLE_F32)
        return fail(TKM_ATTN_EUNSUPPORTED, "dtype %d (supported: TKM_ATTN_F16, TKM_ATTN_BF16, TKM_SAMPLE_F32)", s->dtype);
    if (s->vocab > kMostVocab) return fail(TKM_ATTN_EUNSUPPORTED, "vocab=%d (at most %d)", s->vocab, kMostVocab);
    if (s->row_stride < (size_t)s->vocab || s->row_stride > (size_t)1 << 40)
        return fail(TKM_ATTN_EINVAL, "row_stride=%zu must be at least vocab=%d", s->row_stride, s->vocab);
    const uintptr_t el = s->dtype == TKM_SAMPLE_F32 ? 4 : 2;
    if ((uintptr_t)s->logits % el || ((uintptr_t)s->row_index | (uintptr_t)s->temperature | (uintptr_t)s->top_k | (uintptr_t)s->top_p |
                                      (uintptr_t)s->min_p | (uintptr_t)s->u | (uintptr_t)s->token) % 4)
        return fail(TKM_ATTN_EALIGN, "logits must be aligned to their type, the other arrays to 4 bytes");
    int shift = 62;                          // sums of vocab weights of at most 2^shift stay below 2^63
    while ((s->vocab - 1) >> (62 - shift)) --shift;
    if (shift > 50) shift = 50;
    const Args a{s->logits, s->row_stride, s->vocab, s->row_index, s->temperature, s->top_k, s->top_p, s->min_p, s->u, s->token,
                 s->rows, shift};
    const bool held = s->vocab <= kTurn;
    auto* kernel = s->dtype == TKM_SAMPLE_F32 ? (held ? sample_kernel<DT_F32, true> : sample_kernel<DT_F32, false>)
                   : s->dtype == TKM_ATTN_BF16 ? (held ? sample_kernel<tkm::DT_BF16, true> : sample_kernel<tkm::DT_BF16, false>)
                                               : (held ? sample_kernel<tkm::DT_F16, true> : sample_kernel<tkm::DT_F16, false>);
    hipLaunchKernelGGL(kernel, dim3((unsigned)s->draws), dim3(kThreads), 0, (hipStream_t)stream, a);
    if (hipGetLastError() != hipSuccess) return fail(TKM_ATTN_ELAUNCH, "sample: kernel launch failed");
    return TKM_ATTN_OK;
}
