// tkm_sample.hip -- one token a row of logits, drawn with temperature, top-k, top-p and min-p from a given
// random number (gfx950), and its entry point tkm_hip_sample (include/tkm_hip.h).
//
//   w_i = exp((l_i - max) / T); order: larger l first, equal ones by index
//   top-k: the first k; top-p: of these the shortest head whose sum reaches p of theirs; min-p: of these w >= min_p
//   token: the first i, in the vocabulary's order, at which the running sum of the kept w exceeds u * their sum
//
// Weights are summed as integers, w * 2^shift rounded to nearest (shift 44 at 131072 words and up to 50): integer
// sums are the same in any order, so a draw does not depend on timing, and a border is off by 2^-45 a word at
// most, where fp32 sums would move it by 2^-24 each.
//
// One workgroup of 16 waves has a row and goes over it a few times, 8 words a thread a turn:
//   1  the largest logit and its first index (all that T <= 0 needs)
//   2  a histogram of the logits' order-preserving bits, the upper 13, with the count and sum of each bin
//   3  for each of top-k and top-p: the words of the bin in which its border lies go to a list in LDS (or, where
//      they are too many, stay in memory), and two histograms of it, of 10 and 9 bits, give the border's own bits
//      and how many of the words that equal it are in
//   4  the kept sums of segments of 512 words, whose running sum finds the segment, and in it the word.
// Without top-k and top-p 2 and 3 fall away.  Bound by the passes over the row (from L2 and the Infinity Cache
// after the first), and with few rows by the turns' latency.
#include <hip/hip_runtime.h>
#include <hip/hip_fp16.h>
#include <stdarg.h>
#include <stdint.h>

#include "attn_common.h"
#include "tkm_hip.h"
#include "tkm_prep_internal.h"

namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64, kPer = 8;    // words a thread a turn
constexpr int kTurn = kThreads * kPer;
constexpr int kMostVocab = 1 << 19;
constexpr int kSegs = kMostVocab / (64 * kPer);
constexpr int kBits0 = 13, kBits1 = 10, kBits2 = 9;
constexpr int kList = 4096;
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

struct Lds {
    uint32_t n0[1 << kBits0];
    uint64_t s0[1 << kBits0];   // later: segments' sums
    uint32_t n1[1 << kBits1];
    uint64_t s1[1 << kBits1];
    uint32_t list[kList];
    uint32_t ties[kSegs];
    double pow2[64];
    uint64_t wave64[kWaves];
    uint32_t wave32[kWaves];
    uint64_t found64;
    uint32_t found32, found_bin, list_n;
};

// Order-preserving bits of a logit; NaN counts as -inf, -0 as +0.
__device__ __forceinline__ uint32_t key_of(float x) {
    if (x != x) x = -INFINITY;
    const uint32_t b = __float_as_uint(x + 0.0f);
    return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float logit_of(uint32_t k) { return __uint_as_float((k & 0x80000000u) ? k & 0x7fffffffu : ~k); }
constexpr uint32_t kNone = 0x007fffffu;     // the key of -inf

// Eight words from i on; behind the vocabulary's end -inf.
template <int DT>
__device__ __forceinline__ void load8(const void* row, int i, int vocab, uint32_t (&k)[kPer]) {
    float x[kPer];
    if constexpr (DT == DT_F32) {
        const float* p = (const float*)row + i;
        if (i + kPer <= vocab) {
            __builtin_memcpy(x, p, sizeof x);
        } else {
#pragma unroll
            for (int j = 0; j < kPer; ++j) x[j] = i + j < vocab ? p[j] : -INFINITY;
        }
    } else {
        const uint16_t* p = (const uint16_t*)row + i;
        uint16_t h[kPer];
        if (i + kPer <= vocab) {
            __builtin_memcpy(h, p, sizeof h);
        } else {
#pragma unroll
            for (int j = 0; j < kPer; ++j) h[j] = i + j < vocab ? p[j] : (uint16_t)(DT == tkm::DT_F16 ? 0xfc00 : 0xff80);
        }
#pragma unroll
        for (int j = 0; j < kPer; ++j) x[j] = tkm::to_f32<DT>(h[j]);
    }
#pragma unroll
    for (int j = 0; j < kPer; ++j) k[j] = key_of(x[j]);
}

// exp((x - max) / T) by 2^t = 2^(j/64) 2^r, |r| <= 1/128: the first factor's fraction from a table of 64, the
// second by its Taylor series to r^5 (the next term is below 2^-54).
struct Weight {
    uint32_t top;       // key of the largest logit
    double max, scale;  // scale = log2(e) / T
    int shift;
    const double* pow2;
    __device__ __forceinline__ double of(uint32_t key) const {
        if (key == top) return 1.0;
        const double t = ((double)logit_of(key) - max) * scale;
        if (!(t > -1000.0) || key == kNone) return 0.0;
        const double j = rint(t * 64.0), y = (t - j * 0.015625) * 0.69314718055994530942;
        const double p = fma(fma(fma(fma(fma(y, 1.0 / 120, 1.0 / 24), y, 1.0 / 6), y, 0.5), y, 1.0), y, 1.0);
        const int n = (int)j;
        return ldexp(p * pow2[n & 63], n >> 6);
    }
    // rounded to a multiple of 2^-shift, as an integer: the sum with 2^52 leaves it in the mantissa's low bits
    __device__ __forceinline__ uint64_t fixed(double w) const {
        return (uint64_t)__double_as_longlong(ldexp(w, shift) + 4503599627370496.0) & 0xfffffffffffffull;
    }
};

__device__ __forceinline__ uint64_t shfl_up64(uint64_t v, int o) {
    return ((uint64_t)(uint32_t)__shfl_up((int)(v >> 32), o, 64) << 32) | (uint32_t)__shfl_up((int)(uint32_t)v, o, 64);
}
template <class T>
__device__ __forceinline__ T scan64(T v, int lane) {   // inclusive, over the wave
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const T y = sizeof(T) == 8 ? (T)shfl_up64((uint64_t)v, o) : (T)__shfl_up((int)v, o, 64);
        if (lane >= o) v += y;
    }
    return v;
}

// Where the border lies in a histogram of 2^BITS bins, read from the largest: the first bin at which the running
// count (by_count) or sum reaches `goal`; `count` and `sum` become what lies before it.
template <int BITS>
__device__ void find_bin(Lds& lds, const uint32_t* n, const uint64_t* s, bool by_count, uint64_t goal, uint32_t& bin,
                         uint32_t& count, uint64_t& sum) {
    constexpr int BINS = 1 << BITS, PER = BINS > kThreads ? BINS / kThreads : 1;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int first = BINS - 1 - tid * PER;      // this thread's bins, downwards
    uint32_t c = 0;
    uint64_t m = 0;
    if (tid * PER < BINS)
        for (int i = 0; i < PER; ++i) {
            c += n[first - i];
            m += s[first - i];
        }
    const uint32_t ci = scan64(c, lane);
    const uint64_t mi = scan64(m, lane);
    if (lane == 63) {
        lds.wave32[wave] = ci;
        lds.wave64[wave] = mi;
    }
    __syncthreads();
    uint32_t cb = ci - c;
    uint64_t mb = mi - m;
    for (int w = 0; w < wave; ++w) {
        cb += lds.wave32[w];
        mb += lds.wave64[w];
    }
    const uint64_t before = (by_count ? (uint64_t)cb : mb) + (by_count ? (uint64_t)count : sum);
    const uint64_t mine = by_count ? (uint64_t)c : m;
    if (before < goal && before + mine >= goal) {      // one thread's
        cb += count;
        mb += sum;
        int i = 0;
        for (; i < PER - 1; ++i) {
            const uint64_t at = by_count ? (uint64_t)(cb + n[first - i]) : mb + s[first - i];
            if (at >= goal) break;
            cb += n[first - i];
            mb += s[first - i];
        }
        lds.found_bin = (uint32_t)(first - i);
        lds.found32 = cb;
        lds.found64 = mb;
    }
    __syncthreads();
    bin = lds.found_bin;
    count = lds.found32;
    sum = lds.found64;
}

template <int DT>
__global__ __launch_bounds__(kThreads) void sample_kernel(Args a) {
    __shared__ Lds lds;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r = blockIdx.x;
    const int at_row = a.index ? a.index[r] : r;
    if (a.index && (unsigned)at_row >= (unsigned)a.rows) {
        if (tid == 0) a.token[r] = -1;
        return;
    }
    const void* row = (const char*)a.logits + (size_t)at_row * a.stride * (DT == DT_F32 ? 4 : 2);
    const int V = a.vocab, turns = (V + kTurn - 1) / kTurn;
    auto each = [&](auto f) {          // f(turn, index of the first of 8 words, their keys)
#pragma unroll 2
        for (int t = 0; t < turns; ++t) {
            const int i = t * kTurn + tid * kPer;
            uint32_t k[kPer];
            if (i < V) {
                load8<DT>(row, i, V, k);
            } else {
#pragma unroll
                for (int j = 0; j < kPer; ++j) k[j] = kNone;
            }
            f(t, i, k);
        }
    };

    // 1: the largest, the first of equal ones
    uint64_t best = 0;
    each([&](int, int i, const uint32_t (&k)[kPer]) {
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            const uint64_t x = ((uint64_t)k[j] << 32) | (uint32_t)~(i + j);
            best = x > best ? x : best;
        }
    });
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const uint64_t x = ((uint64_t)(uint32_t)__shfl_xor((int)(best >> 32), o, 64) << 32) | (uint32_t)__shfl_xor((int)(uint32_t)best, o, 64);
        best = x > best ? x : best;
    }
    if (lane == 0) lds.wave64[wave] = best;
    if (tid < 64) lds.pow2[tid] = exp2(tid * 0.015625);
    __syncthreads();
    for (int w = 0; w < kWaves; ++w) best = lds.wave64[w] > best ? lds.wave64[w] : best;
    const uint32_t top = (uint32_t)(best >> 32);
    const float T = a.temperature ? a.temperature[r] : 1.0f;
    if (top == kNone || !(T > 0.f)) {
        if (tid == 0) a.token[r] = top == kNone ? -1 : (int32_t)~(uint32_t)best;
        return;
    }
    const Weight wt{top, (double)logit_of(top), 1.4426950408889634074 / (double)T, a.shift, lds.pow2};
    const int k = a.top_k ? a.top_k[r] : 0;
    const float p = a.top_p ? a.top_p[r] : 1.0f;
    const bool by_k = k > 0 && k < V, by_p = p < 1.0f;
    const float mf = a.min_p ? a.min_p[r] : 0.f;
    const double mp = mf > 0.f ? fmin((double)mf, 1.0) : 0.0;   // the largest always stays

    // 2, 3: the border: kept are the keys above `border`, and the first `in` of those equal to it
    uint32_t border = 0, in = 0;
    bool some = false;       // only some of those equal to it
    if (by_k || by_p) {
        for (int i = tid; i < 1 << kBits0; i += kThreads) {
            lds.n0[i] = 0;
            lds.s0[i] = 0;
        }
        __syncthreads();
        each([&](int, int, const uint32_t (&k)[kPer]) {
#pragma unroll
            for (int j = 0; j < kPer; ++j) {
                if (k[j] == kNone) continue;
                const uint32_t b = k[j] >> (32 - kBits0);
                atomicAdd(&lds.n0[b], 1u);
                if (by_p) {
                    const uint64_t q = wt.fixed(wt.of(k[j]));
                    if (q) atomicAdd((unsigned long long*)&lds.s0[b], (unsigned long long)q);
                }
            }
        });
        __syncthreads();
        // the border's own bits: by count, the goal-th word; by sum, the word at which the sum reaches the goal
        auto descend = [&](bool by_count, uint64_t goal, uint32_t& key, uint32_t& count, uint64_t& sum) {
            uint32_t b0, b1, b2;
            count = 0;
            sum = 0;
            find_bin<kBits0>(lds, lds.n0, lds.s0, by_count, goal, b0, count, sum);
            const uint32_t many = lds.n0[b0];
            const bool listed = many <= kList;
            if (listed) {
                if (tid == 0) lds.list_n = 0;
                __syncthreads();
                each([&](int, int, const uint32_t (&k)[kPer]) {
#pragma unroll
                    for (int j = 0; j < kPer; ++j)
                        if (k[j] >> (32 - kBits0) == b0 && k[j] != kNone) lds.list[atomicAdd(&lds.list_n, 1u)] = k[j];
                });
                __syncthreads();
            }
            auto fill = [&](uint32_t prefix, int shift, int bits) {    // of the words whose bits above are `prefix`
                for (int i = tid; i < 1 << bits; i += kThreads) {
                    lds.n1[i] = 0;
                    lds.s1[i] = 0;
                }
                __syncthreads();
                auto one = [&](uint32_t key) {
                    if (key >> (shift + bits) != prefix || key == kNone) return;
                    const uint32_t b = key >> shift & ((1u << bits) - 1);
                    atomicAdd(&lds.n1[b], 1u);
                    if (by_p) {
                        const uint64_t q = wt.fixed(wt.of(key));
                        if (q) atomicAdd((unsigned long long*)&lds.s1[b], (unsigned long long)q);
                    }
                };
                if (listed) {
                    for (uint32_t i = tid; i < many; i += kThreads) one(lds.list[i]);
                } else {
                    each([&](int, int, const uint32_t (&k)[kPer]) {
#pragma unroll
                        for (int j = 0; j < kPer; ++j) one(k[j]);
                    });
                }
                __syncthreads();
            };
            fill(b0, kBits2, kBits1);
            find_bin<kBits1>(lds, lds.n1, lds.s1, by_count, goal, b1, count, sum);
            fill(b0 << kBits1 | b1, 0, kBits2);
            find_bin<kBits2>(lds, lds.n1, lds.s1, by_count, goal, b2, count, sum);
            key = (b0 << kBits1 | b1) << kBits2 | b2;
            const uint32_t equal = lds.n1[b2];
            __syncthreads();
            return equal;
        };
        // words of some weight, and their sum: a goal beyond them needs no border
        uint32_t words = 0;
        uint64_t all = 0;
        {
            uint32_t c = 0;
            uint64_t m = 0;
            for (int i = tid; i < 1 << kBits0; i += kThreads) {
                c += lds.n0[i];
                m += lds.s0[i];
            }
            c = scan64(c, lane);
            m = scan64(m, lane);
            if (lane == 63) {
                lds.wave32[wave] = c;
                lds.wave64[wave] = m;
            }
            __syncthreads();
            for (int w = 0; w < kWaves; ++w) {
                words += lds.wave32[w];
                all += lds.wave64[w];
            }
            __syncthreads();
        }
        uint32_t count;
        uint64_t sum;
        if (by_k && (uint32_t)k < words) {
            const uint32_t equal = descend(true, (uint64_t)k, border, count, sum);
            in = (uint32_t)k - count;
            some = in < equal;
            all = sum + in * wt.fixed(wt.of(border));
        }
        if (by_p) {
            const double goal = ceil((double)p * (double)all);
            const uint64_t g = goal < 1.0 ? 1 : goal < (double)all ? (uint64_t)goal : all;
            uint32_t equal = descend(false, g, border, count, sum);
            const uint64_t q = wt.fixed(wt.of(border));
            in = (uint32_t)((g - sum + q - 1) / q);      // q > 0: the border's bin has a sum
            some = in < equal;
        }
        if (!some) in = ~0u;
    } else {
        in = ~0u;
    }

    // 4: the sums of what is kept
    auto kept = [&](uint32_t key) -> uint64_t {     // a word above the border (or equal to it, where all of those are in)
        if (key == kNone || key < border || (key == border && some)) return 0;
        const double w = wt.of(key);
        return w >= mp ? wt.fixed(w) : 0;
    };
    const double wb = some ? wt.of(border) : 0.0;
    const uint64_t qb = some && wb >= mp ? wt.fixed(wb) : 0;     // a word equal to the border
    uint64_t* seg = lds.s0;
    each([&](int t, int, const uint32_t (&k)[kPer]) {
        uint64_t m = 0;
        uint32_t e = 0;
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            m += kept(k[j]);
            e += some && k[j] == border ? 1u : 0u;
        }
        m = scan64(m, lane);
        if (some) e = scan64(e, lane);
        if (lane == 63) {
            seg[t * kWaves + wave] = m;
            lds.ties[t * kWaves + wave] = e;
        }
    });
    __syncthreads();
    const int segs = turns * kWaves;     // at most kThreads: one a thread
    uint64_t m = tid < segs ? seg[tid] : 0;
    uint32_t before_ties = 0, ties = 0;
    if (some) {
        ties = tid < segs ? lds.ties[tid] : 0;
        const uint32_t e = scan64(ties, lane);
        if (lane == 63) lds.wave32[wave] = e;
        __syncthreads();
        before_ties = e - ties;
        for (int w = 0; w < wave; ++w) before_ties += lds.wave32[w];
        const uint32_t mine = before_ties >= in ? 0 : min(ties, in - before_ties);
        m += mine * qb;
    }
    const uint64_t mi = scan64(m, lane);
    if (lane == 63) lds.wave64[wave] = mi;
    __syncthreads();
    uint64_t total = 0, base = 0;
    for (int w = 0; w < kWaves; ++w) {
        base += w < wave ? lds.wave64[w] : 0;
        total += lds.wave64[w];
    }
    const double goal = (double)a.u[r] * (double)total;
    uint64_t g = goal > 0.0 ? (uint64_t)fmin(goal, 9.0e18) : 0;    // the running sum has to exceed it
    if (g >= total) g = total - 1;                                 // the largest logit is kept: total > 0
    const uint64_t up = base + mi - m;
    if (up <= g && g < up + m) {
        lds.found_bin = (uint32_t)tid;
        lds.found64 = up;
        lds.found32 = before_ties;
    }
    __syncthreads();
    if (wave != 0) return;
    // the word within its segment, by one wave
    const int s = (int)lds.found_bin, i = s * 64 * kPer + lane * kPer;
    uint32_t key[kPer];
    if (i < V) {
        load8<DT>(row, i, V, key);
    } else {
#pragma unroll
        for (int j = 0; j < kPer; ++j) key[j] = kNone;
    }
    uint32_t e = 0;
#pragma unroll
    for (int j = 0; j < kPer; ++j) e += some && key[j] == border ? 1u : 0u;
    uint32_t rank = lds.found32 + scan64(e, lane) - e;
    uint64_t q[kPer], mine = 0;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        q[j] = kept(key[j]);
        if (some && key[j] == border) q[j] = rank++ < in ? qb : 0;
        mine += q[j];
    }
    uint64_t run = lds.found64 + scan64(mine, lane) - mine;
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
    auto* kernel = s->dtype == TKM_SAMPLE_F32 ? sample_kernel<DT_F32> : s->dtype == TKM_ATTN_BF16 ? sample_kernel<tkm::DT_BF16> : sample_kernel<tkm::DT_F16>;
    hipLaunchKernelGGL(kernel, dim3((unsigned)s->draws), dim3(kThreads), 0, (hipStream_t)stream, a);
    if (hipGetLastError() != hipSuccess) return fail(TKM_ATTN_ELAUNCH, "sample: kernel launch failed");
    return TKM_ATTN_OK;
}
