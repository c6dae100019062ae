/*
 * tkm_attn.h -- C ABI of the MI355X (gfx950) attention kernels (libtkm_attn.so).
 *
 * This is the inner boundary the Tokamak runtime dispatches GQA attention to.  In the
 * reference it is implicit: the OP_GQA_ATTN cases of execute_forward_pass and of the
 * backward node walk launch k_gqa_flash_attn_tc_fwd / _bwd directly
 * (reference src/tkm_gpu.cu:1252-1265 and 1389-1404, kernels at 302-438 and 440-598).
 * The host runtime (tkm_hip.c) calls these functions at those two sites instead.
 *
 * Conventions (unchanged from the reference):
 *   - all tensors are device pointers, row-major, 16-bit elements (fp16 or bf16):
 *       qkv  [B][S][(Hq + 2*Hkv) * D]  Q heads | K heads | V heads   (tkm_registry.c:736-748)
 *       o    [B][S][Hq * D]
 *       lse  [B][Hq][S] fp32, natural log of the row sum of exp(scaled scores) (tkm_gpu.cu:430)
 *       dout [B][S][Hq * D],  dqkv has the layout of qkv and is overwritten
 *   - q-head h attends with kv-head h / (Hq / Hkv)                (tkm_gpu.cu:315-316)
 *   - scores are scale * <q_i, k_j>; the runtime passes scale = 1/sqrtf(D) (tkm_gpu.cu:1258);
 *     scale must be positive and finite
 *   - key j is visible from query i iff j < S and (!causal || j <= i) (tkm_gpu.cu:393)
 * Extension (reference has none, its GQA op has no key-length input):
 *   - kv_len: optional device array of B int32; keys j >= kv_len[b] are masked.  Values are
 *     clamped to [0, S]; a query row with no visible key gets O = 0, LSE = -inf and zero
 *     gradients.  NULL means kv_len[b] = S.
 *   - dtype TKM_ATTN_BF16 in addition to the reference's fp16.
 *
 * All calls are asynchronous on `stream` (a hipStream_t, NULL = null stream), allocate
 * nothing and never synchronize, so they may be captured into a hipGraph.  D must be 64 or
 * 128 (the reference accepts exactly these, tkm_core.c:392-404).  16-bit tensors and the
 * workspace must be 16-byte aligned; lse 4-byte aligned.
 * Return value: TKM_ATTN_OK or a negative status; tkm_attn_last_error() describes the last
 * failure of the calling thread.  Nothing is launched when a call fails validation.
 */
#ifndef TKM_ATTN_H
#define TKM_ATTN_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#if defined(_WIN32)
#define TKM_ATTN_API
#else
#define TKM_ATTN_API __attribute__((visibility("default")))
#endif

enum { TKM_ATTN_F16 = 0, TKM_ATTN_BF16 = 1 };

enum {
    TKM_ATTN_OK = 0,
    TKM_ATTN_EINVAL = -1,       /* null pointer, non-positive size, Hq % Hkv != 0, bad flag */
    TKM_ATTN_EUNSUPPORTED = -2, /* D not in {64, 128}, unknown dtype, size beyond int range */
    TKM_ATTN_EALIGN = -3,       /* misaligned pointer */
    TKM_ATTN_EWORKSPACE = -4,   /* workspace missing or smaller than required */
    TKM_ATTN_ELAUNCH = -5,      /* the HIP runtime rejected a kernel launch */
    TKM_ATTN_ECOMPILE = -6,     /* hipRTC rejected a generated source */
    TKM_ATTN_EDEVICE = -7       /* no device current, a HIP module/graph call failed, or the
                                   gfx950 assembly kernels failed to load */
};

/* Backward stages.  Two valid schedules:
 *   DELTA, then DKDV and DQ (independent of each other: they may run on two streams);
 *   DQ_DELTA, then DKDV (one stream, one pass over O and dO fewer; what tkm_attn_bwd runs).
 * DELTA writes D = <O, dO> per row into the workspace; DQ_DELTA computes D inside the dQ
 * pass and writes it there; DKDV and DQ read it.  Both also write the row pairs
 * (-LSE*log2(e), -D) that DKDV reads. */
enum { TKM_ATTN_BWD_DELTA = 0, TKM_ATTN_BWD_DKDV = 1, TKM_ATTN_BWD_DQ = 2, TKM_ATTN_BWD_DQ_DELTA = 3 };

/* Forward: O and (if lse != NULL) LSE.
 * Replaces k_gqa_flash_attn_tc_fwd + dispatch, reference src/tkm_gpu.cu:302-438, 1252-1265. */
TKM_ATTN_API int tkm_attn_fwd(const void *qkv, void *o, float *lse, const int32_t *kv_len,
                              int B, int S, int Hq, int Hkv, int D, float scale, int causal,
                              int dtype, void *stream);

/* Bytes of device workspace tkm_attn_bwd needs: the per-row D = <O, dO> vector, and the same
 * rows' -LSE*log2(e) and -D values in tiles of 32 rows per (batch, head), for the dK/dV pass.
 * Replaces the per-node save buffer sizing of init_node_resources, src/tkm_gpu.cu:1000-1001. */
TKM_ATTN_API size_t tkm_attn_bwd_workspace_bytes(int B, int S, int Hq);

/* Backward: dqkv (dQ | dK | dV), overwritten.  lse is the forward's LSE.
 * Replaces k_gqa_flash_attn_tc_bwd + dispatch, reference src/tkm_gpu.cu:440-598, 1389-1404
 * (with the true dK/dV; the reference writes dK := dQ and dV := dO, tkm_gpu.cu:588-596). */
TKM_ATTN_API int tkm_attn_bwd(const void *qkv, const void *o, const void *dout,
                              const float *lse, void *dqkv, const int32_t *kv_len,
                              int B, int S, int Hq, int Hkv, int D, float scale, int causal,
                              int dtype, void *workspace, size_t workspace_bytes, void *stream);

/* tkm_attn_bwd without a workspace argument and without any allocation: the workspace is a
 * static device array of TKM_ATTN_NOALLOC_SCRATCH_BYTES (16 MiB) that each GPU holds from
 * the library's first use on it until the process ends.  No reference counterpart: it is
 * for callers that cannot allocate (code under graph capture, tight serving loops, harnesses
 * that forbid hipMalloc).  Results equal tkm_attn_bwd's bit for bit.
 * Limits: tkm_attn_bwd_workspace_bytes(B, S, Hq) must not exceed the scratch size (about
 * 1.4 million (batch, head, row) triples; config 5's 524288 fit), else TKM_ATTN_EWORKSPACE
 * and nothing runs.  Every call on one GPU shares that GPU's array: calls that overlap on
 * one GPU (other streams, other threads) race, so serialize them.  Nothing needs clearing
 * between calls (the dQ stage writes all the dK/dV stage reads).  tkm_attn_init sets the
 * array up per device; call it before capturing, else the first call on a device does. */
#define TKM_ATTN_NOALLOC_SCRATCH_BYTES (16 << 20)
TKM_ATTN_API int tkm_attn_bwd_noalloc(const void *qkv, const void *o, const void *dout,
                                      const float *lse, void *dqkv, const int32_t *kv_len,
                                      int B, int S, int Hq, int Hkv, int D, float scale,
                                      int causal, int dtype, void *stream);

/* One stage of tkm_attn_bwd (same arguments), for callers that split the backward across
 * streams or time its kernels separately.  No reference counterpart (the reference backward
 * is a single kernel). */
TKM_ATTN_API int tkm_attn_bwd_stage(int stage, const void *qkv, const void *o, const void *dout,
                                    const float *lse, void *dqkv, const int32_t *kv_len,
                                    int B, int S, int Hq, int Hkv, int D, float scale, int causal,
                                    int dtype, void *workspace, size_t workspace_bytes,
                                    void *stream);

/* ---- a paged key-value cache, and attention of one new token over it ----------------------
 *
 * No reference counterpart (it has no decoding path).  The operators of token generation, beside
 * the forward that reads a prompt: tkm_attn_fwd gives the prompt's outputs, tkm_attn_kv_append
 * stores its K and V, then each new token is one append and one tkm_attn_decode per layer.
 *
 * A cache is a pool of pages and, per sequence, a row of a table that names its pages:
 *   k       [num_pages][Hkv][page/32][D/32][32 tokens][32 dims]   16-bit
 *   v       [num_pages][Hkv][page/32][D/32][32 dims][32 tokens]   16-bit
 *   table   [B][max_pages] int32: position j of sequence b is token j % page of page
 *           table[b][j / page]; entries behind the last position in use may hold anything
 *   len     [B] int32: tokens each sequence holds
 *   weight  [B][Hkv][max_pages * page] fp32, or NULL: the attention weight each position of each
 *           kv head has gathered (tkm_attn_decode adds to it, tkm_attn_kv_evict goes by it)
 * page is 32, 64, 128 or 256.  Sequences may share pages that are only read.  Every pointer is a
 * device pointer; k and v are 16-byte aligned, the others 4-byte.
 * table and len are read on the device, so a captured call follows them from replay to replay,
 * and no call checks them on the host.  The kernels do: a page outside [0, num_pages) is never
 * touched, and a length outside [0, max_pages * page] is never walked.  A sequence with one of
 * those that it needs gets O and LSE of NaN, loses the appended rows that fall there, is left as
 * it is by the weights and by eviction, which gives it the length -1.
 * Calls that write a cache must not overlap others on the same cache, and no output may share
 * memory with an input unless stated. */
typedef struct {
    void *k, *v;
    const int32_t *table;
    int32_t *len;
    float *weight;
    int B, Hkv, D, page, max_pages, num_pages, dtype;
} tkm_attn_kv;

/* Stores the K and V rows of qkv [B][S][(Hq + 2*Hkv) * D]: row i < n_new[b] of sequence b goes to
 * position start[b] + i, and len[b] becomes start[b] + n_new[b].  start NULL is len itself (rows
 * go behind what is there); n_new NULL is S, values are clamped to [0, S].  Positions that a table
 * does not reach are dropped, the length counts them; a negative start stores nothing and gives
 * the length -1.  Weights of the stored positions become 0. */
TKM_ATTN_API int tkm_attn_kv_append(const tkm_attn_kv *kv, const void *qkv, int S, int Hq, const int32_t *start,
                                    const int32_t *n_new, void *stream);

/* Bytes of device workspace tkm_attn_decode needs for this cache: the pieces of rows that several
 * workgroups share, at most 256 * 8 * 16 * (D + 2) floats (none for tables of few tokens), and with
 * add_weights the scores, B * Hq * (max_pages * page + 1) floats.  0 also if it refuses the
 * arguments.  It holds nothing from call to call; calls that may overlap need one each. */
TKM_ATTN_API size_t tkm_attn_decode_workspace_bytes(const tkm_attn_kv *kv, int Hq, int add_weights);

/* Attention of one query row a sequence over its len[b] cached positions: o [B][Hq * D] and (if
 * lse != NULL) lse [B][Hq].  q: B rows of Hq * D values, q_stride elements apart (a multiple of
 * 8; the packed row of the new token serves as it is, q_stride = (Hq + 2*Hkv) * D).  A sequence
 * of no tokens gets O = 0, LSE = -inf, and so does a head whose scores are all -inf.  NaN and
 * infinities go where the formula takes them, with exp in fp32: a NaN among a row's scores or a score
 * of +inf makes O and LSE of the head NaN, a NaN value that dim of O; an infinite value makes the dim
 * infinite, or NaN where its exp(score_j - LSE) is 0 or infinities of both signs meet.  What
 * lies behind len[b] may be anything.  Sums are fp32 with weights of up to 2^14: bf16 values beyond
 * 2^114 over the number of tokens may overflow them.  add_weights = 1 also adds, for every position j < len[b]
 * and kv head, the sum over its query heads of exp(score_j - LSE) to weight (nothing for a head
 * whose LSE is -inf or NaN).  Results do not depend on timing. */
TKM_ATTN_API int tkm_attn_decode(const tkm_attn_kv *kv, const void *q, long long q_stride, void *o, float *lse,
                                 int Hq, float scale, int add_weights, void *workspace, size_t workspace_bytes,
                                 void *stream);

/* Cuts every sequence of more than `budget` tokens to that many, each kv head by its own weights:
 * it keeps the first `sink` and the last `recent` positions, and of those between them the
 * budget - sink - recent with the largest weight (equal ones: the earlier position; a NaN counts
 * as less than any other).  What is kept keeps its order, moves to positions 0 .. budget-1 with
 * its weights, and len[b] becomes budget; shorter sequences keep everything.  kept
 * [B][Hkv][budget] receives the old position of each new one, -1 behind the last.
 * dst NULL or src: in place (the pages must not be shared with another sequence; slower by some
 * times for large caches, whose tokens then move in turn).  Otherwise src
 * stays as it is and K, V, weights (if dst has any) and lengths go to dst, which has a table, len
 * and weight of its own, of pages that no sequence of src uses, in the same pool or another. */
TKM_ATTN_API int tkm_attn_kv_evict(const tkm_attn_kv *src, const tkm_attn_kv *dst, int32_t *kept, int budget,
                                   int sink, int recent, void *stream);

/* ---- a serving step: packed rows of several sequences over the paged cache -----------------
 *
 * No reference counterpart.  A step's rows are packed: sequence b has n_new[b] of them, from row
 * row_start[b] on, and what lies behind the last sequence's rows is never written.  In the order of
 * use: tkm_attn_kv_plan once a step (pages, lengths, and for each row its sequence, position and
 * slot), then for each layer tkm_attn_kv_append_rows (rotation, and K and V into that layer's pages)
 * and tkm_attn_chunk.  Layers may share table and len, and so the plan; each has its k and v.
 * As above, all arrays are read on the device, nothing is allocated, and every call may be captured. */

/* Rotary positions: pair i of the first `rot` dims of a head turns by pos * turns[i] * 2^-64 of a
 * circle, (x0, x1) -> factor * (x0 cos - x1 sin, x0 sin + x1 cos); the other dims pass as they are.
 * The product with a position is exact modulo whole turns, so angles hold up to position 2^31 - 1.
 * A plain host struct: fill it with one of the calls below, pass it by address, no device memory. */
enum { TKM_ROPE_HALVES = 0,    /* pair i: dims i and i + rot/2 */
       TKM_ROPE_PAIRS = 1 };   /* pair i: dims 2i and 2i + 1 */
typedef struct {
    int rot, layout;
    float factor;
    uint64_t turns[64];
} tkm_attn_rope;

/* Frequencies f_i = theta^(-2i/rot), in radians a position, and how they are scaled for contexts
 * `scale` >= 1 times longer than the `original` ones of training:
 *   NONE    f_i
 *   LINEAR  f_i / scale
 *   NTK     theta * scale^(rot / (rot - 2)) in theta's place
 *   BANDS   t = (original f_i / 2 pi - low) / (high - low) clamped to [0, 1]: (1 - t) f_i / scale + t f_i
 *   YARN    d(x) = rot ln(original / (2 pi x)) / (2 ln theta), a = max(floor(d(high)), 0),
 *           b = min(ceil(d(low)), rot - 1), t = (i - a) / (b - a, or 0.001 if b <= a) clamped to
 *           [0, 1]: t f_i / scale + (1 - t) f_i; factor 0.1 ln(scale) + 1
 * low and high: BANDS turns over the original context (1, 4), YARN likewise (1, 32).  factor 0:
 * the kind's own (1, but for YARN). */
enum { TKM_ROPE_NONE = 0, TKM_ROPE_LINEAR = 1, TKM_ROPE_NTK = 2, TKM_ROPE_BANDS = 3, TKM_ROPE_YARN = 4 };
typedef struct {
    int rot, layout, scaling;
    double theta, scale, original, low, high, factor;
} tkm_attn_rope_params;

TKM_ATTN_API int tkm_attn_rope_init(const tkm_attn_rope_params *p, tkm_attn_rope *rope);
/* The same from rot/2 frequencies, radians a position, each below 2 pi * 2^31 in size. */
TKM_ATTN_API int tkm_attn_rope_from_freqs(const double *freqs, int rot, int layout, double factor, tkm_attn_rope *rope);

/* Rotates the Q and K heads of `rows` rows of (Hq + 2*Hkv) * D values, strides in elements (multiples
 * of 8); Hkv 0: rows of Q heads.  V is copied.  out == in (and the strides equal): in place, V is left
 * alone.  Row r is at position pos[r], or r % S where pos is NULL; a row of a negative position is
 * left as it is in out.  inverse = 1 turns the other way, which is the gradient: din from dout; with
 * TKM_ROPE_CLEAR added to it, rows of negative positions become 0 in out, all heads of them, as a new
 * tensor needs it.  0 rows launch nothing. */
enum { TKM_ROPE_CLEAR = 256 };
TKM_ATTN_API int tkm_attn_rope_rows(const tkm_attn_rope *rope, const void *in, long long in_stride, void *out,
                                    long long out_stride, const int32_t *pos, int S, int rows, int Hq, int Hkv, int D,
                                    int dtype, int inverse, void *stream);

/* The pages that no sequence has, as a stack, and how many each sequence has; all device arrays. */
typedef struct {
    int32_t *free;      /* [num_pages]; the first *n_free are free, the last of them is taken first */
    int32_t *n_free;    /* [1] */
    int32_t *held;      /* [B]: the pages that each table row names, from its beginning on */
} tkm_attn_pages;

/* What a step does, written by tkm_attn_kv_plan; all device arrays. */
typedef struct {
    int32_t *n_new;       /* [B]: rows of each sequence: what it wanted, or 0 */
    int32_t *row_start;   /* [B + 1]: its first row, and behind the last sequence the number of rows */
    int32_t *seq, *pos;   /* [rows]: each row's sequence and position; -1 behind the last row */
    int64_t *slot;        /* [rows]: page * the page's tokens + token; -1 behind the last row, and where
                             the table has no page of the pool */
} tkm_attn_plan;

/* Makes room for want[b] more tokens of each sequence behind start[b] (NULL: len itself), and lays the
 * step's rows out.  A sequence that holds more pages than start[b] + want[b] tokens need gives the rest
 * back, in the order of sequences and positions, and their table entries become -1: want 0 and start 0
 * end a sequence, want 0 after an eviction frees what it left.  Then, in the order of sequences, each
 * takes the pages that it lacks, if the free ones suffice for it and all that lacked pages before it,
 * and its rows, if they fit into `rows` behind the rows of all before it for whom there were pages; else
 * it gets no page and no row.  So from the first whose pages are missing on, only those that lack none go
 * on, and from the first whose rows do not fit on, none does: a want of more than `rows` holds up all
 * behind it, step after step, until it is cut into pieces.  One that would outgrow its table, wants less
 * than 1, or whose start lies outside the table gets none either, and is not counted.  len[b] becomes
 * start[b] + n_new[b].
 * The tables' pages must be theirs alone.  With start given, a second call of the same step changes
 * nothing.  kv's table and len are written; its k and v are not touched and may be any layer's. */
TKM_ATTN_API int tkm_attn_kv_plan(const tkm_attn_kv *kv, const tkm_attn_pages *pages, const int32_t *want,
                                  const int32_t *start, const tkm_attn_plan *plan, int rows, void *stream);

/* Stores the K and V heads of the plan's rows of qkv (rows `stride` elements apart, a multiple of 8) in
 * their slots, and the Q heads in q (rows q_stride apart; NULL: nowhere; qkv itself with its stride: in
 * place), Q and K rotated to the rows' positions if rope is not NULL.  Rows of a negative position are
 * left alone; a slot outside the pool is not written.  Weights of the stored positions become 0 (rows of
 * a sequence or position outside the tables are passed over there).  len is not touched.  Of plan, seq, pos and slot are
 * read; slots of two rows must differ. */
TKM_ATTN_API int tkm_attn_kv_append_rows(const tkm_attn_kv *kv, const tkm_attn_rope *rope, const void *qkv,
                                         long long stride, void *q, long long q_stride, const tkm_attn_plan *plan,
                                         int rows, int Hq, void *stream);

/* Bytes of device workspace tkm_attn_chunk needs; 0 if none (short tables, few rows), also if it refuses
 * the arguments.  It holds nothing from call to call; calls that may overlap need one each.
 * Like the call's form, it goes by what the tables could hold, not by what sequences do: where they are
 * short, tables of up to 2048 tokens (640 for few rows) spare them two launches, about 20 us. */
TKM_ATTN_API size_t tkm_attn_chunk_workspace_bytes(const tkm_attn_kv *kv, int rows, int Hq);

/* Attention of each sequence's new rows over its len[b] cached positions, their own among them: row i
 * of n_new[b] stands at position p = len[b] - n_new[b] + i and sees the positions j < len[b], with
 * causal = 1 those of j <= p, and with window > 0 (causal only) of these j > p - window.
 * q: `rows` rows (1 at least: a step without rows leaves the call out) of Hq * D values, q_stride
 * elements apart (a multiple of 8); o [rows][Hq * D]; lse [rows][Hq] or NULL.  Sequence b has the rows
 * row_start[b] .. row_start[b] + n_new[b] - 1; row_start NULL: from b * (rows / B) on, of which n_new[b]
 * (clamped to rows / B) are its rows; n_new NULL (only then): all.  A sequence that begins outside
 * [0, rows) has no rows, and rows behind them are passed over; no two sequences may have a row, and o
 * must not overlap q.  Rows of no sequence stay as they are in o and lse.
 * A row that sees nothing gets O = 0, LSE = -inf.  What a row does not see has no part in it, whatever
 * it holds; what it sees of NaN and infinities acts as in tkm_attn_decode, and so do lengths and pages
 * outside their bounds.  Infinities and NaN among the values cost a second walk.  No weights are gathered:
 * positions that only these rows attend to keep the 0 that tkm_attn_kv_append_rows gave them, and
 * tkm_attn_kv_evict drops them before all that tkm_attn_decode has added to, but for its sink and recent.
 * Scores, softmax and sums are fp32; the weights are multiplied with the values as 16-bit parts of together
 * 22 bits (fp16) or 24 (bf16), as in tkm_attn_decode.  The sums hold weights of up to 2^16: values of more
 * than 2^100 may overflow in them.  Results do not depend on timing. */
TKM_ATTN_API int tkm_attn_chunk(const tkm_attn_kv *kv, const void *q, long long q_stride, const int32_t *row_start,
                                const int32_t *n_new, int rows, void *o, float *lse, int Hq, float scale, int causal,
                                int window, void *workspace, size_t workspace_bytes, void *stream);

/* Loads this library's gfx950 assembly kernels (D = 128, fp16 and bf16) on the current device.  Call
 * it once per device before capturing a graph, as the runtime does at ignite; otherwise the
 * first call on a device loads them (inside a capture, with the thread's capture mode
 * relaxed so that nothing is recorded).  Returns TKM_ATTN_OK (also on a device that is not
 * gfx950, where the HIP kernels serve every shape) or TKM_ATTN_EDEVICE when a code object
 * fails to load; the calls that need them then fail with TKM_ATTN_EDEVICE too, they never
 * switch to the slower kernels.  No reference counterpart (the reference JIT-compiles its
 * generated kernels at ignite, src/tkm_gpu.cu:1047-1078; its attention kernels are
 * compiled ahead of time). */
TKM_ATTN_API int tkm_attn_init(void);

/* 1 if the assembly kernels are loaded on the current device (gfx950), else 0. */
TKM_ATTN_API int tkm_attn_asm_available(void);

/* Kernels launched by the calling thread's last tkm_attn_fwd / _bwd / _bwd_stage /
 * _decode / _kv_append / _kv_evict / _rope_rows / _kv_plan / _kv_append_rows / _chunk call
 * (OR of the bits below; 0 after a call that failed validation).  No reference counterpart. */
enum {
    TKM_ATTN_K_FWD_ASM = 1,     /* tkm_fa_fwd_d128_f16 (assembly) */
    TKM_ATTN_K_FWD_HIP = 2,     /* fa_fwd_kernel (HIP) */
    TKM_ATTN_K_DQ_ASM = 4,      /* tkm_fa_bwd_dq_d128_f16 (assembly) */
    TKM_ATTN_K_DQ_HIP = 8,      /* fa_bwd_dq_kernel (HIP) */
    TKM_ATTN_K_DKDV_ASM = 16,   /* tkm_fa_bwd_dkdv_d128_f16 (assembly) */
    TKM_ATTN_K_DKDV_HIP = 32,   /* fa_bwd_dkdv_kernel (HIP) */
    TKM_ATTN_K_DELTA_HIP = 64,  /* fa_bwd_delta_kernel (HIP) */
    TKM_ATTN_K_DECODE = 128,    /* decode_kernel */
    TKM_ATTN_K_JOIN = 256,      /* join_kernel: rows that several workgroups of it shared */
    TKM_ATTN_K_WEIGHTS = 512,   /* join_weights_kernel: the same, with the weights (JOIN is set too) */
    TKM_ATTN_K_APPEND = 1024,   /* append_*_kernel */
    TKM_ATTN_K_EVICT = 2048,    /* select_kernel, move_kernel */
    TKM_ATTN_K_ROPE = 4096,     /* rope_kernel */
    TKM_ATTN_K_PLAN = 8192,     /* plan_kernel, slots_kernel */
    TKM_ATTN_K_CHUNK = 16384    /* chunk_kernel (JOIN is set too where rows may be shared) */
};
TKM_ATTN_API unsigned tkm_attn_last_kernels(void);

/* Static description of a status code, and the last failure message of this thread. */
TKM_ATTN_API const char *tkm_attn_status_string(int status);
TKM_ATTN_API const char *tkm_attn_last_error(void);

/* ABI version: major * 10000 + minor * 100 + patch. */
TKM_ATTN_API int tkm_attn_version(void);

#ifdef __cplusplus
}
#endif
#endif /* TKM_ATTN_H */
