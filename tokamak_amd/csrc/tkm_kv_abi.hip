// tkm_kv_abi.hip -- the extern "C" entry points of the paged key-value cache declared in
// include/tkm_attn.h: argument validation, then the launchers of attn_kv.h.
#include <math.h>
#include <stdarg.h>

#include "attn_kv.h"
#include "attn_launch.h"
#include "tkm_prep_internal.h"

namespace {

int fail(int status, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
int fail(int status, const char* fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    tkm_vset_error(status, fmt, ap);
    va_end(ap);
    return status;
}

bool aligned(const void* p, size_t a) { return ((uintptr_t)p % a) == 0; }

int check_kv(const tkm_attn_kv* kv) {
    if (!kv) return fail(TKM_ATTN_EINVAL, "the cache must be non-null");
    if (!kv->k || !kv->v || !kv->table || !kv->len)
        return fail(TKM_ATTN_EINVAL, "the cache's k, v, table and len must be non-null");
    if (kv->B < 1 || kv->Hkv < 1 || kv->num_pages < 1 || kv->max_pages < 1)
        return fail(TKM_ATTN_EINVAL, "sizes must be positive (B=%d Hkv=%d num_pages=%d max_pages=%d)", kv->B, kv->Hkv,
                    kv->num_pages, kv->max_pages);
    if (kv->D != 64 && kv->D != 128) return fail(TKM_ATTN_EUNSUPPORTED, "head dim D=%d (supported: 64, 128)", kv->D);
    if (kv->dtype != TKM_ATTN_F16 && kv->dtype != TKM_ATTN_BF16)
        return fail(TKM_ATTN_EUNSUPPORTED, "dtype %d (supported: TKM_ATTN_F16, TKM_ATTN_BF16)", kv->dtype);
    if (kv->page != 32 && kv->page != 64 && kv->page != 128 && kv->page != 256)
        return fail(TKM_ATTN_EUNSUPPORTED, "pages of %d tokens (supported: 32, 64, 128, 256)", kv->page);
    if ((double)kv->max_pages * kv->page > 1073741824.0)
        return fail(TKM_ATTN_EUNSUPPORTED, "a table of %d pages of %d tokens is too large", kv->max_pages, kv->page);
    if ((double)kv->B * kv->Hkv > 16777216.0) return fail(TKM_ATTN_EUNSUPPORTED, "B * Hkv is too large");
    if (!aligned(kv->k, 16) || !aligned(kv->v, 16) || !aligned(kv->table, 4) || !aligned(kv->len, 4) ||
        !aligned(kv->weight, 4))
        return fail(TKM_ATTN_EALIGN, "the cache's k and v must be 16-byte aligned, table, len and weight 4-byte");
    return TKM_ATTN_OK;
}

int check_heads(const tkm_attn_kv* kv, int Hq) {
    if (Hq < 1) return fail(TKM_ATTN_EINVAL, "sizes must be positive (Hq=%d)", Hq);
    if (Hq % kv->Hkv != 0) return fail(TKM_ATTN_EINVAL, "Hq=%d is not a multiple of Hkv=%d", Hq, kv->Hkv);
    if ((double)kv->B * Hq * kv->D > 1073741824.0) return fail(TKM_ATTN_EUNSUPPORTED, "B * Hq * D is too large");
    return TKM_ATTN_OK;
}

int check_decode(const tkm_attn_kv* kv, int Hq, int add_weights) {
    int rc = check_kv(kv);
    if (!rc) rc = check_heads(kv, Hq);
    if (rc) return rc;
    if (tkm::decode_tiles_most(*kv, Hq) > 1073741824.0)
        return fail(TKM_ATTN_EUNSUPPORTED, "the cache's tables hold too many tiles of 32 tokens");
    if (!tkm::decode_fits(*kv, Hq, add_weights)) return fail(TKM_ATTN_EUNSUPPORTED, "grid too large");
    return TKM_ATTN_OK;
}

int check_chunk(const tkm_attn_kv* kv, int rows, int Hq) {
    int rc = check_kv(kv);
    if (rc) return rc;
    if (rows < 1) return fail(TKM_ATTN_EINVAL, "sizes must be positive (rows=%d)", rows);
    if (Hq < 1) return fail(TKM_ATTN_EINVAL, "sizes must be positive (Hq=%d)", Hq);
    if (Hq % kv->Hkv != 0) return fail(TKM_ATTN_EINVAL, "Hq=%d is not a multiple of Hkv=%d", Hq, kv->Hkv);
    if (!tkm::chunk_fits(*kv, rows, Hq)) return fail(TKM_ATTN_EUNSUPPORTED, "rows * Hq / Hkv is too large");
    return TKM_ATTN_OK;
}

int check_rope(const tkm_attn_rope* r, int D) {
    if (r->rot < 2 || r->rot > D || r->rot % 2 != 0)
        return fail(TKM_ATTN_EINVAL, "rot=%d must be even, 2 to the head dim %d", r->rot, D);
    if (r->layout != TKM_ROPE_HALVES && r->layout != TKM_ROPE_PAIRS)
        return fail(TKM_ATTN_EINVAL, "layout %d (TKM_ROPE_HALVES, TKM_ROPE_PAIRS)", r->layout);
    return TKM_ATTN_OK;
}

bool row_stride_ok(long long stride, double width) { return stride % 8 == 0 && (double)stride >= width; }

}  // namespace

extern "C" {

TKM_ATTN_API int tkm_attn_rope_rows(const tkm_attn_rope* rope, const void* in, long long in_stride, void* out,
                                    long long out_stride, const int32_t* pos, int S, int rows, int Hq, int Hkv, int D,
                                    int dtype, int inverse, void* stream) {
    tkm::reset_kernels();
    if (!rope) return fail(TKM_ATTN_EINVAL, "rope must be non-null");
    if (rows < 0 || Hq < 1 || Hkv < 0) return fail(TKM_ATTN_EINVAL, "sizes must be positive (rows=%d Hq=%d Hkv=%d)", rows, Hq, Hkv);
    if (D != 64 && D != 128) return fail(TKM_ATTN_EUNSUPPORTED, "head dim D=%d (supported: 64, 128)", D);
    if (dtype != TKM_ATTN_F16 && dtype != TKM_ATTN_BF16)
        return fail(TKM_ATTN_EUNSUPPORTED, "dtype %d (supported: TKM_ATTN_F16, TKM_ATTN_BF16)", dtype);
    const int rc = check_rope(rope, D);
    if (rc) return rc;
    if ((inverse & ~TKM_ROPE_CLEAR) != 0 && (inverse & ~TKM_ROPE_CLEAR) != 1)
        return fail(TKM_ATTN_EINVAL, "inverse must be 0 or 1 (and TKM_ROPE_CLEAR), got %d", inverse);
    if (!pos && S < 1) return fail(TKM_ATTN_EINVAL, "without positions S=%d must be positive", S);
    const double width = ((double)Hq + 2.0 * Hkv) * D;
    if (width > 1073741824.0) return fail(TKM_ATTN_EUNSUPPORTED, "rows are too wide");
    if (!row_stride_ok(in_stride, width) || !row_stride_ok(out_stride, width))
        return fail(TKM_ATTN_EINVAL, "row strides %lld and %lld must be multiples of 8 and at least the row", in_stride, out_stride);
    if (in == out && in_stride != out_stride) return fail(TKM_ATTN_EINVAL, "in place both strides must be the same");
    if (rows == 0) return TKM_ATTN_OK;
    if (!in || !out) return fail(TKM_ATTN_EINVAL, "in and out must be non-null");
    if (!aligned(in, 16) || !aligned(out, 16) || !aligned(pos, 4))
        return fail(TKM_ATTN_EALIGN, "in and out must be 16-byte aligned, pos 4-byte");
    if (!tkm::rows_fit(nullptr, rows)) return fail(TKM_ATTN_EUNSUPPORTED, "grid too large");
    const tkm::RopeArgs a{*rope, in, in_stride, out, out_stride, pos, S, rows, Hq, Hkv, D, dtype, inverse & 1, inverse & TKM_ROPE_CLEAR, stream};
    if (tkm::launch_rope(a)) return fail(TKM_ATTN_ELAUNCH, "rope: kernel launch failed");
    return TKM_ATTN_OK;
}

TKM_ATTN_API int tkm_attn_kv_plan(const tkm_attn_kv* kv, const tkm_attn_pages* pages, const int32_t* want,
                                  const int32_t* start, const tkm_attn_plan* plan, int rows, void* stream) {
    tkm::reset_kernels();
    const int rc = check_kv(kv);
    if (rc) return rc;
    if (!pages || !pages->free || !pages->n_free || !pages->held)
        return fail(TKM_ATTN_EINVAL, "the pages' free, n_free and held must be non-null");
    if (!plan || !plan->n_new || !plan->row_start) return fail(TKM_ATTN_EINVAL, "the plan's n_new and row_start must be non-null");
    if (!want) return fail(TKM_ATTN_EINVAL, "want must be non-null");
    if (rows < 0) return fail(TKM_ATTN_EINVAL, "rows=%d must not be negative", rows);
    if (rows && (!plan->seq || !plan->pos || !plan->slot)) return fail(TKM_ATTN_EINVAL, "the plan's seq, pos and slot must be non-null");
    for (const void* p : {(const void*)pages->free, (const void*)pages->n_free, (const void*)pages->held, (const void*)want,
                          (const void*)start, (const void*)plan->n_new, (const void*)plan->row_start, (const void*)plan->seq,
                          (const void*)plan->pos})
        if (!aligned(p, 4)) return fail(TKM_ATTN_EALIGN, "the arrays of int32 must be 4-byte aligned");
    if (!aligned(plan->slot, 8)) return fail(TKM_ATTN_EALIGN, "slot must be 8-byte aligned");
    if (want == plan->n_new || want == kv->len || want == start)
        return fail(TKM_ATTN_EINVAL, "want must not be another of the call's arrays");
    if (start == kv->len) start = nullptr;
    const tkm::PlanArgs a{*kv, *pages, want, start, *plan, rows, stream};
    if (tkm::launch_plan(a)) return fail(TKM_ATTN_ELAUNCH, "plan: kernel launch failed");
    return TKM_ATTN_OK;
}

TKM_ATTN_API int tkm_attn_kv_append_rows(const tkm_attn_kv* kv, const tkm_attn_rope* rope, const void* qkv, long long stride,
                                         void* q, long long q_stride, const tkm_attn_plan* plan, int rows, int Hq, void* stream) {
    tkm::reset_kernels();
    int rc = check_kv(kv);
    if (rc) return rc;
    if (rows < 0 || Hq < 1) return fail(TKM_ATTN_EINVAL, "sizes must be positive (rows=%d Hq=%d)", rows, Hq);
    if (Hq % kv->Hkv != 0) return fail(TKM_ATTN_EINVAL, "Hq=%d is not a multiple of Hkv=%d", Hq, kv->Hkv);
    if (rope && (rc = check_rope(rope, kv->D))) return rc;
    const double width = ((double)Hq + 2.0 * kv->Hkv) * kv->D;
    if (width > 1073741824.0) return fail(TKM_ATTN_EUNSUPPORTED, "rows are too wide");
    if (!row_stride_ok(stride, width)) return fail(TKM_ATTN_EINVAL, "stride=%lld must be a multiple of 8 and at least the row", stride);
    if (q && !row_stride_ok(q_stride, (double)Hq * kv->D))
        return fail(TKM_ATTN_EINVAL, "q_stride=%lld must be a multiple of 8 and at least Hq * D", q_stride);
    if (q && q == qkv && q_stride != stride) return fail(TKM_ATTN_EINVAL, "in place both strides must be the same");
    if (rows == 0) return TKM_ATTN_OK;
    if (!qkv || !plan || !plan->seq || !plan->pos || !plan->slot)
        return fail(TKM_ATTN_EINVAL, "qkv and the plan's seq, pos and slot must be non-null");
    if (!aligned(qkv, 16) || !aligned(q, 16) || !aligned(plan->seq, 4) || !aligned(plan->pos, 4) || !aligned(plan->slot, 8))
        return fail(TKM_ATTN_EALIGN, "qkv and q must be 16-byte aligned, seq and pos 4-byte, slot 8-byte");
    if (!tkm::rows_fit(kv, rows)) return fail(TKM_ATTN_EUNSUPPORTED, "grid too large");
    const tkm::StoreArgs a{*kv, rope, qkv, stride, q, q_stride, plan->seq, plan->pos, plan->slot, rows, Hq, stream};
    if (tkm::launch_store(a)) return fail(TKM_ATTN_ELAUNCH, "append: kernel launch failed");
    return TKM_ATTN_OK;
}

TKM_ATTN_API size_t tkm_attn_chunk_workspace_bytes(const tkm_attn_kv* kv, int rows, int Hq) {
    return check_chunk(kv, rows, Hq) ? 0 : tkm::chunk_workspace(*kv, rows, Hq);
}

TKM_ATTN_API int tkm_attn_chunk(const tkm_attn_kv* kv, const void* q, long long q_stride, const int32_t* row_start,
                                const int32_t* n_new, int rows, void* o, float* lse, int Hq, float scale, int causal, int window,
                                void* workspace, size_t workspace_bytes, void* stream) {
    tkm::reset_kernels();
    const int rc = check_chunk(kv, rows, Hq);
    if (rc) return rc;
    if (!q || !o) return fail(TKM_ATTN_EINVAL, "q and o must be non-null");
    if (row_start && !n_new) return fail(TKM_ATTN_EINVAL, "row_start needs n_new");
    if (!row_start && rows % kv->B != 0)
        return fail(TKM_ATTN_EINVAL, "without row_start the %d rows must be the same number for each of the %d sequences", rows, kv->B);
    if (causal != 0 && causal != 1) return fail(TKM_ATTN_EINVAL, "causal must be 0 or 1, got %d", causal);
    if (window < 0 || (window && !causal)) return fail(TKM_ATTN_EINVAL, "window=%d must not be negative, and needs causal", window);
    if (!row_stride_ok(q_stride, (double)Hq * kv->D))
        return fail(TKM_ATTN_EINVAL, "q_stride=%lld must be a multiple of 8 and at least Hq * D", q_stride);
    if (!aligned(q, 16) || !aligned(o, 16) || !aligned(lse, 4) || !aligned(row_start, 4) || !aligned(n_new, 4))
        return fail(TKM_ATTN_EALIGN, "q and o must be 16-byte aligned, lse, row_start and n_new 4-byte");
    if (!(scale > 0.f) || scale * 1.4426950408889634f == INFINITY)     // scores are in log2 units
        return fail(TKM_ATTN_EINVAL, "scale must be positive and finite, also times log2(e)");
    const size_t need = tkm::chunk_workspace(*kv, rows, Hq);
    if (need && (!workspace || workspace_bytes < need))
        return fail(TKM_ATTN_EWORKSPACE, "workspace of %zu bytes required, %zu given", need, workspace ? workspace_bytes : (size_t)0);
    if (need && !aligned(workspace, 16)) return fail(TKM_ATTN_EALIGN, "workspace must be 16-byte aligned");
    const tkm::ChunkArgs a{*kv, q, q_stride, row_start, n_new, rows, o, lse, Hq, scale, causal, window, workspace, stream};
    if (tkm::launch_chunk(a)) return fail(TKM_ATTN_ELAUNCH, "chunk: kernel launch failed");
    return TKM_ATTN_OK;
}

TKM_ATTN_API int tkm_attn_kv_append(const tkm_attn_kv* kv, const void* qkv, int S, int Hq, const int32_t* start,
                                    const int32_t* n_new, void* stream) {
    tkm::reset_kernels();
    int rc = check_kv(kv);
    if (rc) return rc;
    if (!qkv) return fail(TKM_ATTN_EINVAL, "qkv must be non-null");
    if (S < 1) return fail(TKM_ATTN_EINVAL, "sizes must be positive (S=%d)", S);
    if ((rc = check_heads(kv, Hq))) return rc;
    if (!aligned(qkv, 16) || !aligned(start, 4) || !aligned(n_new, 4))
        return fail(TKM_ATTN_EALIGN, "qkv must be 16-byte aligned, start and n_new 4-byte");
    if (n_new == kv->len) return fail(TKM_ATTN_EINVAL, "n_new must not be the cache's own len");
    if (!tkm::append_fits(*kv, S)) return fail(TKM_ATTN_EUNSUPPORTED, "grid too large");
    if (start == kv->len) start = nullptr;
    const tkm::AppendArgs a{*kv, qkv, S, Hq, start, n_new, stream};
    if (tkm::launch_append(a)) return fail(TKM_ATTN_ELAUNCH, "append: kernel launch failed");
    return TKM_ATTN_OK;
}

TKM_ATTN_API size_t tkm_attn_decode_workspace_bytes(const tkm_attn_kv* kv, int Hq, int add_weights) {
    return check_decode(kv, Hq, add_weights != 0) ? 0 : tkm::decode_workspace(*kv, Hq, add_weights);
}

TKM_ATTN_API int tkm_attn_decode(const tkm_attn_kv* kv, const void* q, long long q_stride, void* o, float* lse, int Hq,
                                 float scale, int add_weights, void* workspace, size_t workspace_bytes, void* stream) {
    tkm::reset_kernels();
    int rc = check_decode(kv, Hq, add_weights != 0);
    if (rc) return rc;
    if (!q || !o) return fail(TKM_ATTN_EINVAL, "q and o must be non-null");
    if (add_weights != 0 && add_weights != 1) return fail(TKM_ATTN_EINVAL, "add_weights must be 0 or 1, got %d", add_weights);
    if (add_weights && !kv->weight) return fail(TKM_ATTN_EINVAL, "add_weights needs a cache with weights");
    if (q_stride < (long long)Hq * kv->D || q_stride % 8 != 0)
        return fail(TKM_ATTN_EINVAL, "q_stride=%lld must be a multiple of 8 and at least Hq * D", q_stride);
    if (!aligned(q, 16) || !aligned(o, 16) || !aligned(lse, 4))
        return fail(TKM_ATTN_EALIGN, "q and o must be 16-byte aligned, lse 4-byte");
    if (!(scale > 0.f) || scale * 1.4426950408889634f == INFINITY)     // scores are in log2 units
        return fail(TKM_ATTN_EINVAL, "scale must be positive and finite, also times log2(e)");
    const size_t need = tkm::decode_workspace(*kv, Hq, add_weights);
    if (need && (!workspace || workspace_bytes < need))
        return fail(TKM_ATTN_EWORKSPACE, "workspace of %zu bytes required, %zu given", need,
                    workspace ? workspace_bytes : (size_t)0);
    if (need && !aligned(workspace, 16)) return fail(TKM_ATTN_EALIGN, "workspace must be 16-byte aligned");
    const tkm::DecodeArgs a{*kv, q, q_stride, o, lse, Hq, scale, add_weights, workspace, stream};
    if (tkm::launch_decode(a)) return fail(TKM_ATTN_ELAUNCH, "decode: kernel launch failed");
    return TKM_ATTN_OK;
}

TKM_ATTN_API int tkm_attn_kv_evict(const tkm_attn_kv* src, const tkm_attn_kv* dst, int32_t* kept, int budget, int sink,
                                   int recent, void* stream) {
    tkm::reset_kernels();
    int rc = check_kv(src);
    if (rc) return rc;
    if (dst && (rc = check_kv(dst))) return rc;
    if (!dst) dst = src;
    const bool in_place = dst->table == src->table;
    if (!src->weight) return fail(TKM_ATTN_EINVAL, "eviction needs a cache with weights");
    if (!kept) return fail(TKM_ATTN_EINVAL, "kept must be non-null");
    if (!aligned(kept, 4)) return fail(TKM_ATTN_EALIGN, "kept must be 4-byte aligned");
    if (dst->B != src->B || dst->Hkv != src->Hkv || dst->D != src->D || dst->page != src->page || dst->dtype != src->dtype)
        return fail(TKM_ATTN_EINVAL, "both caches must have the same B, Hkv, D, page and dtype");
    if (in_place && (dst->k != src->k || dst->v != src->v || dst->len != src->len || dst->weight != src->weight ||
                     dst->max_pages != src->max_pages || dst->num_pages != src->num_pages))
        return fail(TKM_ATTN_EINVAL, "in place both caches must be the same");
    if (!in_place && (dst->len == src->len || dst->weight == src->weight))
        return fail(TKM_ATTN_EINVAL, "a cache with a table of its own needs its own len and weight");
    if (budget < 1 || sink < 0 || recent < 0 || sink > budget || recent > budget - sink)
        return fail(TKM_ATTN_EINVAL, "budget=%d must hold sink=%d and recent=%d", budget, sink, recent);
    if ((double)budget > (double)dst->max_pages * dst->page)
        return fail(TKM_ATTN_EINVAL, "budget=%d exceeds the %d pages of a table", budget, dst->max_pages);
    if (!tkm::evict_fits(*src, *dst, budget)) return fail(TKM_ATTN_EUNSUPPORTED, "grid too large");
    const tkm::EvictArgs a{*src, *dst, kept, budget, sink, recent, stream};
    if (tkm::launch_evict(a)) return fail(TKM_ATTN_ELAUNCH, "evict: kernel launch failed");
    return TKM_ATTN_OK;
}

}  // extern "C"
