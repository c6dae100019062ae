/*
 * tkm_rope.c -- frequencies of the rotary positions declared in include/tkm_attn.h, on the host.
 *
 * A pair's frequency is kept as the part of a circle that it turns by a position, in units of 2^-64:
 * pos * turns then wraps around just as the angle does, so that the kernels form the angle of any
 * position by integer products, exactly.  In long double (64 bits of mantissa): a frequency of at most 1
 * radian, 0.16 of a circle, is formed in up to 16 roundings of 2^-64 of itself and cut to whole units, so that
 * it is off by less than 2^-62 of a circle (plain ones by less than 2^-64), at position 2^31 by 2^-31 (2^-33).
 */
#include <math.h>
#include <string.h>

#include "tkm_prep.h"
#include "tkm_prep_internal.h"

static const long double kCircle = 6.283185307179586476925286766559L;

static int check_shape(int rot, int layout, double factor) {
    if (rot < 2 || rot > 128 || rot % 2 != 0)
        return tkm_set_error(TKM_ATTN_EINVAL, "rot=%d must be even, 2 to 128", rot);
    if (layout != TKM_ROPE_HALVES && layout != TKM_ROPE_PAIRS)
        return tkm_set_error(TKM_ATTN_EINVAL, "layout %d (TKM_ROPE_HALVES, TKM_ROPE_PAIRS)", layout);
    if (!(factor >= 0.0) || !isfinite((float)factor) || (factor != 0.0 && (float)factor == 0.0f))
        return tkm_set_error(TKM_ATTN_EINVAL, "factor must be 0 or positive, and neither infinite nor 0 in fp32");
    return TKM_ATTN_OK;
}

static uint64_t turns_of(long double freq) {
    long double x = freq / kCircle;
    x = (x - floorl(x)) * 0x1p64L;
    return x < 0x1p64L ? (uint64_t)x : 0;     /* a tiny negative frequency rounds up to the whole circle */
}

TKM_ATTN_API int tkm_attn_rope_from_freqs(const double *freqs, int rot, int layout, double factor, tkm_attn_rope *rope) {
    if (!freqs || !rope) return tkm_set_error(TKM_ATTN_EINVAL, "freqs and rope must be non-null");
    const int rc = check_shape(rot, layout, factor);
    if (rc) return rc;
    for (int i = 0; i < rot / 2; ++i)
        if (!(fabs(freqs[i]) < 6.283185307179586 * 2147483648.0))
            return tkm_set_error(TKM_ATTN_EINVAL, "frequency %d is too large or not a number", i);
    memset(rope, 0, sizeof *rope);
    rope->rot = rot;
    rope->layout = layout;
    rope->factor = factor == 0.0 ? 1.0f : (float)factor;
    for (int i = 0; i < rot / 2; ++i) rope->turns[i] = turns_of(freqs[i]);
    return TKM_ATTN_OK;
}

static long double ramp(long double x) { return x < 0.0L ? 0.0L : x > 1.0L ? 1.0L : x; }

TKM_ATTN_API int tkm_attn_rope_init(const tkm_attn_rope_params *p, tkm_attn_rope *rope) {
    if (!p || !rope) return tkm_set_error(TKM_ATTN_EINVAL, "the parameters and rope must be non-null");
    const int rc = check_shape(p->rot, p->layout, p->factor);
    if (rc) return rc;
    const int kind = p->scaling, rot = p->rot;
    if (kind < TKM_ROPE_NONE || kind > TKM_ROPE_YARN) return tkm_set_error(TKM_ATTN_EINVAL, "scaling %d (TKM_ROPE_*)", kind);
    /* theta < 1 would give frequencies that grow past any bound */
    if (!(p->theta >= 1.0) || !isfinite(p->theta)) return tkm_set_error(TKM_ATTN_EINVAL, "theta must be finite and at least 1");
    if (kind != TKM_ROPE_NONE && (!(p->scale >= 1.0) || !isfinite(p->scale)))
        return tkm_set_error(TKM_ATTN_EINVAL, "scale must be finite and at least 1");
    if (kind == TKM_ROPE_BANDS || kind == TKM_ROPE_YARN) {
        if (!(p->original > 0.0) || !isfinite(p->original) || !(p->low > 0.0) || !(p->high > p->low) || !isfinite(p->high))
            return tkm_set_error(TKM_ATTN_EINVAL, "scaling needs original > 0 and 0 < low < high");
        if (kind == TKM_ROPE_YARN && !(p->theta > 1.0)) return tkm_set_error(TKM_ATTN_EINVAL, "this scaling needs theta > 1");
    }
    memset(rope, 0, sizeof *rope);
    rope->rot = rot;
    rope->layout = p->layout;
    rope->factor = p->factor != 0.0 ? (float)p->factor : kind == TKM_ROPE_YARN ? (float)(0.1 * log(p->scale) + 1.0) : 1.0f;
    const long double s = p->scale, wide = p->original;
    long double theta = p->theta, a = 0.0L, b = 0.0L;
    if (kind == TKM_ROPE_NTK && rot > 2) theta *= powl(s, (long double)rot / (rot - 2));
    if (kind == TKM_ROPE_YARN) {
        a = floorl(rot * logl(wide / (kCircle * p->high)) / (2.0L * logl(theta)));
        b = ceill(rot * logl(wide / (kCircle * p->low)) / (2.0L * logl(theta)));
        if (a < 0.0L) a = 0.0L;
        if (b > rot - 1) b = rot - 1;
    }
    for (int i = 0; i < rot / 2; ++i) {
        long double f = powl(theta, -2.0L * i / rot), t;
        if (kind == TKM_ROPE_LINEAR) f /= s;
        if (kind == TKM_ROPE_BANDS) {
            t = ramp((wide * f / kCircle - p->low) / ((long double)p->high - p->low));
            f = (1.0L - t) * f / s + t * f;
        }
        if (kind == TKM_ROPE_YARN) {
            t = ramp((i - a) / (b > a ? b - a : 0.001L));
            f = t * f / s + (1.0L - t) * f;
        }
        rope->turns[i] = turns_of(f);
    }
    return TKM_ATTN_OK;
}

TKM_ATTN_API int tkm_prep_rope(const tkm_prep_desc *d, tkm_attn_rope *rope) {
    const int rc = tkm_prep_check_desc(d);
    if (rc) return rc;
    if (!d->has_rope) return tkm_set_error(TKM_ATTN_EINVAL, "the descriptor has no RoPE");
    double f[64];
    for (int i = 0; i < d->head_dim / 2; ++i) f[i] = tkm_rope_inv_freq(d, i);
    return tkm_attn_rope_from_freqs(f, d->head_dim, TKM_ROPE_PAIRS, 1.0, rope);
}
