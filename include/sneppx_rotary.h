/*
 * sneppx_rotary.h - positions of queries and keys on gfx950: every head turned
 * to its token's position, normalised first where that is asked for, in one pass
 * between the QKV projection and the key-value cache (sneppx_kv.h).
 *
 *   x = x / sqrt(mean(x^2) + eps) * norm[d]          (where norm is given)
 *   (a, b) = (a cos - b sin, b cos + a sin) * magnitude
 *
 * for the dims / 2 pairs (a, b) of the head's first `dims` elements, by the angle
 * position * freqs[pair]; the elements behind them are left as they are.  Angles
 * and their sines and cosines are taken in fp64 (a position of 10^6 has no fraction of a
 * turn left in fp32) and rounded to fp32 with the magnitude; everything else is fp32
 * (elements whose squares pass its range, from 10^19 on, have an infinite mean), with one
 * rounding at the end.
 *
 * The reference has rotary positions on the CPU (SNEPPX_rope_precompute, called at
 * kernel/inference/inference_engine.c:247).
 * Pointers are DEVICE pointers unless stated, calls are asynchronous on
 * `stream`, allocate nothing and return 0, or -1 with the reason in
 * SNEPPX_qlinear_last_error().
 */
#ifndef SNEPPX_ROTARY_H
#define SNEPPX_ROTARY_H

#include <stddef.h>
#include <stdint.h>

#include "sneppx_qlinear.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef struct {
    const double* freqs;   /* [dims / 2] radians per position, 16-byte aligned */
    size_t dims;           /* rotated elements of a head, a multiple of 8; 0: none (freqs may be NULL) */
    int interleaved;       /* pairs (2 i, 2 i + 1); else (i, i + dims / 2) */
    float magnitude;       /* factor of cos and sin, 1 without scaling */
    const float* q_norm;   /* [head_dim] factors of the queries' norm, 16-byte aligned, or NULL: no norm */
    const float* k_norm;   /* the same of the keys */
    float eps;
} SNEPPXRotary;

/* How frequencies base^(-2 i / dims) are changed for contexts longer than the
 * `original` positions that a model was trained on. */
typedef enum {
    SNEPPX_ROTARY_PLAIN = 0,
    SNEPPX_ROTARY_LINEAR = 1,  /* all / factor */
    SNEPPX_ROTARY_BASE = 2,    /* base * factor^(dims / (dims - 2)): the lowest / factor, the highest as they are */
    SNEPPX_ROTARY_BANDS = 3,   /* by the turns over `original` positions: below `low` / factor, from `high` on as
                                  they are, in between in proportion to the turns */
    SNEPPX_ROTARY_RAMP = 4     /* the same with `low` and `high` turns, in between in proportion to the pair's
                                  index, and a magnitude of 1 + ln(factor) / 10 */
} SNEPPXRotaryScaling;

/* freqs (HOST, [dims / 2]) and *magnitude (HOST, may be NULL).  factor >= 1;
 * original, low < high of the two last kinds (else not read). */
int SNEPPX_rotary_frequencies(double* freqs, float* magnitude, size_t dims, double base, SNEPPXRotaryScaling kind,
                              double factor, double original, double low, double high);

/* Turns q_heads heads of q and kv_heads heads of k of every token, bf16 rows of
 * heads * head_dim values at q + t * q_stride (elements), e.g. slices of the QKV
 * projection's rows, into q_out and k_out.  An output may be its input (the same
 * address and stride), and must not overlap it otherwise.  No heads: nothing is read
 * or written there, and its pointers may be NULL.  positions int32 [tokens].
 * head_dim up to 256, a multiple of 8. */
int SNEPPX_rotary_apply(const SNEPPXRotary* rotary, const uint16_t* q, size_t q_stride, uint16_t* q_out,
                        size_t q_out_stride, size_t q_heads, const uint16_t* k, size_t k_stride, uint16_t* k_out,
                        size_t k_out_stride, size_t kv_heads, size_t head_dim, const int32_t* positions,
                        size_t tokens, SNEPPXStream stream);

#ifdef __cplusplus
}
#endif

#endif /* SNEPPX_ROTARY_H */
