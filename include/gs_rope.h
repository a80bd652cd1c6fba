/*
 * gs_rope.h -- C ABI of the rotary positions.
 *
 * gguf-rs-cli turns queries and keys with one frequency base and one layout
 * (src/math/rope.rs:1-12; the rope shader, dispatched at
 * src/gpu/mod.rs:451-457).  Here: both layouts, a part of the head, and the
 * scalings that GGUF files name for long contexts (rope.scaling.type "linear"
 * and "yarn", and the divisors of a rope_freqs tensor).
 * Same status codes as gs_sampler.h.
 */
#ifndef GS_ROPE_H
#define GS_ROPE_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Value types, numbered as GgmlType (src/gguf/types.rs:39-41). */
#define GS_TYPE_F32   0u
#define GS_TYPE_F16   1u
#define GS_TYPE_BF16 30u

/* Which two values of a head form pair i < rot / 2. */
#define GS_ROPE_INTERLEAVED 0u  /* 2 i and 2 i + 1 */
#define GS_ROPE_HALF        1u  /* i and i + rot / 2 */

#define GS_ROPE_NONE   0u
#define GS_ROPE_LINEAR 1u
#define GS_ROPE_YARN   2u

/* Pair (a, b) at position p becomes (a cos t - b sin t, b cos t + a sin t)
 * times the gain, t = p f_i, f_i = base^(-2 i / rot) / divisors[i].
 * Linear scaling: f_i / factor.  YaRN (Peng et al. 2023): f_i (1 - y_i) +
 * f_i / factor y_i with the ramp y_i = clamp((i - low) / (high - low), 0, 1)
 * between low = floor(c(beta_fast)) and high = ceil(c(beta_slow)), held to
 * 0 .. rot - 1, c(r) = rot ln(context / (2 pi r)) / (2 ln base): pairs that
 * turn more than beta_fast times in the trained context keep their frequency,
 * those that turn less than beta_slow times are divided; and a gain of
 * 0.1 ln(factor) + 1. */
typedef struct gs_rope_params {
    uint32_t d;             /* values of a head, even, at most 512 */
    uint32_t rot;           /* values that are turned, even, 2 .. d: the first `rot`; the others are copied */
    uint32_t layout;        /* GS_ROPE_INTERLEAVED or GS_ROPE_HALF */
    uint32_t scaling;       /* GS_ROPE_NONE, _LINEAR, _YARN */
    double base;            /* above 1 */
    double factor;          /* at least 1 (scaling) */
    uint32_t context;       /* positions the model was trained on (YaRN) */
    double beta_fast, beta_slow;  /* 0: 32 and 1 (YaRN) */
    double gain;            /* 0: the scaling's own (1, or YaRN's) */
    const float *divisors;  /* [rot / 2] host array, positive, or NULL */
} gs_rope_params;

typedef struct gs_rope gs_rope;

/* The plan: each pair's turns per position as a 64-bit fraction, on the
 * current HIP device (calls with it on another one are GS_ERR_INVALID).  A position's turns are then an integer product whose
 * whole turns fall off by themselves: angles are as exact at position 2^31 as
 * at 1, where p f_i in f32 is off by p 2^-25 radians.  Synchronous. */
int gs_rope_create(const gs_rope_params *p, gs_rope **out);
int gs_rope_destroy(gs_rope *r);

/* out[t][h] = x[t][h] turned to position pos[t], for n_tokens tokens of n_heads
 * heads: device memory, both of `type` (GS_TYPE_*), token t at t * ld values,
 * its heads d values apart.  Sums and products are f32, rounded once.  out
 * may be x with the same stride (in place); otherwise they do not overlap.
 * pos: [n_tokens], read as signed 32-bit.  Asynchronous on `stream`. */
int gs_rope_apply(const gs_rope *r, uint32_t type, const void *x, size_t ld_x, void *out, size_t ld_out,
                  size_t n_tokens, uint32_t n_heads, const int32_t *pos, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* GS_ROPE_H */
