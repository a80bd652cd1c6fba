/*
 * gs_attn.h -- C ABI of the attention of new tokens over a paged cache.
 *
 * gguf-rs-cli runs one token at a time through its attention shader, one
 * workgroup per head over a contiguous f32 cache (src/gpu/mod.rs:467-474).
 * Here one call takes the newest tokens of many rows: one token each
 * (decoding), chunks of prompts, or both.  Same status codes as gs_sampler.h.
 */
#ifndef GS_ATTN_H
#define GS_ATTN_H

#include <stddef.h>
#include <stdint.h>

#include "gs_cache.h"

#ifdef __cplusplus
extern "C" {
#endif

/* For token t of sequence i of `b` (at position p, see gs_kv_batch) and head h:
 *   out = sum_j w_j v_j,  w = softmax over j of scale * (q . k_j),
 * over the tokens j of the row with p - window < j <= p (window 0: all
 * j <= p), with the keys and values of head h / (n_heads / n_kv).  A token
 * without such j (at a position below 0, or of a row out of range) gets zeros.
 * What a masked key or value holds does not count, NaN and infinities
 * included; nor does what the pages hold past the row's tokens. */
typedef struct gs_attn_args {
    uint32_t type;          /* of q and out: the cache's, or GS_TYPE_F32 */
    uint32_t n_heads;       /* a multiple of n_kv */
    const void *q;          /* [n_tokens][n_heads][d], 16-byte aligned */
    size_t ld_q;            /* values from token to token: a multiple of 8, at least n_heads * d */
    void *out;              /* [n_tokens][n_heads][d], 16-byte aligned; not q */
    size_t ld_out;
    float scale;            /* 0: 1 / sqrt(d) */
    uint32_t window;
    uint32_t max_q;         /* the most tokens that a sequence has (0: n_tokens); a smaller number only costs time */
    void *ws;               /* [gs_attn_workspace] bytes, 16-byte aligned */
    size_t ws_bytes;
} gs_attn_args;

/* Bytes of workspace of a call of any number of tokens with n_heads heads
 * (0 if the sizes are out of range).  No value is kept in it from call to
 * call; calls that may overlap need one each. */
size_t gs_attn_workspace(const gs_kv_cache *c, uint32_t n_heads);

/* Scores, weights' sums and outputs are summed in f32.  The matrix cores take
 * both factors of a product in one type.  With F32 q, q and the weights go
 * through them in three parts of the cache's type, which hold 24 bits.  With q
 * of the cache's type the weights are rounded to that type once, but BF16 weights
 * go in two parts, 16 bits, in calls whose sequences have at most 16 rows of
 * queries per head of keys, as single tokens mostly are.  Two calls with the
 * same arguments give the same bits.  Asynchronous on `stream`. */
int gs_attn(const gs_kv_cache *c, uint32_t layer, const gs_kv_batch *b, const gs_attn_args *a, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* GS_ATTN_H */
