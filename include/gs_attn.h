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

/* gs_attn that also leaves, for each token and head, the logarithm of its
 * softmax's sum: lse[t * n_heads + h] = log(sum over j of exp(scale * (q . k_j))),
 * -inf where the token sees no key (NULL: none). */
int gs_attn_lse(const gs_kv_cache *c, uint32_t layer, const gs_kv_batch *b, const gs_attn_args *a, float *lse, void *stream);

/* gs_attn_lse for a batch whose sequences come in families: sequences
 * families[j] .. families[j + 1] - 1 of the batch, j < n_families, whose rows begin
 * with the same pages, as gs_kv_fork leaves them.  The pages that all rows of a
 * family have in common are read once for the family, with the queries of all
 * its sequences; results are those of gs_attn, whatever the rows hold.
 * `families` [n_families + 1] is device memory, ascending; sequences before the
 * first or after the last family are by themselves.  The workspace is larger
 * and grows with the tokens: gs_attn_shared_workspace bytes.
 * Weights reach the values in parts that hold 22 bits or more, of 16-bit queries
 * too (gs_attn rounds theirs to the cache's type, but for few query rows). */
int gs_attn_shared(const gs_kv_cache *c, uint32_t layer, const gs_kv_batch *b, const uint32_t *families, uint32_t n_families,
                   const gs_attn_args *a, float *lse, void *stream);

/* Bytes of gs_attn_args.ws of a call of gs_attn_shared with up to n sequences,
 * n_families families and n_tokens tokens (0 if the sizes are out of range). */
size_t gs_attn_shared_workspace(const gs_kv_cache *c, uint32_t n_heads, uint32_t n, uint32_t n_families, uint32_t n_tokens);

/* The weight that the tokens of a row get from the row's newest ones, summed over
 * those and the heads, of one layer: for token j of the row r of sequence i of
 * `b`, j < len[r],
 *   mass[r][j] = keep * mass[r][j] + sum over t, h of exp(scale * (q_th . k_j) - lse_th),
 * over the sequence's tokens t that see j (as in gs_attn) and all heads h.  lse
 * is what gs_attn_lse or gs_attn_shared left for the same tokens.  Called for
 * each layer with keep = 1 it adds the layers up; keep = 0 begins anew (what
 * mass held does not count).  Of sequences of the same row the first counts;
 * rows out of range are skipped.  What masked keys hold does not count. */
typedef struct gs_weigh_args {
    uint32_t type;          /* of q: the cache's, or GS_TYPE_F32 */
    uint32_t n_heads;       /* a multiple of n_kv */
    const void *q;          /* as in gs_attn_args */
    size_t ld_q;
    const float *lse;       /* [n_tokens][n_heads] */
    float *mass;            /* [rows][ld_mass] */
    size_t ld_mass;         /* at least ld_table * page_size */
    float keep;
    float scale;            /* 0: 1 / sqrt(d) */
    uint32_t window;
    uint32_t max_q;         /* the most tokens that a sequence has (0: n_tokens); a smaller number only costs time */
    void *ws;               /* [gs_attn_weigh_workspace] bytes, 16-byte aligned */
    size_t ws_bytes;
} gs_weigh_args;

/* Bytes of workspace of any call (0 if the sizes are out of range).  No value is
 * kept in it from call to call; calls that may overlap need one each. */
size_t gs_attn_weigh_workspace(const gs_kv_cache *c);

/* Scores and sums are f32; f32 q goes through the matrix cores in three parts,
 * as in gs_attn.  Two calls with the same arguments give the same bits. */
int gs_attn_weigh(const gs_kv_cache *c, uint32_t layer, const gs_kv_batch *b, const gs_weigh_args *a, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* GS_ATTN_H */
