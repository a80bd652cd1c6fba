/*
 * gs_cache.h -- C ABI of the paged cache of keys and values, and of what
 * happens to its pages: rows grow, are forked, freed, lose tokens, and are cut
 * to a budget.
 *
 * gguf-rs-cli keeps one contiguous f32 cache per layer and writes one position
 * of it per token (the kv_write shader, dispatched at src/gpu/mod.rs:458-466);
 * when its context is full it drops the oldest quarter of the history and runs
 * the prompt through the model again (src/main.rs:205-256, 284-297).  Here many
 * rows (conversations) share one pool of pages: a row takes a page when its
 * tokens need one, rows made from one another share their full pages, and a
 * range of tokens leaves a row without a second run of the prompt
 * (gs_kv_drop).
 *
 * All state is memory of the current HIP device that the caller owns, and every call is
 * asynchronous on its stream, allocates nothing and can be captured in a HIP
 * graph, as the calls of gs_decode.h.  Calls on one cache are ordered by the
 * caller (one stream, or events between them): each reads what the last one
 * wrote.  Same status codes as gs_sampler.h.
 */
#ifndef GS_CACHE_H
#define GS_CACHE_H

#include <stddef.h>
#include <stdint.h>

#include "gs_rope.h"
#include "gs_sampler.h"

#ifdef __cplusplus
extern "C" {
#endif

#define GS_KV_NONE 0xffffffffu  /* no page, or no row */

#define GS_KV_MAX_HEAD 256u     /* values of one head */

/* The cache of `rows` rows.  Keys and values are F16 or BF16, at
 *   k[layer][page][head][slot][d]
 * so that a head's slots of one page are contiguous.  Token t of row r is in
 * slot t % page_size of page table[r * ld_table + t / page_size].
 * Between calls: ref[p] is the number of rows that hold page p (0: free);
 * places of `table` past a row's last page hold GS_KV_NONE; a row's last page,
 * unless it is full, is held by no other row. */
typedef struct gs_kv_cache {
    void *k, *v;            /* [n_layers][n_pages][n_kv][page_size][d], 16-byte aligned */
    uint32_t type;          /* GS_TYPE_F16 or GS_TYPE_BF16 */
    uint32_t n_layers;
    uint32_t n_pages;
    uint32_t n_kv;          /* heads of keys and values */
    uint32_t page_size;     /* tokens of a page: a power of two, 16 to 1024 */
    uint32_t d;             /* values of a head: a multiple of 8, at most GS_KV_MAX_HEAD */
    uint32_t rows;
    uint32_t ld_table;      /* most pages of a row; ld_table * page_size is at most 2^30 */
    uint32_t *table;        /* [rows][ld_table] */
    uint32_t *len;          /* [rows] tokens held */
    uint32_t *ref;          /* [n_pages] */
    uint32_t *ws;           /* [gs_kv_workspace] words for the calls below; no value is kept in it from call to call */
} gs_kv_cache;

/* Words of gs_kv_cache.ws (0 if the cache's sizes are out of range). */
size_t gs_kv_workspace(const gs_kv_cache *c);

/* The calls below take at most `rows` rows, and all but gs_kv_extend at most
 * 65535. */

/* Every row empty, every page free. */
int gs_kv_reset(const gs_kv_cache *c, void *stream);

/* Row rows[i] (row i where rows is NULL) grows by add[i] tokens (by add_all
 * where add is NULL), i < n: the pages it needs are taken, and len grows.  The
 * tokens' keys and values are for gs_kv_append to write.  New pages are the
 * lowest-numbered free ones, in the order of i, then of their place.
 * status[i] (or NULL): GS_OK; GS_ERR_NOMEM once the free pages have run out,
 * for that row and those after it that need a page; GS_ERR_UNSUPPORTED where
 * the row would not fit its table; GS_ERR_INVALID where rows[i] >= rows.  A
 * row with an error is as before.  The n rows are different ones.  All
 * pointers are device memory. */
int gs_kv_extend(const gs_kv_cache *c, const uint32_t *rows, size_t n, const uint32_t *add, uint32_t add_all,
                 int32_t *status, void *stream);

/* Row dst[i] becomes a copy of row src[i] as it was before the call, for all i
 * at once (so a beam search's reordering is one call); src[i] = GS_KV_NONE
 * empties it.  Full pages are shared, the tokens of a partial last page are
 * copied to a new page (of every layer; the page's other slots keep what they
 * hold).  New pages are the lowest-numbered free ones in the order of i, and
 * are taken before the pages of the old rows dst are released.  A pair with
 * src = dst does nothing.  status[i] (or NULL): GS_ERR_NOMEM from the first
 * row on for which no page is free (only rows that need one); GS_ERR_INVALID
 * for a row out of range, or a dst that an earlier i has.  Rows with an error
 * are as before. */
int gs_kv_fork(const gs_kv_cache *c, const uint32_t *src, const uint32_t *dst, size_t n, int32_t *status, void *stream);

/* Rows rows[i] become empty; a page that no row holds any more is free.  Rows
 * out of range are skipped. */
int gs_kv_free(const gs_kv_cache *c, const uint32_t *rows, size_t n, void *stream);

/* Weights of cached tokens, mass[row * ld_mass + token] (gs_attn_weigh adds them
 * up, gs_kv_evict goes by them), belong to places of rows, so they go with every
 * call that moves or removes tokens: gs_kv_evict moves them, and these two do
 * what gs_kv_free and gs_kv_drop do and clear a freed row's weights, or move
 * those of a drop's tokens and clear the places behind.  ld_mass is at least
 * ld_table * page_size; mass NULL: there are none.  After gs_kv_reset and
 * gs_kv_fork the caller clears them, or copies row src[i]'s to row dst[i]. */
int gs_kv_free_mass(const gs_kv_cache *c, const uint32_t *rows, size_t n, float *mass, size_t ld_mass, void *stream);
int gs_kv_drop_mass(const gs_kv_cache *c, const uint32_t *rows, size_t n, const uint32_t *from, const uint32_t *to,
                    const gs_rope *rope, float *mass, size_t ld_mass, int32_t *status, void *stream);

/* Tokens from[i] .. to[i] - 1 (cut to the row's tokens) leave row rows[i], and
 * those after them move down to their place; with `rope` their keys are turned
 * by -(to - from) positions too, as if they had been written at their new
 * ones (its gain is not applied again).  Values are rounded to the cache's
 * type once more.  to >= len cuts the row's end off.
 * A page of the row that is written and that another row holds too is
 * replaced by a new one (lowest-numbered free pages, in the order of i, then
 * of their place), others are written in place; pages that are no longer
 * needed are released.  status[i] as of gs_kv_extend, GS_ERR_INVALID also for
 * a row that an earlier i has.  At most 2^23 - 1 layers times heads. */
int gs_kv_drop(const gs_kv_cache *c, const uint32_t *rows, size_t n, const uint32_t *from, const uint32_t *to,
               const gs_rope *rope, int32_t *status, void *stream);

/* Rows that hold more tokens than their budget are cut to it: of row rows[i]
 * stay its newest `recent` tokens, its first `first` ones, and of those between
 * the ones of greatest weight, as many as the budget has left (budgets below
 * first + recent: the newest come first).  Of equal weights the lowest token
 * stays; NaN is more than any number.  Weights are mass[row * ld_mass + token],
 * which gs_attn_weigh adds up.  Those that stay keep their order and move down
 * to places 0 .. budget - 1, their weights with them (those of the places
 * behind, up to the old length, become 0); with `rope` keys are turned back by as
 * many positions as they move (the gain is not applied again).  Pages, rounding
 * and status[i] as of gs_kv_drop; a row with an error is as before.
 * At most 2^23 - 1 layers times heads.  Device memory, but for the struct. */
typedef struct gs_kv_evict_args {
    const uint32_t *rows;   /* [n] */
    size_t n;
    const uint32_t *budget; /* [n] tokens, or NULL: budget_all for each */
    uint32_t budget_all;
    uint32_t first, recent;
    float *mass;            /* [rows][ld_mass] */
    size_t ld_mass;         /* at least ld_table * page_size */
    const gs_rope *rope;    /* or NULL */
    int32_t *status;        /* [n], or NULL */
    void *ws;               /* [gs_kv_evict_workspace] bytes, 16-byte aligned */
    size_t ws_bytes;
} gs_kv_evict_args;

/* Bytes of workspace of an eviction of n rows with budgets of at most `budget`
 * (the budget_all of the call; 0, or where `budget` is given: any).  0 if the
 * sizes are out of range.  No value is kept in it from call to call. */
size_t gs_kv_evict_workspace(const gs_kv_cache *c, size_t n, uint32_t budget);

int gs_kv_evict(const gs_kv_cache *c, const gs_kv_evict_args *x, void *stream);

/* The sequences of a call of gs_kv_append or gs_attn, device pointers: the
 * newest tokens of n rows, one row after the other.  Sequence i has the tokens
 * start[i] .. start[i + 1] - 1 of the n_tokens given (start NULL: token i
 * alone, and n_tokens = n); the last of them is the last token of row rows[i]
 * (row i where rows is NULL), so token t of the sequence is at position
 * len - (start[i + 1] - start[i]) + t.  start is ascending with start[0] = 0. */
typedef struct gs_kv_batch {
    uint32_t n;
    uint32_t n_tokens;
    const uint32_t *rows;
    const uint32_t *start;
} gs_kv_batch;

/* New keys, values and queries of one layer, device memory, of `type`
 * (GS_TYPE_F32, or the cache's); token t's heads are at t * ld, each d values
 * after the one before. */
typedef struct gs_kv_new {
    uint32_t type;
    const void *k, *v;      /* [n_tokens][n_kv][d] */
    size_t ld_k, ld_v;      /* values from token to token, at least n_kv * d */
    const void *q;          /* [n_tokens][n_heads][d], or NULL */
    size_t ld_q;
    void *q_out;            /* q turned to its positions (may be q itself where types and strides are equal) */
    size_t ld_q_out;
    uint32_t q_out_type;    /* `type` or the cache's */
    uint32_t n_heads;
} gs_kv_new;

/* The new tokens of one layer, after gs_kv_extend has made room for them: keys
 * (and queries) are turned to their positions by `rope` (NULL: not at all),
 * keys and values rounded to the cache's type and written to the rows' pages.
 * Tokens at positions below 0 or of rows out of range are not written. */
int gs_kv_append(const gs_kv_cache *c, uint32_t layer, const gs_kv_batch *b, const gs_rope *rope, const gs_kv_new *x,
                 void *stream);

#ifdef __cplusplus
}
#endif

#endif /* GS_CACHE_H */
