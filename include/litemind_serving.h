/*
 * litemind_serving.h -- C ABI of the operators that serve many requests at once
 * on one MI355X (gfx950): a latent KV cache in pages that the requests share,
 * multi-head latent attention of each request's new tokens over it, and the
 * choice of the next tokens.
 *
 * LiteMind runs one sequence (KvCache, Attention and Sampler::select_next's
 * greedy branch: include/litemind_attention.h, lm_head_forward); nothing here
 * has a counterpart in it.  Conventions are those of include/litemind_moe.h:
 * int status, lm_last_error, *_dev device pointers, work on the context stream,
 * one host thread at a time per context.
 *
 * lm_page_plan, lm_paged_attention and lm_sample take their lengths, tables and
 * settings from device memory, make no allocation after their first call of a
 * kind on the context, and may be captured into a HIP graph on the context's
 * stream after that (before it, a call under capture is LM_EINVAL).  Replays
 * share the context's scratch: they run on the context's stream, or on another
 * one that waits for it and that it waits for.  lm_paged_forward and
 * lm_paged_decoder_forward refuse capture (LM_EINVAL).
 */
#ifndef LITEMIND_SERVING_H
#define LITEMIND_SERVING_H

#include "litemind_attention.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- one step of the requests in service ----
 * A request is a row: cached tokens in its pages, and added new ones.  Token
 * position p of request r lies in slot table[r][p / page_size] * page_size +
 * p % page_size of the pool.  All arrays are device memory of the caller. */
typedef struct lm_paged_step {
    int64_t requests;         /* rows of the tables, at least 1 */
    int64_t tokens;           /* rows that the step's token arrays hold: at least the sum of added */
    int64_t pages;            /* pages of the pool; pages * page_size at most 2^31 - 1 */
    int32_t page_size;        /* tokens of a page: a multiple of 16, at most 4096 */
    int32_t table_width;      /* pages that a request can hold */
    int32_t max_added;        /* no request adds more tokens than this */
    int32_t reserved;         /* 0 */
    const int32_t* cached;    /* [requests] tokens in the cache before the step */
    const int32_t* added;     /* [requests] new tokens (0: none); negative: the request is over */
    int32_t* table;           /* [requests][table_width] page ids; entries past a request's pages are not read */
    int32_t* ring;            /* [pages] the free pages, a ring: entries head .. head + count - 1, modulo pages */
    const int32_t* queue_in;  /* [2] head and count of the ring before the step */
    int32_t* queue_out;       /* [2] after it; may equal queue_in */
    int32_t* lengths;         /* [requests] tokens in the cache with the step's, 0 of a request that is over; may equal cached */
    int32_t* starts;          /* [requests + 1] first row of each request's new tokens */
    int32_t* positions;       /* [tokens] position of each new token; 0 past the last */
    int32_t* slots;           /* [tokens] slot of each new token; -1 past the last */
    int32_t* info;            /* [4] LM_STEP_*, new tokens, pages taken, pages given back */
} lm_paged_step;

#define LM_STEP_OK 0
#define LM_STEP_LENGTH 1  /* a negative cached length, or a request longer than its table row */
#define LM_STEP_TOKENS 2  /* the new tokens exceed `tokens`, or a request's exceed max_added */
#define LM_STEP_PAGES 3   /* the ring holds fewer pages than the step needs */
#define LM_STEP_RING 4    /* a negative count, or more pages free and given back together than the pool has */

/* Plans a step from cached and added: writes lengths, starts, positions, slots,
 * queue_out and info.  A request takes the pages that its new tokens start from
 * the ring's head, requests in order, and enters them in its table row; the
 * pages of a request that is over go behind the ring's last free page, in
 * request and column order.  No input is changed that the plan reads, but where
 * queue_out or lengths are queue_in or cached themselves, so planning the same
 * step again gives the same.  A step that cannot be
 * served (info[0] is the first LM_STEP_* that applies, in their order) takes and
 * gives back nothing: starts are 0, slots -1, lengths the cached ones, the table
 * and the ring as they were.  A page id outside the pool makes the slots of its
 * tokens -1.  A page is one request's or the ring's: one that two requests name
 * (attention may read it for both) comes back once for each that is over, so the
 * caller takes it out of one row first.  Asynchronous. */
int lm_page_plan(lm_context* ctx, const lm_paged_step* step);

/* Attention of the step's new tokens over the pages, in the latent space that
 * the heads share.  A pool row holds a token's latent c [rank] and rotary key
 * [rope]; a query row holds, per head, W_uk^T q_nope [rank] and the rotated
 * q_rope [rope].  For token t of request r at position p:
 *     s_j = scale * q_t,h . pool_row(r, j), j = 0 .. p
 *     out_t,h = sum_j softmax(s)_j c_j
 * with p = lengths[r] - (starts[r + 1] - starts[r]) + (t - starts[r]).  Reads
 * requests, tokens, pages, page_size, table_width, max_added, table, lengths and
 * starts of the step.
 *   q_dev    [tokens][heads][rank + rope], pool_dev [pages][page_size][rank + rope],
 *   out_dev  [tokens][heads][rank], all of `dtype` (LM_DT_F16 or LM_DT_BF16),
 *            16-byte aligned; out_dev overlaps neither of the others
 *   rank     a multiple of 8 up to 1024, rope a multiple of 8 up to 256
 *   heads    tokens * heads under 2^30, and (tokens * heads / 16 + tokens) blocks
 *            of heads times the tokens of a table row under 2^62
 * Products have the inputs' 16 bits, sums 32; the softmax weights round to 16
 * bits before the second product (fp16 ones under 2^-19 of their row's largest to
 * a multiple of 2^-29 of it) and are added up as rounded, the output once at the
 * end.  Rows past the last request's are not written.  What lies in a page past a
 * request's length, or after a token's own position, does not reach its output,
 * NaN and infinity included.  Page ids outside the pool are not followed: the row
 * reads page 0, and the next lm_synchronize or lm_copy_d2h returns LM_EKERNEL.
 * Asynchronous. */
int lm_paged_attention(lm_context* ctx, const lm_paged_step* step, const void* q_dev, const void* pool_dev,
                       int32_t dtype, int32_t heads, int32_t rank, int32_t rope, float scale, void* out_dev);

/* ---- the model's layers over the pages ----
 * Gives every layer of the context a pool of `pages` pages of page_size tokens
 * in HBM (fp16, 2 (kv_lora_rank + qk_rope) bytes per token and layer: 1152 on
 * DeepSeek-V2, where lm_attention_configure's cache takes 16640 on V2-Lite).
 * After lm_attention_configure, once per context.  Needs kv_lora_rank (up to
 * 1024), qk_nope, hidden_size, q_lora_rank and heads * v_head_dim in multiples of
 * 32, v_head_dim of 16 and qk_rope of 8.  The pages start as zeros. */
int lm_paged_configure(lm_context* ctx, int64_t pages, int32_t page_size);
/* A layer's pool [pages][page_size][kv_lora_rank + qk_rope] fp16, to read or
 * fill pages (a row: the normalised latent, then the rotated key). */
int lm_paged_pool(lm_context* ctx, int32_t layer, void** out_dev);

/* lm_attention_forward for the new tokens of all requests of a planned step:
 * x_dev [tokens, hidden] at the step's positions, their latents stored in the
 * step's slots of the layer's pool, attention over each request's pages, and
 * out_dev [tokens, hidden] = o_proj . context, or added to it (accumulate = 1).
 * The step's pages and page_size are those of lm_paged_configure; max_added,
 * positions and slots are read too.  Rows past the last new token may hold
 * anything in x_dev and reach no other row; in out_dev they become 0, or stay as
 * they were (accumulate = 1).  Positions at or past context_length are not
 * rotated, as lm_attention_forward's.  kv_b_proj is absorbed into the query and
 * the output; queries, latents and weights round to fp16, within the MFMA
 * path's tolerance.  out_dev must not overlap x_dev.  tokens under 2^24, tokens *
 * heads at most 2^24, and tokens times the widest of hidden_size, q_lora_rank and
 * heads * v_head_dim under 2^30.  Asynchronous. */
int lm_paged_forward(lm_context* ctx, int32_t layer, const lm_paged_step* step, const float* x_dev, float* out_dev,
                     int32_t accumulate);
/* lm_decoder_forward's layer loop with lm_paged_forward as the attention:
 * hidden_dev [tokens, H] in place.  Rows past the last new token are taken as
 * zeros; what they come out as means nothing.  `path` as there.  A call that is
 * refused, for a layer whose weights are not there or do not fit fp16 too, leaves
 * hidden_dev and the pools as they were. */
int lm_paged_decoder_forward(lm_context* ctx, int32_t first_layer, int32_t last_layer, const lm_paged_step* step,
                             float* hidden_dev, int32_t path);

/* ---- sampled tokens, beside lm_head_forward's greedy ones ----
 * The settings of one row of logits. */
typedef struct lm_sampling {
    float temperature;  /* 0 (or less, or NaN): the greedy token */
    int32_t top_k;      /* 0 (or less): every token */
    float top_p;        /* 1 (or more, or NaN): every token */
    float min_p;        /* 0 (or less, or NaN): every token */
} lm_sampling;
/* The next token of each row of logits_dev [rows] (row_stride floats apart, at
 * least vocab), from its settings and one given random number in [0, 1).  With
 * the tokens in order of falling logit, equal ones of rising index, and
 * e_i = exp((logit_i - largest) / temperature), a row keeps the longest prefix
 * of at most top_k tokens, whose tokens each have less than top_p of the top_k
 * tokens' sum of e before them, and an e of at least min_p; the first token
 * always.  Its token is then the first kept one, in index order, up to which the
 * kept e add up to more than uniform times their total; probability_dev (may be
 * NULL) receives the token's e over that total.  The sums are exact in 64-bit
 * fixed point, so a token does not depend on how the work was shared out.  NaN
 * counts as -infinity, which is never chosen: a row of nothing else gives token
 * -1 and probability 0.  vocab at most 2^24.  Asynchronous. */
int lm_sample(lm_context* ctx, const float* logits_dev, int64_t rows, int64_t vocab, int64_t row_stride,
              const lm_sampling* settings_dev, const float* uniform_dev, int32_t* token_dev, float* probability_dev);

#ifdef __cplusplus
}
#endif
#endif
