/* mk_serve.h -- C ABI of the serving operators on B200 (sm_100a): cache pages, query and key heads on their way into a
 * paged cache, attention over it, and the choice of the next token.  Each call stands alone (one or two launches); the
 * engines of mk_b200.h and mk_stage.h call them where a cache is shared, held in 4 bits, or a token is not the arg-max.
 *
 * Conventions as in mk_b200.h: the caller owns every device buffer and passes raw addresses, every function returns MK_OK
 * or a negative MK_ERR_* (nothing was launched then), mk_last_error() has the text, nothing throws, no call synchronises,
 * allocates or keeps anything, and the current device is the caller's again on return.
 */
#ifndef MK_SERVE_H
#define MK_SERVE_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

enum { MKV_BF16 = 0, MKV_F16 = 1, MKV_F32 = 2, MKV_INT4 = 3 };   /* element types (F32: inputs only, INT4: caches only) */

enum {
    MKV_MAX_REQUESTS = 4096,     /* requests of one call                                                       */
    MKV_GROUP = 64,              /* values that share a scale in a 4-bit cache                                 */
    MKV_MAX_VOCAB = 524288,      /* logits of one row                                                          */
    MKV_MAX_GROUP_HEADS = 128    /* query heads per KV head                                                    */
};

/* ---- cache pages --------------------------------------------------------------------------------------------
 * Requests hold pages of `page` tokens; free pages lie on a stack.  lengths[r] tokens of request r are in the cache,
 * new_tokens[r] are about to enter.  In request order: what a request holds beyond its first lengths[r] tokens goes back
 * on the stack (the first returned page on top), then pages for the new tokens come from the top.  The first request
 * that does not fit (pages or `room`), and every later one that asks for anything, waits: granted[r] = 0, it keeps the
 * pages of its first lengths[r] tokens, its new tokens get no slot.  A request whose length or new tokens are negative, or
 * that needs more than max_pages pages, is not granted and holds up nobody (its context is 0). */
typedef struct {
    uint64_t lengths, new_tokens;    /* i32[requests]                                                          */
    uint64_t table;                  /* i32[requests][max_pages], in and out: page of every held page number, 0 behind  */
    uint64_t held;                   /* i32[requests], in and out: pages held                                  */
    uint64_t free_pages, n_free;     /* i32[pages - 1] and i32[1], in and out: the stack and its height (page 0 is never on it) */
    uint64_t scratch;                /* i32[8 * requests + 8]                                                  */
    uint64_t slots, positions, rows; /* i32[room], out: cache slot (page * page size + offset), position and request of every new
                                        token, requests one after the other; -1, 0, -1 behind the last         */
    uint64_t starts;                 /* i32[requests + 1], out: first new token of every request               */
    uint64_t context;                /* i32[requests], out: tokens in the cache once the granted ones have entered */
    uint64_t granted;                /* i32[requests], out                                                     */
    int32_t requests, max_pages, page, pages, room, device;
} mk_plan_args;
int mk_page_plan(const mk_plan_args* args, void* stream);

/* ---- a paged cache -------------------------------------------------------------------------------------------
 * 16 bits: element (page, head, offset, d) at page * s_page + head * s_head + offset * s_pos + d (strides in elements,
 * multiples of 8).  4 bits: `codes` rows of head_dim / 2 bytes [page][head][offset], and per row head_dim / 64 pairs
 * (scale, low) of bf16: value = low + scale * code.  A 32-bit word holds 8 consecutive values, the first in the lowest
 * bits; word i * (head_dim / 64) + g of a row holds values 64 g + 8 i ... 64 g + 8 i + 7 (what a lane of the attention
 * kernels multiplies is then one run of bytes). */
typedef struct {
    uint64_t k, v;                   /* 16-byte aligned                                                        */
    uint64_t k_scales, v_scales;     /* INT4 only                                                              */
    int64_t s_page, s_head, s_pos;   /* 16-bit types only                                                      */
    int32_t type, pages, kv_heads, head_dim, page;   /* head_dim 64, 128 or 256; page: a power of two >= 16     */
    int32_t reserved;
} mk_cache;

/* ---- heads: norm, rotation, cache write --------------------------------------------------------------------------
 * q, k: y = x * rsqrt(mean(x^2) + eps) * (norm_offset + weight) where a weight is given (else x), then pairs (d, d + rot/2)
 * (interleaved: (2d, 2d+1)), d < pairs, turned by angle d of row positions[t] of the tables.  v: as it is, or
 * normed without a weight (v_norm).  With a cache, k and v of token t enter slot slots[t]; a token whose slot is outside
 * the cache, or whose position is outside the tables, is padding: zeros in q_out (and k_out), nothing written. */
typedef struct {
    uint64_t q, k, v;                /* [tokens][heads][head_dim] of `source`; v 0 without a cache; q 0 with no query heads */
    uint64_t q_out, k_out;           /* [tokens][heads][head_dim] of `type`, contiguous; k_out only without a cache */
    uint64_t positions, slots;       /* i32[tokens]; slots only with a cache                                   */
    uint64_t q_norm, k_norm;         /* fp32 [head_dim] or 0: no norm                                          */
    uint64_t cos, sin;               /* fp32 [max_position][pairs]; 0: no rotation                             */
    int64_t q_tok, q_head, k_tok, k_head, v_tok, v_head;   /* strides in elements                              */
    mk_cache cache;                  /* cache.k 0: none                                                        */
    float eps, norm_offset;
    int32_t tokens, q_heads, kv_heads, head_dim, source, type, rot, pairs, max_position, interleaved, v_norm, device;
} mk_heads_args;
int mk_heads(const mk_heads_args* args, void* stream);

/* Rows of the cache as values: k_out, v_out [tokens][kv_heads][head_dim], contiguous, fp32 for a 4-bit cache and the cache's type
 * else; a slot outside the cache gives zeros. */
int mk_cache_rows(const mk_cache* cache, uint64_t slots, int tokens, uint64_t k_out, uint64_t v_out, int device, void* stream);

/* ---- attention -----------------------------------------------------------------------------------------------
 * Query t of request r (starts[r] <= t < starts[r + 1]; without starts, t = r) is at position context[r] - (starts[r + 1] - t)
 * and sees the cached keys j <= position with j > position - window or j < sinks (window 0: all of them).
 * out = sum_j softmax_j(scale q k_j) v_j, query head h with KV head h / (q_heads / kv_heads); a query that sees nothing gives
 * zeros.  Keys in a page that the table does not place inside the cache are not seen.  Rows of out outside
 * [starts[0], starts[requests]) are left alone.  What no query of the call sees is not looked at and may hold anything; values
 * that some query sees have to be finite (queries of a tile that do not see them multiply them by 0).  scale > 0. */
typedef struct {
    uint64_t q, out;                 /* [tokens][q_heads][head_dim] of `type`                                  */
    uint64_t table, context, starts; /* i32[requests][table_stride], i32[requests], i32[requests + 1] or 0     */
    uint64_t workspace;              /* mk_attend_bytes() bytes, 16-byte aligned, not shared by calls that may overlap */
    uint64_t status;                 /* i32[4], zero: {code, site, CTA, thread} of the first device-side wait that ran out */
    int64_t q_tok, q_head, out_tok, out_head, table_stride;  /* strides in elements; q, out: multiples of 8    */
    mk_cache cache;
    int64_t spin_limit_ns;           /* bound of every device-side wait; 0 = 2 s                               */
    float scale;
    int32_t type, requests, tokens, q_heads, max_pages, max_new, window, sinks, device;   /* max_new: no request has more new tokens */
} mk_attend_args;
int64_t mk_attend_bytes(const mk_attend_args* args);
int mk_attend(const mk_attend_args* args, void* stream);

/* ---- the next token -------------------------------------------------------------------------------------------
 * Per row, with weights w = exp((x - max) / temperature): candidates in the order (x falling, index rising); the first top_k
 * (0: all), of these the fewest that hold top_p of their weight (1: all), of these those with w >= min_p; the token is the
 * first, by index, at which the running weight of the kept ones exceeds u times their sum.  temperature 0: the largest x, the
 * lowest index among equals.  -inf and NaN are masked: never kept.  A row that has nothing else gives id -1, log-probability
 * -inf, 0 kept.  Weights count in steps of 2^-44, so sums are exact and do not depend on an order. */
typedef struct {
    uint64_t logits;                 /* [rows][vocab] of `type`, rows `stride` elements apart                  */
    uint64_t u;                      /* fp32 [rows] in [0, 1)                                                  */
    uint64_t temperature, top_p, min_p;   /* fp32 [rows]                                                       */
    uint64_t top_k;                  /* i32 [rows]                                                             */
    uint64_t ids, logprobs, kept;    /* i32, fp32 (natural log of the token's share of the kept weight), i32 [rows], out */
    int64_t stride;
    int32_t rows, vocab, type, device;
} mk_sample_args;
int mk_sample(const mk_sample_args* args, void* stream);

#ifdef __cplusplus
}
#endif
#endif
