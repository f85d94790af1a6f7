/*
 * popcorn_serve.h -- operators of a decoder's serving step around the
 * quantized linears: a paged key/value cache held in 8 bits (append with the
 * position rotation, read-back, attention) and a mixture-of-experts layer on
 * int8 experts. popcorn has no counterpart of any of them; nothing here
 * changes popcorn.h.
 *
 * Conventions are those of popcorn.h: device pointers owned by the caller,
 * a null buffer that is not marked optional -> POPCORN_ERROR_INVALID_VALUE
 * before any size is looked at, a call without work (no sequences, no
 * tokens) -> POPCORN_SUCCESS, asynchronous on `stream`, scratch from the
 * library's stream-ordered pool.
 */
#ifndef POPCORN_SERVE_H
#define POPCORN_SERVE_H

#include "popcorn.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Element type of activations (queries, keys, values, outputs). */
typedef enum {
    POPCORN_TYPE_F32 = 0,
    POPCORN_TYPE_F16 = 1,
    POPCORN_TYPE_BF16 = 2,
} popcornType_t;

/*
 * A paged key/value cache: pages of `page_size` tokens, codes int8
 * [pages, heads, page_size, dim] and one f32 scale per page and head
 * [pages, heads], keys and values apart; a cached value is code * scale.
 * page_size: a power of two, 16 to 256; dim: a multiple of 16, 16 to 256;
 * k and v 16-byte aligned. (page, head) blocks are contiguous, so a block's
 * codes are one run of page_size * dim bytes.
 *
 * Scales are not negative, and below 2^126 or not finite. Attention takes a
 * value scale below 2^-80 for that of a block of zeros, as an append writes
 * it. Where the value scales that a query sees (at least 2^-80 for this) are
 * up to 2^96 apart, softmax weights down to 2^-30 of the largest are kept.
 *
 * A sequence's token at position p is row p % page_size of page
 * table[sequence, p / page_size]. Only table entries of pages that hold one
 * of the sequence's tokens are read; the others may hold anything. A page
 * index outside [0, pages), a position outside the table or a length beyond
 * it is skipped (never followed) and reported by popcornB200DeviceErrors.
 */
typedef struct {
    int8_t* k;
    int8_t* v;
    float* k_scale;
    float* v_scale;
    int64_t pages;
    int64_t heads;
    int64_t page_size;
    int64_t dim;
} popcornKvCache_t;

/*
 * Appends `tokens` new keys and values to `seqs` sequences, rotating keys
 * (and, if q is given, queries) by their position on the way.
 *
 *   k, v      [tokens, heads, dim] of `type`, strides in elements per token
 *             and per head, dim contiguous
 *   first     [seqs + 1]: sequence b's new tokens are rows first[b] to
 *             first[b + 1] - 1 (NULL: one token each, tokens == seqs); rows
 *             before first[0] and from first[seqs] on are not looked at, and
 *             outputs of theirs are left as they are
 *   start     [seqs]: tokens that sequence b holds before the call; its new
 *             tokens take positions start[b], start[b] + 1, ...
 *   table     [seqs, table_pages] int32 page indices (table_pages wide)
 *   q, q_out  optional (both or neither): [tokens, q_heads, dim], q strided
 *             like k, q_out contiguous; q_out may be q where q is contiguous
 *   cos, sin  f32 [positions, rot_dim / 2], both NULL for no rotation
 *             (rot_dim is then ignored). rot_dim: a multiple of 8, at most
 *             dim; elements from rot_dim on pass through unrotated.
 *   interleaved  0: element j of the first half pairs with element
 *             j + rot_dim / 2; otherwise 2j pairs with 2j + 1. A pair (a, b)
 *             becomes (a cos - b sin, b cos + a sin), each product and sum
 *             rounded to f32 on its own.
 *
 * A (page, head) block's scale becomes max(old scale, max|new| / 127), where
 * a block whose row 0 is written by this call has no old scale and a
 * quotient below 2^-80 counts as 0; NaN is skipped by the maximum. If the
 * scale grew, the rows below the sequence's first new one are re-encoded as
 * rint(code * (old / new)); new rows become rint(value / scale) clamped to
 * [-128, 127] (0 where the scale is 0). All of it is IEEE f32, so codes and
 * scales are reproducible bit for bit. Rows after the new ones keep their
 * bytes. Appending the same tokens at the same positions again changes
 * nothing. An infinite value makes its block's scale infinite.
 *
 * Two sequences of one call must not write to the same page.
 */
popcornStatus_t popcornKvAppend(
    const popcornKvCache_t* cache,
    const void* k,
    int64_t k_token_stride,
    int64_t k_head_stride,
    const void* v,
    int64_t v_token_stride,
    int64_t v_head_stride,
    popcornType_t type,
    const int32_t* table,
    int64_t table_pages,
    const int32_t* first,
    const int32_t* start,
    int64_t seqs,
    int64_t tokens,
    void* q_out,
    const void* q,
    int64_t q_token_stride,
    int64_t q_head_stride,
    int64_t q_heads,
    const float* cos,
    const float* sin,
    int64_t positions,
    int64_t rot_dim,
    int interleaved,
    cudaStream_t stream
);

/*
 * Reads pages back as values: k_out, v_out [count, heads, page_size, dim] of
 * `type` = code * scale (the f32 product, rounded once), for the `count`
 * page indices in `list`. Every row of a page is read, used or not. An index
 * outside [0, pages) gives zeros and is reported by popcornB200DeviceErrors.
 */
popcornStatus_t popcornKvRead(
    void* k_out,
    void* v_out,
    popcornType_t type,
    const popcornKvCache_t* cache,
    const int32_t* list,
    int64_t count,
    cudaStream_t stream
);

/*
 * Attention of `tokens` queries over the cache:
 *   out[t, i] = sum_j softmax_j(scale * q[t, i] . key[j]) value[j]
 * where query head i reads cache head i / (q_heads / heads) and j runs over
 * the tokens of t's sequence that t sees.
 *
 *   q         [tokens, q_heads, dim] of `type`, strides in elements per token
 *             and per head, dim contiguous; out contiguous, of the same type
 *   first     as in popcornKvAppend (NULL: one query each, tokens == seqs)
 *   length    [seqs]: cached tokens of each sequence, the queries' own
 *             included; sequence b's queries are its last positions
 *   max_tokens  an upper bound of the queries of one sequence
 *   causal    non-zero: a query at position p sees positions <= p;
 *             0: it sees every position below length[b]
 *   window    > 0: a query at position p sees only positions > p - window
 *             (0 or less: no window)
 *   lse       optional f32 [tokens, q_heads]: the natural logarithm of the
 *             softmax's denominator, -inf where a query sees nothing
 *   workspace  optional, 16-byte aligned, popcornKvAttentionWorkspace bytes
 *             (independent of lengths; nothing in it needs to start at zero
 *             and nothing is kept in it); NULL: from the library's pool
 *
 * A query that sees nothing gives zeros. Scores, statistics and sums are
 * f32 or exact integers; f32 queries keep 23 bits relative to their row's
 * largest element, f16 and bf16 queries 16 bits; probabilities keep 22 bits,
 * those of bf16 queries 11. A query row that holds a NaN or an infinity and sees a
 * token, or sees a block with a non-finite scale, gives NaN; so is its lse,
 * which may stay that of the scores where only a value scale is not finite.
 * Results do not depend on the order in which blocks of the GPU run. The cut of
 * the work and, for 16-bit types, the kernel are chosen by the sizes given, the
 * width of the block table among them: calls of other sizes may differ in the
 * last bits for the same tokens.
 */
popcornStatus_t popcornKvAttention(
    void* out,
    float* lse,
    const void* q,
    int64_t q_token_stride,
    int64_t q_head_stride,
    popcornType_t type,
    const popcornKvCache_t* cache,
    const int32_t* table,
    int64_t table_pages,
    const int32_t* first,
    const int32_t* length,
    int64_t seqs,
    int64_t tokens,
    int64_t max_tokens,
    int64_t q_heads,
    int causal,
    int64_t window,
    float scale,
    void* workspace,
    int64_t workspace_bytes,
    cudaStream_t stream
);

/* Bytes of workspace that popcornKvAttention takes for these sizes (0 where
 * the call would be refused or has no work). Launches nothing. */
int64_t popcornKvAttentionWorkspace(
    const popcornKvCache_t* cache,
    popcornType_t type,
    int64_t seqs,
    int64_t tokens,
    int64_t max_tokens,
    int64_t q_heads
);

/*
 * A mixture-of-experts layer for a few tokens, experts in popcorn's
 * per-channel int8 (W[n, k] = q[n, k] * s[n]):
 *   z = x @ router^T                       [M, E]
 *   p = softmax(z); each token picks the top_k experts of largest z, the
 *       lowest index first among equals; with renormalize their p are
 *       divided by their sum
 *   out[m] = sum over its picks e of p_e *
 *            (silu(x W_gate[e]^T) * (x W_up[e]^T)) W_down[e]^T
 *
 *   x [M, K], out [M, K], router [E, K] f32
 *   q_gate, q_up int8 [E, F, K], s_gate, s_up f32 [E, F]
 *   q_down int8 [E, K, F], s_down f32 [E, K]
 *   experts int32 [M, top_k], weights f32 [M, top_k]: optional (both or
 *             neither), the picks, largest first
 *   workspace optional, 256-byte aligned, popcornMoeWorkspace bytes; NULL:
 *             from the library's pool
 *
 * Limits (else POPCORN_ERROR_INVALID_VALUE): E <= 256, 1 <= top_k <=
 * min(E, 16), K and F <= 65536. Any M, meant for up to a few tens: 64 tokens
 * are one pass over the chosen experts. K and F that are multiples of 16 with
 * 16-byte aligned codes run on the warp-level tensor path: activations and
 * hidden values as 30-bit fixed point, exact integer dot products (of 32
 * columns for the down product, joined in f32). Other sizes and alignments
 * sum in f32. A token with a NaN or an infinity gives NaN for that token.
 * Results do not depend on the order in which blocks of the GPU run.
 */
popcornStatus_t popcornMoe_i8f32(
    float* out,
    int32_t* experts,
    float* weights,
    const float* x,
    const float* router,
    const int8_t* q_gate,
    const float* s_gate,
    const int8_t* q_up,
    const float* s_up,
    const int8_t* q_down,
    const float* s_down,
    int64_t M,
    int64_t K,
    int64_t F,
    int64_t E,
    int64_t top_k,
    int renormalize,
    void* workspace,
    int64_t workspace_bytes,
    cudaStream_t stream
);

/* Bytes of workspace that popcornMoe_i8f32 takes for these sizes (0 where the
 * call would be refused or has no work). Launches nothing. */
int64_t popcornMoeWorkspace(
    int64_t M,
    int64_t K,
    int64_t F,
    int64_t E,
    int64_t top_k
);

#ifdef __cplusplus
}
#endif

#endif /* POPCORN_SERVE_H */
