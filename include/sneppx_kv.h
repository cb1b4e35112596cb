/*
 * sneppx_kv.h - a paged key-value cache on gfx950: append, the attention of one
 * new token per row, and eviction by accumulated attention weight.
 *
 * The reference decodes with a contiguous fp32 cache on the CPU
 * (SNEPPX_attn_forward_cached, kernel/attention/attention.c:491-584, between
 * the projections at :500-502 and :584).  These entry points are what stands
 * there when the projections are the device linears of sneppx_qlinear.h: they
 * take the QKV projection's bf16 rows as they are and leave rows that the O
 * projection reads.  As there, every pointer is a DEVICE pointer (the cache
 * descriptor itself is a host struct, read during the call), every call is
 * asynchronous on `stream`, allocates no output, and returns 0, or -1 with the
 * reason in SNEPPX_qlinear_last_error().  A call of no rows or no tokens does
 * nothing and returns 0; pointers to what is empty may be NULL then.
 *
 * The pool: pages of page_size tokens each, k and v [pages][kv_heads]
 * [page_size][head_dim], so that a head's tokens of one page lie together.
 * block_tables int32 [rows][table_width] names the pages of each row (a
 * sequence): its slot t is token t % page_size of page block_tables[row][t /
 * page_size].  lengths int32 [rows]: the slots in use.  An entry outside [0,
 * pages) is a page that is not there: its tokens are not attended to, not
 * written and not moved; nothing is read outside the pool.  A length below 0
 * counts as 0, one beyond the table (or max_length) as that.
 *
 * Rows may share pages (a common prompt) that are only read.  Pages that a call
 * writes (an append, an eviction, the sums of an attention with `accumulate`)
 * belong to one row of that call.
 */
#ifndef SNEPPX_KV_H
#define SNEPPX_KV_H

#include <stddef.h>
#include <stdint.h>

#include "sneppx_qlinear.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef struct {
    void* k;               /* [pages][kv_heads][page_size][head_dim] in dtype, 16-byte aligned */
    void* v;
    float* k_scales;       /* SNEPPX_INT8: [pages][kv_heads][page_size]; else NULL */
    float* v_scales;
    float* weights;        /* [pages][kv_heads][page_size] attention received, or NULL */
    int32_t* positions;    /* [pages][kv_heads][page_size] position of the token in its sequence, or NULL */
    SNEPPXDtype dtype;     /* SNEPPX_BFLOAT16 or SNEPPX_INT8 */
    size_t pages, page_size, kv_heads;
    size_t head_dim;       /* up to 256, a multiple of 8 (int8: of 16) */
} SNEPPXKVCache;

/* Writes new tokens into the last slots of their rows.  k, v: bf16, token t's
 * kv_heads * head_dim values at k + t * k_stride (elements), e.g. slices of the
 * QKV projection's rows.  starts int32 [rows + 1] (ascending): row r has the
 * tokens starts[r] .. starts[r + 1]; NULL: one token for each row (tokens ==
 * rows).  lengths and next_pos (int32 [rows]) count them already: token i of
 * row r's n goes to slot lengths[r] - n + i and is given position next_pos[r] -
 * n + i (next_pos may be NULL without cache->positions).  Tokens whose slot is
 * below 0 or beyond the table, and those past starts[rows], are skipped.
 * SNEPPX_INT8: codes and scale of each token's head by the rule of
 * SNEPPX_quantize_int8_channel (quantize_int8.c:157-177).  weights, if there,
 * start at 0.  k_stored, v_stored (both or neither): bf16
 * [tokens][kv_heads][head_dim], the rows as the cache holds them (code * scale
 * in fp32, rounded to bf16), for a prompt's attention among its own tokens. */
int SNEPPX_kv_append(const SNEPPXKVCache* cache, const uint16_t* k, size_t k_stride, const uint16_t* v,
                     size_t v_stride, size_t tokens, const int32_t* starts, uint16_t* k_stored,
                     uint16_t* v_stored, const int32_t* block_tables, size_t table_width,
                     const int32_t* lengths, const int32_t* next_pos, size_t rows, SNEPPXStream stream);

/* Attention of one new token per row: out[r][h] = sum_t p[t] v[t] with p the
 * softmax over row r's tokens of scale * q[r][h] . k[t]; query head h reads
 * key-value head h / (q_heads / kv_heads).  q bf16, row r's q_heads * head_dim
 * values at q + r * q_stride; out [rows][q_heads][head_dim] in out_dtype
 * (SNEPPX_BFLOAT16 or SNEPPX_FLOAT32), rows out_stride elements apart.
 * Products and sums are fp32 quality throughout; a bf16 result is rounded once.
 * A row without tokens gives zeros.  max_length: no row is longer (it sizes
 * the launch and the scratch; the lengths stay on the device).
 * accumulate: cache->weights of every token attended to grows by the sum of
 * its p over the query heads of its head.  Scratch: a workspace of the calling
 * thread on `stream`; results do not depend on the launch order. */
int SNEPPX_kv_attention(const SNEPPXKVCache* cache, const uint16_t* q, size_t q_stride, void* out,
                        size_t out_stride, SNEPPXDtype out_dtype, const int32_t* block_tables,
                        size_t table_width, const int32_t* lengths, size_t rows, size_t q_heads,
                        size_t max_length, float scale, int accumulate, SNEPPXStream stream);

/* Cuts every row that is longer than `budget` to `budget` tokens, for each
 * key-value head by itself: the tokens with position >= next_pos[row] - recent
 * stay, and of the others those with the largest cache->weights (equal ones:
 * the lower slot; a NaN ranks below every number; if more than `budget` are
 * recent, those in the lower slots).  The kept tokens in slots from `budget` on
 * move, in order, into the slots below that are left free, in order, with
 * everything the cache has of them; the others stay where they are, so a step
 * that drops one token moves one.  Slots from the new length on keep what they
 * held.  new_lengths int32 [rows] (or NULL; not in the memory of `lengths` or
 * `next_pos`): min(length, budget).  A row with a page that is not there keeps its
 * tokens and length.  cache->weights and cache->positions have to be there. */
int SNEPPX_kv_evict(const SNEPPXKVCache* cache, const int32_t* block_tables, size_t table_width,
                    const int32_t* lengths, const int32_t* next_pos, int32_t* new_lengths, size_t rows,
                    size_t max_length, size_t budget, size_t recent, SNEPPXStream stream);

#ifdef __cplusplus
}
#endif

#endif /* SNEPPX_KV_H */
