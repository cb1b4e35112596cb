/*
 * sneppx_kv.h - a paged key-value cache on gfx950: append, the attention of one
 * new token per row, and eviction by accumulated attention weight; append with
 * rotary positions, block tables on the device, attention behind shared prefixes and
 * over picked pages.
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
#include "sneppx_rotary.h"

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

/* SNEPPX_kv_append with the rotation of sneppx_rotary.h in the same pass: q's heads
 * (q_heads of them, 0 for none) turned into q_out as SNEPPX_rotary_apply does, k's
 * turned and written to the cache, v's written as they are.  Tokens have their places
 * from a map: slots int32 [tokens], token t's page * page_size + offset, as
 * SNEPPX_kv_reserve writes it; a token whose slot is outside the pool is not written
 * (its query is turned all the same).  No two tokens have one slot.  positions int32
 * [tokens] are those of the rotation and of cache->positions.  SNEPPX_INT8 quantizes
 * the turned fp32 rows.  k_stored, v_stored, weights as in SNEPPX_kv_append. */
int SNEPPX_kv_append_rotated(const SNEPPXKVCache* cache, const SNEPPXRotary* rotary, const uint16_t* q,
                             size_t q_stride, uint16_t* q_out, size_t q_out_stride, size_t q_heads,
                             const uint16_t* k, size_t k_stride, const uint16_t* v, size_t v_stride,
                             size_t tokens, const int32_t* slots, const int32_t* positions, uint16_t* k_stored,
                             uint16_t* v_stored, SNEPPXStream stream);

/* ---- pages --------------------------------------------------------------
 * Which pages are in use is held on the device in one array: refs int32 [pages], the
 * number of rows that hold a page, 0 for a free one.  (A program starts with zeros,
 * and -1 in every entry of its block tables.)  The three calls below change refs,
 * block tables and lengths in the order of the stream, without asking the device, so a
 * program can record them into a graph together with the rest of a step.  A row holds
 * the pages that its table names; an entry outside [0, pages) names none.  Tokens go into
 * the pages that a row holds behind its length before it is given others, so what it shares
 * there (a row cut, or begun anew by kv_share) is given back by kv_release first. */

/* Room for new tokens: counts int32 [rows] of them for each row (NULL: one each; below
 * 0 counts as 0), behind its lengths[row].  Entries of the table that they need beyond
 * the pages the row is in, and that name no page, get the lowest free ones, rows in
 * order.  A row is granted all its tokens or none: none if the table has no entries
 * for them, or if it needs pages and the rows up to and with it need more than are
 * free.  granted int32 [rows]: counts or 0; lengths and next_pos (int32 [rows], or
 * NULL) grow by that.
 * starts int32 [rows + 1]: sums of counts (granted or not; cut at INT32_MAX).  The
 * tokens of row r are starts[r] .. starts[r + 1] of `tokens`; slots int32 [tokens] gets
 * page * page_size + offset, or -1 for tokens that are not granted, whose page is not
 * there, or past starts[rows]; positions (int32 [tokens], or NULL) the row's next_pos
 * (without it, its length) from before the call on, -1 for those not granted and past
 * the end.  With tokens below starts[rows] the others are left out.  None of these arrays
 * overlaps another. */
int SNEPPX_kv_reserve(int32_t* refs, size_t pages, size_t page_size, int32_t* block_tables, size_t table_width,
                      int32_t* lengths, int32_t* next_pos, const int32_t* counts, size_t rows, int32_t* starts,
                      int32_t* granted, int32_t* slots, int32_t* positions, size_t tokens, SNEPPXStream stream);

/* Gives back the pages behind lengths[row] tokens (of a row that has ended: length 0;
 * of one cut by an eviction or a rejected draft: its new length): their entries become
 * -1, their refs one less. */
int SNEPPX_kv_release(int32_t* refs, size_t pages, size_t page_size, int32_t* block_tables, size_t table_width,
                      const int32_t* lengths, size_t rows, SNEPPXStream stream);

/* Has rows begin with another row's pages: row r with sources[r] in [0, rows) takes the
 * first counts[r] / page_size entries of row sources[r] (whole pages within that row's
 * length), each one's refs one more, and gives back what its own entries there named;
 * its length becomes what it took, and so does next_pos (or NULL).  Other rows are
 * left as they are, as is a row whose source is itself, or has a source of its own among
 * the other rows in this call (whether or not it takes pages by it). */
int SNEPPX_kv_share(int32_t* refs, size_t pages, size_t page_size, int32_t* block_tables, size_t table_width,
                    int32_t* lengths, int32_t* next_pos, const int32_t* sources, const int32_t* counts, size_t rows,
                    SNEPPXStream stream);

/* ---- attention behind shared prefixes ------------------------------------
 * SNEPPX_kv_attention (without `accumulate`) for rows in groups that begin with the
 * same pages, which are read once for a group and not once for each row.
 * group_starts int32 [groups + 1] (ascending): group g is the rows group_starts[g] ..
 * group_starts[g + 1], and their first prefix_lengths[g] tokens (int32 [groups]) are
 * the same, read once by the table of its first row that is as long; a row is in one
 * group at most, and there are no more groups than rows.  Rows of no group, and rows
 * shorter than their group's prefix, read all their tokens by themselves.  max_length: no
 * row is longer; max_prefix and max_own: about the longest prefix, and the most tokens that
 * a row reads by itself, behind its prefix or all of them.  The last two size the launch:
 * results depend on them by their rounding only, but the time does, for what a row reads
 * by itself beyond max_own is read by one wave for each key-value head and 16 query heads
 * (16 rows behind 16384 tokens 26 us; with one of them a token shorter than that 900 with a
 * max_own of 128 and 137 with one of 16384).  Scratch: a workspace of the calling thread on
 * `stream`. */
int SNEPPX_kv_attention_shared(const SNEPPXKVCache* cache, const uint16_t* q, size_t q_stride, void* out,
                               size_t out_stride, SNEPPXDtype out_dtype, const int32_t* block_tables,
                               size_t table_width, const int32_t* lengths, size_t rows, size_t q_heads,
                               size_t max_length, const int32_t* group_starts, const int32_t* prefix_lengths,
                               size_t groups, size_t max_prefix, size_t max_own, float scale, SNEPPXStream stream);

/* ---- attention over picked pages -----------------------------------------
 * For long rows: of each page and head the least and largest value of every element of
 * its keys is held in bounds, bf16 [pages][kv_heads][2][head_dim]; a query q cannot have
 * a logit in that page beyond sum_d max(q_d least_d, q_d largest_d), and the pages with
 * the largest such sums are attended to. */

/* Renews the bounds of the pages that the last counts[row] (NULL: one) tokens of each
 * row are in, from all tokens of the row in them.  max_count: no count is larger.  Keys
 * count as the cache gives them back (int8: code * scale in fp32, rounded to bf16); a
 * NaN makes both bounds of its element NaN.  An eviction moves tokens between pages: what
 * a row has left is renewed behind it (counts of the new lengths).  Rows that share a page
 * here have the same number of tokens in it. */
int SNEPPX_kv_key_bounds(const SNEPPXKVCache* cache, uint16_t* bounds, const int32_t* block_tables,
                         size_t table_width, const int32_t* lengths, const int32_t* counts, size_t max_count,
                         size_t rows, SNEPPXStream stream);

/* Picks `budget` pages of each row and key-value head: the first `first` and last
 * `recent` of the row's pages (recent >= 1, first + recent <= budget), and the others by
 * their score: the largest sum above over the query heads of the key-value head, taken in
 * fp64 and rounded to fp32 (a product of either bound that is NaN, 0 * inf too, makes it
 * NaN).  Of equal ones the earlier page; a NaN, and a page that is not
 * there, rank below every number.  picked int32 [rows][kv_heads][budget]: the pages in the
 * order of the row, -1 behind the last; picked_lengths int32 [rows]: the tokens in them
 * (the row's last page is the last one picked).  A row of no more than `budget` pages has
 * them all.  picked and picked_lengths do not overlap what is read.  q as in
 * SNEPPX_kv_attention; max_length: no row is longer.  Scratch: a workspace of the calling
 * thread on `stream`. */
int SNEPPX_kv_pick(const SNEPPXKVCache* cache, const uint16_t* bounds, const uint16_t* q, size_t q_stride,
                   size_t q_heads, const int32_t* block_tables, size_t table_width, const int32_t* lengths,
                   size_t rows, size_t max_length, size_t budget, size_t first, size_t recent, int32_t* picked,
                   int32_t* picked_lengths, SNEPPXStream stream);

/* SNEPPX_kv_attention with a block table for each key-value head: picked int32
 * [rows][kv_heads][budget], picked_lengths int32 [rows], as SNEPPX_kv_pick leaves them. */
int SNEPPX_kv_attention_picked(const SNEPPXKVCache* cache, const uint16_t* q, size_t q_stride, void* out,
                               size_t out_stride, SNEPPXDtype out_dtype, const int32_t* picked, size_t budget,
                               const int32_t* picked_lengths, size_t rows, size_t q_heads, float scale,
                               int accumulate, SNEPPXStream stream);

#ifdef __cplusplus
}
#endif

#endif /* SNEPPX_KV_H */
