/*
 * kv.c - entry points of the paged key-value cache (include/sneppx_kv.h):
 * argument checks and workspaces, then the HIP launchers.
 */
#include <stdint.h>

#include "sneppx_kv.h"
#include "../snx_internal.h"

#define SLOT_KV_MOVES 8

#define REQUIRE(cond, ...)               \
    do {                                 \
        if (!(cond)) {                   \
            snx_set_error(__VA_ARGS__);  \
            return -1;                   \
        }                                \
    } while (0)

/* slots of a row are counted in 32 bits on the device, with room to round up */
#define MAX_SLOTS ((size_t)1 << 30)
/* a workgroup of 1024 for each row and head: a grid has below 2^32 threads */
#define MAX_PAIRS (((size_t)1 << 22) - 1)

static int aligned16(const void* p) { return ((uintptr_t)p & 15u) == 0; }

static int overlap(const int32_t* a, const int32_t* b, size_t n) {
    const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b, bytes = n * sizeof(int32_t);
    return a && b && x < y + bytes && y < x + bytes;
}

static int cache_ok(const char* who, const SNEPPXKVCache* c) {
    REQUIRE(c, "%s: NULL cache", who);
    REQUIRE(c->k && c->v, "%s: NULL pointer in the cache", who);
    REQUIRE(aligned16(c->k) && aligned16(c->v), "%s: k and v must be 16-byte aligned", who);
    REQUIRE(c->dtype == SNEPPX_BFLOAT16 || c->dtype == SNEPPX_INT8, "%s: cache dtype %d is neither bf16 nor int8", who,
            (int)c->dtype);
    REQUIRE(c->dtype != SNEPPX_INT8 || (c->k_scales && c->v_scales), "%s: an int8 cache needs k_scales and v_scales", who);
    REQUIRE(c->pages && c->page_size && c->kv_heads && c->head_dim, "%s: empty cache", who);
    const size_t step = c->dtype == SNEPPX_INT8 ? 16 : 8;
    REQUIRE(c->head_dim <= 256 && c->head_dim % step == 0, "%s: head_dim %zu is not a multiple of %zu up to 256", who,
            c->head_dim, step);
    /* token rows of the pool are numbered in 32 bits */
    REQUIRE(c->page_size <= MAX_SLOTS && c->pages <= INT32_MAX && c->kv_heads <= 65535 &&
                c->pages <= (size_t)UINT32_MAX / c->page_size / c->kv_heads,
            "%s: pages * kv_heads * page_size = %zu * %zu * %zu is too large", who, c->pages, c->kv_heads, c->page_size);
    return 0;
}

/* (of no rows nothing is read, and what holds nothing need not have an address) */
static int rows_ok(const char* who, const SNEPPXKVCache* c, const int32_t* tables, size_t width,
                   const int32_t* lengths, size_t rows) {
    if (!rows) return 0;
    REQUIRE(tables && lengths, "%s: NULL block_tables or lengths", who);
    REQUIRE(width, "%s: empty block_tables", who);
    REQUIRE(width <= MAX_SLOTS / c->page_size, "%s: table_width %zu * page_size %zu is too large", who, width,
            c->page_size);
    REQUIRE(rows <= MAX_PAIRS / c->kv_heads, "%s: %zu rows of %zu heads are too many", who, rows, c->kv_heads);
    return 0;
}

int SNEPPX_kv_append(const SNEPPXKVCache* cache, const uint16_t* k, size_t k_stride, const uint16_t* v,
                     size_t v_stride, size_t tokens, const int32_t* starts, uint16_t* k_stored,
                     uint16_t* v_stored, const int32_t* block_tables, size_t table_width,
                     const int32_t* lengths, const int32_t* next_pos, size_t rows, SNEPPXStream stream) {
    static const char who[] = "kv_append";
    if (cache_ok(who, cache) || rows_ok(who, cache, block_tables, table_width, lengths, rows)) return -1;
    const int none = !tokens || !rows;
    REQUIRE(none || (k && v), "kv_append: NULL pointer");
    REQUIRE(!k_stored == !v_stored, "kv_append: k_stored and v_stored go together");
    REQUIRE(none || !cache->positions || next_pos, "kv_append: a cache with positions needs next_pos");
    REQUIRE(starts || tokens == rows, "kv_append: %zu tokens for %zu rows without starts", tokens, rows);
    REQUIRE(tokens <= MAX_SLOTS, "kv_append: %zu tokens are too many", tokens);
    const size_t n = cache->kv_heads * cache->head_dim;
    REQUIRE(tokens < 2 || (k_stride >= n && v_stride >= n), "kv_append: strides %zu, %zu are below kv_heads * head_dim = %zu",
            k_stride, v_stride, n);
    snx_clear_error();
    if (none) return 0;
    return snx_k_kv_append(cache, k, k_stride, v, v_stride, tokens, starts, k_stored, v_stored, block_tables, table_width,
                           lengths, next_pos, rows, stream);
}

int SNEPPX_kv_attention(const SNEPPXKVCache* cache, const uint16_t* q, size_t q_stride, void* out,
                        size_t out_stride, SNEPPXDtype out_dtype, const int32_t* block_tables,
                        size_t table_width, const int32_t* lengths, size_t rows, size_t q_heads,
                        size_t max_length, float scale, int accumulate, SNEPPXStream stream) {
    static const char who[] = "kv_attention";
    if (cache_ok(who, cache) || rows_ok(who, cache, block_tables, table_width, lengths, rows)) return -1;
    REQUIRE(!rows || (q && out), "kv_attention: NULL pointer");
    REQUIRE(out_dtype == SNEPPX_BFLOAT16 || out_dtype == SNEPPX_FLOAT32, "kv_attention: out_dtype %d is neither bf16 nor fp32",
            (int)out_dtype);
    REQUIRE(q_heads && q_heads % cache->kv_heads == 0 && q_heads <= 65535,
            "kv_attention: %zu query heads are not a multiple of %zu key-value heads", q_heads, cache->kv_heads);
    const size_t n = q_heads * cache->head_dim;
    REQUIRE(rows < 2 || (q_stride >= n && out_stride >= n), "kv_attention: strides %zu, %zu are below q_heads * head_dim = %zu",
            q_stride, out_stride, n);
    REQUIRE(!accumulate || cache->weights, "kv_attention: accumulate needs the cache's weights");
    snx_clear_error();
    if (!rows) return 0;
    const size_t slots = table_width * cache->page_size;
    if (max_length > slots) max_length = slots;
    return snx_k_kv_attention(cache, q, q_stride, out, out_stride, out_dtype == SNEPPX_FLOAT32, block_tables, table_width,
                              lengths, rows, q_heads, max_length, scale, accumulate != 0, stream);
}

int SNEPPX_kv_evict(const SNEPPXKVCache* cache, const int32_t* block_tables, size_t table_width,
                    const int32_t* lengths, const int32_t* next_pos, int32_t* new_lengths, size_t rows,
                    size_t max_length, size_t budget, size_t recent, SNEPPXStream stream) {
    static const char who[] = "kv_evict";
    if (cache_ok(who, cache) || rows_ok(who, cache, block_tables, table_width, lengths, rows)) return -1;
    REQUIRE(!rows || next_pos, "kv_evict: NULL next_pos");
    REQUIRE(cache->weights && cache->positions, "kv_evict: needs the cache's weights and positions");
    REQUIRE(budget, "kv_evict: budget == 0");
    REQUIRE(recent <= budget, "kv_evict: recent %zu is beyond the budget %zu", recent, budget);
    /* (written by one head's workgroup while others still read) */
    REQUIRE(!overlap(new_lengths, lengths, rows), "kv_evict: new_lengths must not be lengths, nor overlap them");
    REQUIRE(!overlap(new_lengths, next_pos, rows), "kv_evict: new_lengths must not be next_pos, nor overlap it");
    snx_clear_error();
    if (!rows) return 0;
    const size_t slots = table_width * cache->page_size;
    if (max_length > slots) max_length = slots;
    if (budget > max_length) budget = max_length;    /* nothing is longer */
    const size_t bytes = snx_kv_evict_ws(cache, rows, max_length, budget);
    void* ws = bytes ? snx_workspace(bytes, SLOT_KV_MOVES, stream) : NULL;
    if (bytes && !ws) return -1;
    return snx_k_kv_evict(cache, block_tables, table_width, lengths, next_pos, new_lengths, rows, max_length, budget,
                          recent, ws, stream);
}
