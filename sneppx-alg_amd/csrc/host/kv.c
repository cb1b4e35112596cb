/*
 * kv.c - entry points of the paged key-value cache (include/sneppx_kv.h):
 * argument checks and workspaces, then the HIP launchers.
 */
#include <stdint.h>

#include "sneppx_kv.h"
#include "../snx_internal.h"

#define SLOT_KV_MOVES 8
#define SLOT_KV_SCORES 9

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

/* of arrays of m and n entries */
static int meet(const int32_t* a, size_t m, const int32_t* b, size_t n) {
    const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
    return a && b && m && n && x < y + n * sizeof(int32_t) && y < x + m * sizeof(int32_t);
}

static int overlap(const int32_t* a, const int32_t* b, size_t n) { return meet(a, n, b, n); }

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
    return snx_k_kv_attention(cache, q, q_stride, out, out_stride, out_dtype == SNEPPX_FLOAT32, block_tables, table_width, 0,
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

int SNEPPX_kv_append_rotated(const SNEPPXKVCache* cache, const SNEPPXRotary* rotary, const uint16_t* q,
                             size_t q_stride, uint16_t* q_out, size_t q_out_stride, size_t q_heads,
                             const uint16_t* k, size_t k_stride, const uint16_t* v, size_t v_stride,
                             size_t tokens, const int32_t* slots, const int32_t* positions, uint16_t* k_stored,
                             uint16_t* v_stored, SNEPPXStream stream) {
    static const char who[] = "kv_append_rotated";
    if (cache_ok(who, cache) || snx_rotary_check(who, rotary, cache->head_dim)) return -1;
    REQUIRE(!tokens || (k && v && slots && positions), "%s: NULL pointer", who);
    REQUIRE(!tokens || !q_heads || (q && q_out), "%s: NULL q or q_out", who);
    REQUIRE(!k_stored == !v_stored, "%s: k_stored and v_stored go together", who);
    REQUIRE(q_heads <= 65535, "%s: %zu query heads are too many", who, q_heads);
    REQUIRE(tokens <= MAX_SLOTS, "%s: %zu tokens are too many", who, tokens);
    REQUIRE(cache->pages <= (size_t)INT32_MAX / cache->page_size, "%s: slots of %zu pages of %zu pass 31 bits", who,
            cache->pages, cache->page_size);
    const size_t n = cache->kv_heads * cache->head_dim, nq = q_heads * cache->head_dim;
    REQUIRE(tokens < 2 || (k_stride >= n && v_stride >= n && q_stride >= nq && q_out_stride >= nq),
            "%s: a stride (k %zu, v %zu, q %zu, q_out %zu) is below its row of %zu or %zu", who, k_stride, v_stride,
            q_stride, q_out_stride, n, nq);
    REQUIRE(!nq || tokens < 2 || q != q_out || q_stride == q_out_stride, "%s: q in place with another stride", who);
    snx_clear_error();
    if (!tokens) return 0;
    return snx_k_kv_append_rotated(cache, rotary, q, q_stride, q_out, q_out_stride, q_heads, k, k_stride, v, v_stride,
                                   tokens, slots, positions, k_stored, v_stored, stream);
}

/* ---- pages ---- */
static int pages_ok(const char* who, const int32_t* refs, size_t pages, size_t page_size, const int32_t* tables,
                    size_t width, const int32_t* lengths, size_t rows) {
    REQUIRE(pages && page_size, "%s: no pages, or none of their size", who);
    REQUIRE(page_size <= MAX_SLOTS && pages <= (size_t)INT32_MAX / page_size, "%s: slots of %zu pages of %zu pass 31 bits",
            who, pages, page_size);
    if (!rows) return 0;
    REQUIRE(refs && tables && lengths, "%s: NULL refs, block_tables or lengths", who);
    REQUIRE(width, "%s: empty block_tables", who);
    REQUIRE(width <= MAX_SLOTS / page_size, "%s: table_width %zu * page_size %zu is too large", who, width, page_size);
    REQUIRE(rows <= MAX_SLOTS / width, "%s: %zu rows of %zu entries are too many", who, rows, width);
    return 0;
}

int SNEPPX_kv_reserve(int32_t* refs, size_t pages, size_t page_size, int32_t* block_tables, size_t table_width,
                      int32_t* lengths, int32_t* next_pos, const int32_t* counts, size_t rows, int32_t* starts,
                      int32_t* granted, int32_t* slots, int32_t* positions, size_t tokens, SNEPPXStream stream) {
    static const char who[] = "kv_reserve";
    if (pages_ok(who, refs, pages, page_size, block_tables, table_width, lengths, rows)) return -1;
    REQUIRE(!rows || (starts && granted), "%s: NULL starts or granted", who);
    REQUIRE(!rows || !tokens || slots, "%s: NULL slots", who);
    REQUIRE(tokens <= MAX_SLOTS, "%s: %zu tokens are too many", who, tokens);
    /* (written while other threads still read, or what others write) */
    const int32_t* const arrays[] = {lengths, next_pos, counts, granted, starts, slots, positions};
    const size_t entries[] = {rows, rows, rows, rows, rows + 1, tokens, tokens};
    for (int i = 1; i < 7; i++)
        for (int j = 0; j < i; j++)
            REQUIRE(!rows || !meet(arrays[i], entries[i], arrays[j], entries[j]),
                    "%s: lengths, next_pos, counts, granted, starts, slots and positions must not overlap", who);
    snx_clear_error();
    if (!rows) return 0;
    return snx_k_kv_reserve(refs, pages, page_size, block_tables, table_width, lengths, next_pos, counts, rows, starts,
                            granted, slots, positions, tokens, stream);
}

int SNEPPX_kv_release(int32_t* refs, size_t pages, size_t page_size, int32_t* block_tables, size_t table_width,
                      const int32_t* lengths, size_t rows, SNEPPXStream stream) {
    if (pages_ok("kv_release", refs, pages, page_size, block_tables, table_width, lengths, rows)) return -1;
    snx_clear_error();
    if (!rows) return 0;
    return snx_k_kv_release(refs, pages, page_size, block_tables, table_width, lengths, rows, stream);
}

int SNEPPX_kv_share(int32_t* refs, size_t pages, size_t page_size, int32_t* block_tables, size_t table_width,
                    int32_t* lengths, int32_t* next_pos, const int32_t* sources, const int32_t* counts, size_t rows,
                    SNEPPXStream stream) {
    static const char who[] = "kv_share";
    if (pages_ok(who, refs, pages, page_size, block_tables, table_width, lengths, rows)) return -1;
    REQUIRE(!rows || (sources && counts), "%s: NULL sources or counts", who);
    REQUIRE(!overlap(lengths, sources, rows) && !overlap(lengths, counts, rows) && !overlap(lengths, next_pos, rows) &&
                !overlap(next_pos, sources, rows) && !overlap(next_pos, counts, rows),
            "%s: lengths or next_pos overlap sources, counts or one another", who);
    snx_clear_error();
    if (!rows) return 0;
    return snx_k_kv_share(refs, pages, page_size, block_tables, table_width, lengths, next_pos, sources, counts, rows,
                          stream);
}

/* ---- attention of queries over shared prefixes and picked pages ---- */
static int queries_ok(const char* who, const SNEPPXKVCache* c, const uint16_t* q, size_t q_stride, size_t q_heads,
                      size_t rows) {
    REQUIRE(!rows || q, "%s: NULL pointer", who);
    REQUIRE(q_heads && q_heads % c->kv_heads == 0 && q_heads <= 65535,
            "%s: %zu query heads are not a multiple of %zu key-value heads", who, q_heads, c->kv_heads);
    REQUIRE(rows < 2 || q_stride >= q_heads * c->head_dim, "%s: q_stride %zu is below q_heads * head_dim = %zu", who,
            q_stride, q_heads * c->head_dim);
    return 0;
}

static int out_ok(const char* who, const SNEPPXKVCache* c, const void* out, size_t out_stride, SNEPPXDtype dtype,
                  size_t q_heads, size_t rows) {
    REQUIRE(!rows || out, "%s: NULL pointer", who);
    REQUIRE(dtype == SNEPPX_BFLOAT16 || dtype == SNEPPX_FLOAT32, "%s: out_dtype %d is neither bf16 nor fp32", who,
            (int)dtype);
    REQUIRE(rows < 2 || out_stride >= q_heads * c->head_dim, "%s: out_stride %zu is below q_heads * head_dim = %zu", who,
            out_stride, q_heads * c->head_dim);
    return 0;
}

int SNEPPX_kv_attention_shared(const SNEPPXKVCache* cache, const uint16_t* q, size_t q_stride, void* out,
                               size_t out_stride, SNEPPXDtype out_dtype, const int32_t* block_tables,
                               size_t table_width, const int32_t* lengths, size_t rows, size_t q_heads,
                               size_t max_length, const int32_t* group_starts, const int32_t* prefix_lengths,
                               size_t groups, size_t max_prefix, size_t max_own, float scale, SNEPPXStream stream) {
    static const char who[] = "kv_attention_shared";
    if (cache_ok(who, cache) || rows_ok(who, cache, block_tables, table_width, lengths, rows) ||
        queries_ok(who, cache, q, q_stride, q_heads, rows) || out_ok(who, cache, out, out_stride, out_dtype, q_heads, rows))
        return -1;
    REQUIRE(!rows || !groups || (group_starts && prefix_lengths), "%s: NULL group_starts or prefix_lengths", who);
    REQUIRE(groups <= rows, "%s: %zu groups of %zu rows", who, groups, rows);
    snx_clear_error();
    if (!rows) return 0;
    const size_t slots = table_width * cache->page_size;
    if (max_length > slots) max_length = slots;
    if (max_prefix > max_length) max_prefix = max_length;
    if (max_own > max_length) max_own = max_length;
    return snx_k_kv_attention_shared(cache, q, q_stride, out, out_stride, out_dtype == SNEPPX_FLOAT32, block_tables,
                                     table_width, lengths, rows, q_heads, max_length, group_starts, prefix_lengths, groups,
                                     max_prefix, max_own, scale, stream);
}

int SNEPPX_kv_key_bounds(const SNEPPXKVCache* cache, uint16_t* bounds, const int32_t* block_tables,
                         size_t table_width, const int32_t* lengths, const int32_t* counts, size_t max_count,
                         size_t rows, SNEPPXStream stream) {
    static const char who[] = "kv_key_bounds";
    if (cache_ok(who, cache) || rows_ok(who, cache, block_tables, table_width, lengths, rows)) return -1;
    REQUIRE(!rows || bounds, "%s: NULL bounds", who);
    REQUIRE(aligned16(bounds), "%s: bounds must be 16-byte aligned", who);
    snx_clear_error();
    if (!rows || !max_count) return 0;
    const size_t slots = table_width * cache->page_size;
    if (!counts) max_count = 1;
    if (max_count > slots) max_count = slots;
    return snx_k_kv_key_bounds(cache, bounds, block_tables, table_width, lengths, counts, max_count, rows, stream);
}

int SNEPPX_kv_pick(const SNEPPXKVCache* cache, const uint16_t* bounds, const uint16_t* q, size_t q_stride,
                   size_t q_heads, const int32_t* block_tables, size_t table_width, const int32_t* lengths,
                   size_t rows, size_t max_length, size_t budget, size_t first, size_t recent, int32_t* picked,
                   int32_t* picked_lengths, SNEPPXStream stream) {
    static const char who[] = "kv_pick";
    if (cache_ok(who, cache) || rows_ok(who, cache, block_tables, table_width, lengths, rows) ||
        queries_ok(who, cache, q, q_stride, q_heads, rows))
        return -1;
    REQUIRE(!rows || (bounds && picked && picked_lengths), "%s: NULL bounds, picked or picked_lengths", who);
    REQUIRE(aligned16(bounds), "%s: bounds must be 16-byte aligned", who);
    REQUIRE(budget && budget <= MAX_SLOTS / cache->page_size, "%s: budget %zu is 0 or too large", who, budget);
    REQUIRE(recent && recent <= budget && first <= budget - recent, "%s: first %zu and recent %zu (1 at least) do not fit the budget %zu",
            who, first, recent, budget);
    REQUIRE(!overlap(picked_lengths, lengths, rows), "%s: picked_lengths must not be lengths, nor overlap them", who);
    const size_t all = rows * cache->kv_heads * budget;
    REQUIRE(!rows || !(meet(picked, all, block_tables, rows * table_width) || meet(picked, all, lengths, rows) ||
                       meet(picked, all, picked_lengths, rows) || meet(picked_lengths, rows, block_tables, rows * table_width)),
            "%s: picked and picked_lengths must not overlap block_tables, lengths or one another", who);
    snx_clear_error();
    if (!rows) return 0;
    const size_t slots = table_width * cache->page_size;
    if (max_length > slots) max_length = slots;
    const size_t most = (max_length + cache->page_size - 1) / cache->page_size;
    void* ws = NULL;
    if (most > budget) {                              /* (rows of whole 16 bytes) */
        ws = snx_workspace(rows * cache->kv_heads * ((most + 3) / 4 * 4) * sizeof(uint32_t), SLOT_KV_SCORES, stream);
        if (!ws) return -1;
    }
    return snx_k_kv_pick(cache, bounds, q, q_stride, q_heads, block_tables, table_width, lengths, rows, max_length, budget,
                         first, recent, picked, picked_lengths, ws, stream);
}

int SNEPPX_kv_attention_picked(const SNEPPXKVCache* cache, const uint16_t* q, size_t q_stride, void* out,
                               size_t out_stride, SNEPPXDtype out_dtype, const int32_t* picked, size_t budget,
                               const int32_t* picked_lengths, size_t rows, size_t q_heads, float scale,
                               int accumulate, SNEPPXStream stream) {
    static const char who[] = "kv_attention_picked";
    if (cache_ok(who, cache) || rows_ok(who, cache, picked, budget, picked_lengths, rows) ||
        queries_ok(who, cache, q, q_stride, q_heads, rows) || out_ok(who, cache, out, out_stride, out_dtype, q_heads, rows))
        return -1;
    REQUIRE(!accumulate || cache->weights, "%s: accumulate needs the cache's weights", who);
    snx_clear_error();
    if (!rows) return 0;
    return snx_k_kv_attention(cache, q, q_stride, out, out_stride, out_dtype == SNEPPX_FLOAT32, picked, budget, 1,
                              picked_lengths, rows, q_heads, budget * cache->page_size, scale, accumulate != 0, stream);
}
