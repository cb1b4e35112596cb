// kv_pool.h - a paged key-value pool and the rows' block tables as the kernels
// see them (see include/sneppx_kv.h for the layout).
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "sneppx_kv.h"

namespace snx {

// Division of numbers below 2^31 by d: with 2^(l-1) < d <= 2^l and mul =
// ceil(2^(31+l) / d), x * mul / 2^(31+l) is the quotient plus less than
// x * 2^l / (d 2^(31+l)) < 1 / d.
struct Divider {
    uint32_t mul, shift;
    __device__ __forceinline__ uint32_t operator()(uint32_t x) const { return (uint32_t)(((uint64_t)x * mul) >> shift); }
};
inline Divider divider(size_t d) {
    uint32_t l = 0;
    while (((uint64_t)1 << l) < d) l++;
    return Divider{(uint32_t)((((uint64_t)1 << (31 + l)) + d - 1) / d), 31 + l};
}

struct KVPool {
    uint8_t *k, *v;
    float *ks, *vs, *weights;
    int32_t* positions;
    const int32_t* tables;
    uint32_t width, pages, heads, page_size;
    Divider page_of;           // of a slot (below 2^30)
    uint32_t dim;
    uint32_t row_tables, head_tables;    // tables of a row, and from a head to the next: 1 and 0, or heads and 1

    __device__ __forceinline__ const int32_t* table(uint32_t b, uint32_t h) const {
        return tables + ((size_t)b * row_tables + h * head_tables) * width;
    }

    // Row of the pool (of head_dim values, and of each plane) that holds slot
    // `slot` of head h in row b's pages; false where that page is not there.
    __device__ __forceinline__ bool row(uint32_t b, uint32_t h, uint32_t slot, uint32_t& r) const {
        const uint32_t e = page_of(slot);
        const uint32_t page = (uint32_t)table(b, h)[e];
        r = (page * heads + h) * page_size + (slot - e * page_size);
        return page < pages;
    }
};

inline KVPool kv_pool(const SNEPPXKVCache* c, const int32_t* tables, size_t width, bool of_heads = false) {
    KVPool p;
    p.k = static_cast<uint8_t*>(c->k);
    p.v = static_cast<uint8_t*>(c->v);
    p.ks = c->k_scales;
    p.vs = c->v_scales;
    p.weights = c->weights;
    p.positions = c->positions;
    p.tables = tables;
    p.width = (uint32_t)width;
    p.pages = (uint32_t)c->pages;
    p.heads = (uint32_t)c->kv_heads;
    p.page_size = (uint32_t)c->page_size;
    p.dim = (uint32_t)c->head_dim;
    p.page_of = divider(c->page_size);
    p.row_tables = of_heads ? p.heads : 1;
    p.head_tables = of_heads;
    return p;
}

// Has a kernel's arguments loaded at once at its start: each 64 bytes of them that
// the scalar cache lacks take their time where they are first used otherwise
// (attention of one token: 8.2 us, 7.9 so).  One field of each 64 bytes is named.
template <typename A, typename B, typename C, typename D>
__device__ __forceinline__ void ask_for(A a, B b, C c, D d) {
    asm volatile("" ::"s"(a), "s"(b), "s"(c), "s"(d));
}

// a row's slots in use, of at most `most`
__device__ __forceinline__ uint32_t kv_length(const int32_t* lengths, uint32_t b, uint32_t most) {
    const int32_t n = lengths[b];
    return n < 0 ? 0u : (uint32_t)n < most ? (uint32_t)n : most;
}

// Over the lanes of a wave: a step takes each row of 16 from the lanes `ctrl`
// says (row_shr 1, 2, 4, 8, then row_bcast 15 and 31), `none` where there is none.
template <int CTRL, int ROWS, typename T>
__device__ __forceinline__ T lane_step(T x, T none) {
    return __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(__builtin_bit_cast(int, none), __builtin_bit_cast(int, x), CTRL,
                                                             ROWS, 0xf, false));
}
// inclusive prefixes of an associative operation
template <typename T, typename F>
__device__ __forceinline__ T lane_scan(T x, T none, F op) {
    x = op(x, lane_step<0x111, 0xf>(x, none));
    x = op(x, lane_step<0x112, 0xf>(x, none));
    x = op(x, lane_step<0x114, 0xf>(x, none));
    x = op(x, lane_step<0x118, 0xf>(x, none));
    x = op(x, lane_step<0x142, 0xa>(x, none));
    return op(x, lane_step<0x143, 0xc>(x, none));
}
template <typename T>
__device__ __forceinline__ T last_lane(T x) {
    return __builtin_bit_cast(T, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), 63));
}
__device__ __forceinline__ uint32_t lane_prefix(uint32_t x) {
    return lane_scan(x, 0u, [](uint32_t a, uint32_t b) { return a + b; });
}
__device__ __forceinline__ uint32_t lane_max(uint32_t x) {
    return last_lane(lane_scan(x, 0u, [](uint32_t a, uint32_t b) { return a > b ? a : b; }));
}
__device__ __forceinline__ float lane_max(float x) {
    return last_lane(lane_scan(x, -INFINITY, [](float a, float b) { return fmaxf(a, b); }));
}
__device__ __forceinline__ float lane_sum(float x) {
    return last_lane(lane_scan(x, 0.0f, [](float a, float b) { return a + b; }));
}

}  // namespace snx
