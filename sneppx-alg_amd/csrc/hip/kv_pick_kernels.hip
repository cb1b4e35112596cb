// kv_pick_kernels.hip - which pages of a long row a step attends to
// (include/sneppx_kv.h): bounds of a page's keys, the largest logit that they allow a
// query, and the pages with the largest.
//
//   score[page] = max over the head's queries of sum_d max(q_d least_d, q_d largest_d)
//
// Scores of a row's pages lie close together (2000 of them in a few percent), and one
// that an fp32 sum puts on the other side of the border is another page: they are
// summed in fp64, where products of bf16 numbers are exact and their sums all but so,
// and rounded to fp32 once, whatever the order of the sum.
#include <hip/hip_runtime.h>

#include <cstdint>

#include "codec.h"
#include "kv_pool.h"
#include "launch.h"
#include "../snx_internal.h"

using namespace snx;

namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef u32x4 bf16x8_any __attribute__((aligned(2)));

hipStream_t S(void* s) { return reinterpret_cast<hipStream_t>(s); }

__device__ __forceinline__ void widen(u32x4 w, float (&f)[8]) {
#pragma unroll
    for (int e = 0; e < 4; e++) {
        f[2 * e] = u2f(w[e] << 16);
        f[2 * e + 1] = u2f(w[e] & 0xFFFF0000u);
    }
}

// ------------------------------------------------------------------- bounds
struct Renew {
    uint16_t* bounds;
    const int32_t *lengths, *counts;
    uint32_t rows, each;      // each: pages of a row that its new tokens are in, at most
};

// A workgroup for each page and head: LR lanes a token, eight elements each.
template <bool I8, int LR>
__global__ void __launch_bounds__(256) k_kv_key_bounds(const KVPool p, const Renew a) {
    constexpr int TOKENS = 256 / LR;
    __shared__ float ends[2][TOKENS][LR * 8];
    const uint32_t h = blockIdx.x % p.heads, at = blockIdx.x / p.heads, b = at / a.each, i = at - b * a.each;
    const uint32_t n = kv_length(a.lengths, b, p.width * p.page_size);
    int32_t c = a.counts ? a.counts[b] : 1;
    c = c < 0 ? 0 : (uint32_t)c < n ? c : (int32_t)n;
    if (c == 0) return;
    const uint32_t e = p.page_of(n - (uint32_t)c) + i;
    if (e > p.page_of(n - 1)) return;
    const uint32_t page = (uint32_t)p.table(b, h)[e];
    if (page >= p.pages) return;
    const uint32_t left = n - e * p.page_size, used = left < p.page_size ? left : p.page_size;
    const uint32_t lane = threadIdx.x % LR, first = threadIdx.x / LR, d = 8 * lane;
    const bool in = d < p.dim;
    const size_t r0 = ((size_t)page * p.heads + h) * p.page_size;
    float lo[8], hi[8];
#pragma unroll
    for (int j = 0; j < 8; j++) {
        lo[j] = INFINITY;
        hi[j] = -INFINITY;
    }
    for (uint32_t t = first; t < used && in; t += TOKENS) {
        float f[8];
        if (I8) {
            const u32x2 w = *reinterpret_cast<const u32x2*>(p.k + (r0 + t) * p.dim + d);
            const float s = p.ks[r0 + t];
#pragma unroll
            for (int j = 0; j < 8; j++) f[j] = bf16_to_f32(bf16_out((float)(int8_t)(w[j >> 2] >> (8 * (j & 3))) * s));
        } else {
            widen(*reinterpret_cast<const u32x4*>(p.k + ((r0 + t) * p.dim + d) * 2), f);
        }
#pragma unroll
        for (int j = 0; j < 8; j++) {
            lo[j] = f[j] < lo[j] || f[j] != f[j] ? f[j] : lo[j];       // (a NaN stays)
            hi[j] = f[j] > hi[j] || f[j] != f[j] ? f[j] : hi[j];
        }
    }
#pragma unroll
    for (int j = 0; j < 8; j++) {
        ends[0][first][d + j] = lo[j];
        ends[1][first][d + j] = hi[j];
    }
    __syncthreads();
    uint16_t* const to = a.bounds + ((size_t)page * p.heads + h) * 2 * p.dim;
    const uint32_t groups = used < TOKENS ? used : TOKENS;
    for (uint32_t x = threadIdx.x; x < 2 * p.dim; x += 256) {
        const bool top = x >= p.dim;
        const uint32_t at_d = top ? x - p.dim : x;
        float m = ends[top][0][at_d];
        for (uint32_t k = 1; k < groups; k++) {
            const float f = ends[top][k][at_d];
            m = (top ? f > m : f < m) || f != f ? f : m;
        }
        to[x] = (uint16_t)(f2u(m) >> 16);          // (bf16 already)
    }
}

// -------------------------------------------------------------------- picks
struct Pick {
    const uint16_t *bounds, *q;
    size_t q_stride;
    const int32_t* lengths;
    uint32_t* keys;            // [rows][heads][most]
    int32_t *picked, *picked_lengths;
    uint32_t rows, group, most, max_length, budget, first, recent;
};

constexpr int kHeadsAtOnce = 4;

// Numbers that order as scores do: NaN lowest, zeros alike, all ones above any.
__device__ __forceinline__ uint32_t score_key(float s) {
    if (s != s) return 0u;
    const uint32_t u = f2u(s + 0.0f);
    return (u >> 31) ? ~u : u | 0x80000000u;
}

template <int CTRL>
__device__ __forceinline__ double lane_step64(double x) {
    const uint64_t u = __builtin_bit_cast(uint64_t, x);
    const uint32_t lo = lane_step<CTRL, 0xf>((uint32_t)u, 0u), hi = lane_step<CTRL, 0xf>((uint32_t)(u >> 32), 0u);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
template <int LR>
__device__ __forceinline__ double row_sum64(double x) {
    x += lane_step64<0xB1>(x);
    x += lane_step64<0x4E>(x);
    x += lane_step64<0x141>(x);
    if (LR >= 16) x += lane_step64<0x140>(x);
    if (LR >= 32) x += __shfl_xor(x, 16);
    return x;
}

// LR lanes a page, eight elements each; blockIdx.y (and z): row and head.
template <int LR>
__global__ void __launch_bounds__(256) k_kv_scores(const KVPool p, const Pick a) {
    const uint32_t bh = blockIdx.y + blockIdx.z * 65535u;
    if (bh >= a.rows * p.heads) return;
    const uint32_t b = bh / p.heads, h = bh - b * p.heads;
    const uint32_t n = kv_length(a.lengths, b, a.max_length), have = p.page_of(n + p.page_size - 1);
    const uint32_t e = blockIdx.x * (256 / LR) + threadIdx.x / LR;
    if (have <= a.budget || e >= have) return;
    uint32_t* const key = a.keys + (size_t)bh * a.most + e;
    const uint32_t lane = threadIdx.x % LR, d = 8 * lane;
    const bool always = e < a.first || e >= have - a.recent;
    const uint32_t page = (uint32_t)p.table(b, h)[e];
    if (always || page >= p.pages) {
        if (lane == 0) *key = always ? 0xFFFFFFFFu : 0u;
        return;
    }
    const bool in = d < p.dim;
    float lo[8] = {}, hi[8] = {};
    if (in) {
        const uint16_t* const x = a.bounds + ((size_t)page * p.heads + h) * 2 * p.dim + d;
        widen(*reinterpret_cast<const u32x4*>(x), lo);
        widen(*reinterpret_cast<const u32x4*>(x + p.dim), hi);
    }
    float best = -INFINITY;
    for (uint32_t g0 = 0; g0 < a.group; g0 += kHeadsAtOnce) {
        double sum[kHeadsAtOnce];
#pragma unroll
        for (int g = 0; g < kHeadsAtOnce; g++) {
            sum[g] = 0.0;
            const uint32_t j = g0 + g < a.group ? g0 + g : a.group - 1;
            float q[8] = {};
            if (in) widen(*reinterpret_cast<const bf16x8_any*>(a.q + b * a.q_stride + (size_t)(h * a.group + j) * p.dim + d), q);
#pragma unroll
            for (int k = 0; k < 8; k++) sum[g] += (double)q[k] * (double)(q[k] > 0.0f ? hi[k] : lo[k]);
        }
#pragma unroll
        for (int g = 0; g < kHeadsAtOnce; g++) {
            const float s = (float)row_sum64<LR>(sum[g]);
            best = s > best || s != s ? s : best;             // (a NaN stays)
        }
    }
    if (lane == 0) *key = score_key(best);
}

constexpr int kWaves = 16, kThreads = 64 * kWaves;

// Over the workgroup: inclusive prefixes and the total.
__device__ __forceinline__ uint32_t block_prefix(uint32_t x, uint32_t* sh, uint32_t& total) {
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t mine = lane_prefix(x);
    __syncthreads();
    if (lane == 63) sh[w] = mine;
    __syncthreads();
    const uint32_t upto = lane_prefix(lane < kWaves ? sh[lane] : 0u);
    total = __builtin_amdgcn_readlane(upto, kWaves - 1);
    return mine + (w ? (uint32_t)__builtin_amdgcn_readlane(upto, w - 1) : 0u);
}

// A workgroup for each row and head: the budget-th largest key by digits of 8 bits,
// each a histogram of the keys that agree so far, then the pages above it and the
// first of those that equal it, in order.
__global__ void __launch_bounds__(kThreads) k_kv_pick(const KVPool p, const Pick a) {
    __shared__ uint32_t bins[256], sh[kWaves], chosen[2];
    const uint32_t tid = threadIdx.x, bh = blockIdx.x, b = bh / p.heads, h = bh - b * p.heads;
    const uint32_t n = kv_length(a.lengths, b, a.max_length), have = p.page_of(n + p.page_size - 1);
    const int32_t* const table = p.table(b, h);
    int32_t* const to = a.picked + (size_t)bh * a.budget;
    if (h == 0 && tid == 0)
        a.picked_lengths[b] = (int32_t)(have > a.budget ? n - (have - a.budget) * p.page_size : n);
    if (have <= a.budget) {
        for (uint32_t i = tid; i < a.budget; i += kThreads) to[i] = i < have ? table[i] : -1;
        return;
    }
    const uint32_t* const keys = a.keys + (size_t)bh * a.most;
    uint32_t left = a.budget, prefix = 0;       // of the keys that agree so far, how many are to be kept
    for (int shift = 24; shift >= 0; shift -= 8) {
        if (tid < 256) bins[tid] = 0;
        __syncthreads();
        for (uint32_t e = tid; e < have; e += kThreads) {
            const uint32_t k = keys[e];
            if (shift == 24 || (k >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&bins[(k >> shift) & 255], 1u);
        }
        __syncthreads();
        // the digit in which the left-th largest is: counts from the top
        uint32_t total;
        const uint32_t c = tid < 256 ? bins[255 - tid] : 0, upto = block_prefix(c, sh, total);
        if (tid < 256 && upto >= left && upto - c < left) {
            chosen[0] = 255 - tid;
            chosen[1] = left - (upto - c);
        }
        __syncthreads();
        prefix |= chosen[0] << shift;
        left = chosen[1];
    }
    uint32_t above = 0, equal = 0;              // of the pages before
    for (uint32_t e0 = 0; e0 < have; e0 += kThreads) {
        const uint32_t e = e0 + tid, k = e < have ? keys[e] : 0;
        const uint32_t is_above = e < have && k > prefix, is_equal = e < have && k == prefix;
        uint32_t total;
        const uint32_t before = block_prefix(is_above | is_equal << 16, sh, total) - (is_above | is_equal << 16);
        const uint32_t eq = equal + (before >> 16), at = above + (before & 0xFFFFu) + (eq < left ? eq : left);
        if (is_above || (is_equal && eq < left)) to[at] = table[e];
        above += total & 0xFFFFu;
        equal += total >> 16;
    }
}

template <bool I8>
void bounds(unsigned grid, const KVPool& p, const Renew& a, hipStream_t s) {
    if (p.dim <= 64) k_kv_key_bounds<I8, 8><<<grid, 256, 0, s>>>(p, a);
    else if (p.dim <= 128) k_kv_key_bounds<I8, 16><<<grid, 256, 0, s>>>(p, a);
    else k_kv_key_bounds<I8, 32><<<grid, 256, 0, s>>>(p, a);
}

}  // namespace

extern "C" {

int snx_k_kv_key_bounds(const SNEPPXKVCache* c, uint16_t* to, const int32_t* tables, size_t width,
                        const int32_t* lengths, const int32_t* counts, size_t max_count, size_t rows, void* st) {
    const KVPool p = kv_pool(c, tables, width);
    // (new tokens from the last slot of one page to the first of another)
    size_t each = (max_count + c->page_size - 2) / c->page_size + 1;
    if (each > width) each = width;
    const size_t grid = rows * each * c->kv_heads;
    if (grid > 0xffffff) {            // a grid has below 2^32 threads
        snx_set_error("kv_key_bounds: %zu pages of %zu rows are too many", each, rows);
        return -1;
    }
    Renew a;
    a.bounds = to;
    a.lengths = lengths;
    a.counts = counts;
    a.rows = (uint32_t)rows;
    a.each = (uint32_t)each;
    if (c->dtype == SNEPPX_INT8) bounds<true>((unsigned)grid, p, a, S(st));
    else bounds<false>((unsigned)grid, p, a, S(st));
    return snx_launch_check("k_kv_key_bounds");
}

int snx_k_kv_pick(const SNEPPXKVCache* c, const uint16_t* bounds, const uint16_t* q, size_t q_stride, size_t q_heads,
                  const int32_t* tables, size_t width, const int32_t* lengths, size_t rows, size_t max_length,
                  size_t budget, size_t first, size_t recent, int32_t* picked, int32_t* picked_lengths, void* ws,
                  void* st) {
    const KVPool p = kv_pool(c, tables, width);
    Pick a;
    a.bounds = bounds;
    a.q = q;
    a.q_stride = q_stride;
    a.lengths = lengths;
    a.keys = static_cast<uint32_t*>(ws);
    a.picked = picked;
    a.picked_lengths = picked_lengths;
    a.rows = (uint32_t)rows;
    a.group = (uint32_t)(q_heads / c->kv_heads);
    a.most = (uint32_t)((max_length + c->page_size - 1) / c->page_size);
    a.max_length = (uint32_t)max_length;
    a.budget = (uint32_t)budget;
    a.first = (uint32_t)first;
    a.recent = (uint32_t)recent;
    const size_t bh = rows * c->kv_heads;
    if (ws) {
        const int lr = c->head_dim <= 64 ? 8 : c->head_dim <= 128 ? 16 : 32;
        const size_t gx = ((size_t)a.most * lr + 255) / 256;
        if (gx * bh > 0xffffff) {     // a grid has below 2^32 threads
            snx_set_error("kv_pick: %zu rows of up to %zu tokens are too many", rows, max_length);
            return -1;
        }
        const dim3 grid((unsigned)gx, (unsigned)(bh < 65535 ? bh : 65535), (unsigned)((bh + 65534) / 65535));
        if (lr == 8) k_kv_scores<8><<<grid, 256, 0, S(st)>>>(p, a);
        else if (lr == 16) k_kv_scores<16><<<grid, 256, 0, S(st)>>>(p, a);
        else k_kv_scores<32><<<grid, 256, 0, S(st)>>>(p, a);
        if (snx_launch_check("k_kv_scores")) return -1;
    }
    k_kv_pick<<<(unsigned)bh, kThreads, 0, S(st)>>>(p, a);
    return snx_launch_check("k_kv_pick");
}

}  // extern "C"
