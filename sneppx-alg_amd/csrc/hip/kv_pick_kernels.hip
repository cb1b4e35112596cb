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
#include "kv_rows.h"
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

__device__ __forceinline__ float least_of(float a, float b) { return b < a || b != b ? b : a; }        // (a NaN stays)
__device__ __forceinline__ float largest_of(float a, float b) { return b > a || b != b ? b : a; }

// A workgroup for each page and head: LR lanes a token, eight elements each; tokens meet
// over the lanes of a wave, then in LDS.  What bounds it: length, page, keys and result,
// one after the other (4 us for the newest page of 8 heads, of 16 rows in int8 4.8).
template <bool I8, int LR>
__global__ void __launch_bounds__(256) k_kv_key_bounds(const KVPool p, const Renew a) {
    constexpr int TOKENS = 256 / LR;
    __shared__ float ends[2][4][LR * 8];
    ask_for(p.tables, p.heads, p.page_of.mul, a.rows);
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
    const uint32_t lane = threadIdx.x % LR, d = 8 * lane, wave = threadIdx.x >> 6;
    const bool in = d < p.dim;
    const size_t r0 = ((size_t)page * p.heads + h) * p.page_size;
    float lo[8], hi[8];
#pragma unroll
    for (int j = 0; j < 8; j++) {
        lo[j] = INFINITY;
        hi[j] = -INFINITY;
    }
    constexpr int U = 4;              // tokens in flight
    for (uint32_t t0 = threadIdx.x / LR; t0 < used; t0 += U * TOKENS) {
        u32x4 w[U];
        float s[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            // (past the last token: that one again)
            const uint32_t t = t0 + u * TOKENS < used ? t0 + u * TOKENS : used - 1;
            if (I8) {
                const u32x2 x = *reinterpret_cast<const u32x2*>(p.k + (r0 + t) * p.dim + (in ? d : 0));
                w[u][0] = x[0];
                w[u][1] = x[1];
                s[u] = p.ks[r0 + t];
            } else {
                w[u] = *reinterpret_cast<const u32x4*>(p.k + ((r0 + t) * p.dim + (in ? d : 0)) * 2);
            }
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            float f[8];
            if (I8)
#pragma unroll
                for (int j = 0; j < 8; j++)
                    f[j] = bf16_to_f32(bf16_out((float)(int8_t)(w[u][j >> 2] >> (8 * (j & 3))) * s[u]));
            else widen(w[u], f);
#pragma unroll
            for (int j = 0; j < 8; j++) {
                lo[j] = least_of(lo[j], f[j]);
                hi[j] = largest_of(hi[j], f[j]);
            }
        }
    }
#pragma unroll
    for (int o = LR; o < 64; o <<= 1)
#pragma unroll
        for (int j = 0; j < 8; j++) {
            lo[j] = least_of(lo[j], __shfl_xor(lo[j], o));
            hi[j] = largest_of(hi[j], __shfl_xor(hi[j], o));
        }
    if ((threadIdx.x & 63) < LR)
#pragma unroll
        for (int j = 0; j < 8; j++) {
            ends[0][wave][d + j] = lo[j];
            ends[1][wave][d + j] = hi[j];
        }
    __syncthreads();
    uint16_t* const to = a.bounds + ((size_t)page * p.heads + h) * 2 * p.dim;
    for (uint32_t x = threadIdx.x; x < 2 * p.dim; x += 256) {
        const bool top = x >= p.dim;
        const uint32_t k = top ? x - p.dim : x;
        float m = ends[top][0][k];
#pragma unroll
        for (int j = 1; j < 4; j++) m = top ? largest_of(m, ends[1][j][k]) : least_of(m, ends[0][j][k]);
        to[x] = (uint16_t)(f2u(m) >> 16);          // (bf16 already)
    }
}

// -------------------------------------------------------------------- picks
struct Pick {
    const uint16_t *bounds, *q;
    size_t q_stride;
    const int32_t* lengths;
    uint32_t* keys;            // [rows][heads][most], rows of whole 16 bytes
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
// Four numbers of LR lanes, each summed over them: lane l gets the sum of number l % 4
// (neighbours share two of the four each, pairs one, and so on).
template <int LR>
__device__ __forceinline__ double row_sums64(const double (&x)[4]) {
    const bool odd = threadIdx.x & 1, high = threadIdx.x & 2;
    const double a = (odd ? x[1] : x[0]) + lane_step64<0xB1>(odd ? x[0] : x[1]);
    const double b = (odd ? x[3] : x[2]) + lane_step64<0xB1>(odd ? x[2] : x[3]);
    double y = (high ? b : a) + lane_step64<0x4E>(high ? a : b);
    if (LR == 8) return y + __shfl_xor(y, 4);
    y += lane_step64<0x124>(y);       // (rotations of 16 lanes by 4 and 8 keep l % 4)
    y += lane_step64<0x128>(y);
    if (LR >= 32) y += __shfl_xor(y, 16);
    return y;
}

// LR lanes a page, eight elements each; blockIdx.y (and z): row and head, whose pages the
// workgroups of a row take in turn, so that all have the same of a short one.  For finite
// bounds
//   max(q least, q largest) = q/2 (largest + least) + |q|/2 |largest - least|,
// two fp64 products and no choice, with the queries' conversions once for all pages (FEW:
// up to four query heads).  The end that a query does not take is in both sums and costs
// bits where it is far the larger: a page with a lane whose second sum is beyond 2^20 of what
// is left (below that 33 of 53 bits stand, and 24 are kept), or not finite, is summed up by
// the definition.  (The sums apart need more registers than four waves a SIMD have, which
// would spill 22: one row of 2048 pages 28.7 us with its attention, 30.4 with four waves, 16
// of up to 1024 in int8 45 and 52.6; without that check and four waves 27.9 and 44.3.)
// What bounds it: the bounds' bytes and, near them, fp64 conversions and products: 16 rows
// of up to 1024 pages and 8 heads 15 us (38 MB, 2.5 TB/s), with fp32 sums 11.5; one row of
// 2048 pages 6.9.
template <int LR, bool FEW>
__global__ void __launch_bounds__(256, FEW ? 3 : 2) k_kv_scores(const KVPool p, const Pick a) {
    const uint32_t bh = blockIdx.y + blockIdx.z * 65535u;
    if (bh >= a.rows * p.heads) return;
    const uint32_t b = bh / p.heads, h = bh - b * p.heads;
    const uint32_t lane = threadIdx.x % LR, d = 8 * lane;
    const bool in = d < p.dim;
    const uint32_t stride = gridDim.x * (256 / LR);
    const uint32_t n = kv_length(a.lengths, b, a.max_length), have = p.page_of(n + p.page_size - 1);
    uint32_t e = blockIdx.x * (256 / LR) + threadIdx.x / LR;
    if (have <= a.budget || e >= have) return;
    const int32_t* const table = p.table(b, h);
    uint32_t* const keys = a.keys + (size_t)bh * a.most;

    double x[kHeadsAtOnce][8];        // q / 2
    auto query = [&](uint32_t g) {
        const uint32_t j = g < a.group ? g : a.group - 1;
        u32x4 w = {0u, 0u, 0u, 0u};
        if (in) w = *reinterpret_cast<const bf16x8_any*>(a.q + b * a.q_stride + (size_t)(h * a.group + j) * p.dim + d);
        return w;
    };
    auto queries = [&](uint32_t g0) {
#pragma unroll
        for (int g = 0; g < kHeadsAtOnce; g++) {
            float q[8];
            widen(query(g0 + g), q);
#pragma unroll
            for (int k = 0; k < 8; k++) x[g][k] = (double)(0.5f * q[k]);
        }
    };
    u32x4 next_lo, next_hi;
    auto fetch = [&](uint32_t page, u32x4& lo, u32x4& hi) {
        const uint16_t* const at = a.bounds + ((size_t)(page < p.pages ? page : 0) * p.heads + h) * 2 * p.dim + (in ? d : 0);
        lo = *reinterpret_cast<const u32x4*>(at);
        hi = *reinterpret_cast<const u32x4*>(at + p.dim);
    };
    // a page's sums of four heads by the definition, from memory again
    auto by_definition = [&](uint32_t page, uint32_t g0, double (&sum)[kHeadsAtOnce]) {
        asm volatile("" : "+v"(page), "+v"(g0));       // (nothing is kept for it in registers)
        u32x4 lo, hi;
        fetch(page, lo, hi);
#pragma unroll
        for (int g = 0; g < kHeadsAtOnce; g++) {
            float q[8], l[8], u[8];
            widen(query(g0 + g), q);
            widen(lo, l);
            widen(hi, u);
            sum[g] = 0.0;
#pragma unroll
            for (int k = 0; k < 8; k++) {
                // (a NaN of either stays: 0 * inf; lanes past the head's end have others' bounds)
                const double low = (double)q[k] * (double)l[k], high = (double)q[k] * (double)u[k];
                sum[g] += !in ? 0.0 : high > low || high != high ? high : low;
            }
        }
    };
    uint32_t page = (uint32_t)table[e], next = e + stride < have ? (uint32_t)table[e + stride] : 0u;
    fetch(page, next_lo, next_hi);
    if (FEW) queries(0);
#pragma unroll 1
    for (; e < have; e += stride) {
        float l[8], u[8];
        widen(next_lo, l);
        widen(next_hi, u);
        const uint32_t seen = page;
        page = next;
        if (e + stride < have) {
            fetch(page, next_lo, next_hi);
            if (e + 2 * stride < have) next = (uint32_t)table[e + 2 * stride];
        }
        float best = -INFINITY;
#pragma unroll 1
        for (uint32_t g0 = 0; g0 < (FEW ? 1u : a.group); g0 += kHeadsAtOnce) {
            if (!FEW) queries(g0);
            double sum[kHeadsAtOnce] = {}, wide[kHeadsAtOnce] = {};
#pragma unroll
            for (int k = 0; k < 8; k++) {
                const double mid = (double)u[k] + (double)l[k], half = (double)u[k] - (double)l[k];
#pragma unroll
                for (int g = 0; g < kHeadsAtOnce; g++) {
                    sum[g] = __builtin_fma(x[g][k], mid, sum[g]);
                    wide[g] = __builtin_fma(__builtin_fabs(x[g][k]), __builtin_fabs(half), wide[g]);
                }
            }
            bool fine = true;
#pragma unroll
            for (int g = 0; g < kHeadsAtOnce; g++) {
                sum[g] += wide[g];
                fine &= wide[g] <= 0x1p20 * __builtin_fabs(sum[g]) && __builtin_fabs(sum[g]) < INFINITY;
            }
            if (__any(!fine)) by_definition(seen, g0, sum);
            const double s = row_sums64<LR>(sum);
            // the largest of the four heads (a NaN stays)
            float f = (float)s;
            f = largest_of(f, lane_step<0xB1, 0xf>(f, 0.0f));
            f = largest_of(f, lane_step<0x4E, 0xf>(f, 0.0f));
            best = largest_of(best, f);
        }
        if (lane == 0) keys[e] = seen < p.pages ? score_key(best) : 0u;
    }
}

constexpr int kWaves = 16, kThreads = 64 * kWaves;
constexpr uint32_t kChunk = 4 * kThreads;      // pages of a workgroup at a time
constexpr uint32_t kBins = 2 * kThreads;

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

// A workgroup for each row and head, four pages next to one another to a thread (the first
// 4096 keys stay in registers).  Scores of a row lie close together, so what is searched for
// the smallest key that is kept is the range from the smallest to the largest: cut into
// 2048 equal parts, of the part that it is in again, until all of a part are kept or it
// has one key.  Then the pages that are kept, in order; of those that equal that key the
// first.  What bounds it: two or three rounds of some five barriers, 5.5 us for 2048 pages
// (digits of the key from the top would need all three, their first bins shared by all).
__global__ void __launch_bounds__(kThreads) k_kv_pick(const KVPool p, const Pick a) {
    __shared__ uint32_t bins[kBins], sh[kWaves], ends[2][kWaves], chosen[3];
    const uint32_t tid = threadIdx.x, bh = blockIdx.x, b = bh / p.heads, h = bh - b * p.heads;
    ask_for(p.tables, p.heads, a.rows, a.keys);
    const uint32_t n = kv_length(a.lengths, b, a.max_length), have = p.page_of(n + p.page_size - 1);
    const int32_t* const table = p.table(b, h);
    int32_t* const to = a.picked + (size_t)bh * a.budget;
    if (h == 0 && tid == 0)
        a.picked_lengths[b] = (int32_t)(have > a.budget ? n - (have - a.budget) * p.page_size : n);
    if (have <= a.budget) {
        for (uint32_t i = tid; i < a.budget; i += kThreads) to[i] = i < have ? table[i] : -1;
        return;
    }
    const u32x4* const keys = reinterpret_cast<const u32x4*>(a.keys + (size_t)bh * a.most);
    const uint32_t last = have - a.recent;         // pages from a.first to here are picked among
    auto load = [&](uint32_t c0) { return c0 + 4 * tid < have ? keys[c0 / 4 + tid] : u32x4{0u, 0u, 0u, 0u}; };
    const u32x4 first = load(0);
    auto each = [&](auto&& f) {
        f(0u, first);
        for (uint32_t c0 = kChunk; c0 < have; c0 += kChunk) f(c0, load(c0));
    };
    auto among = [&](uint32_t e) { return e >= a.first && e < last; };

    uint32_t left = a.budget - a.first - a.recent, from = 0xFFFFFFFFu, trim = 0;      // keys from `from` on are kept, of equal ones `trim`
    if (left) {
        uint32_t lo = 0xFFFFFFFFu, hi = 0u;
        each([&](uint32_t c0, u32x4 k) {
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (among(c0 + 4 * tid + j)) {
                    lo = lo < k[j] ? lo : k[j];
                    hi = hi > k[j] ? hi : k[j];
                }
        });
        lo = ~lane_max(~lo);
        hi = lane_max(hi);
        if ((tid & 63) == 0) {
            ends[0][tid >> 6] = lo;
            ends[1][tid >> 6] = hi;
        }
        bins[tid] = bins[tid + kThreads] = 0;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kWaves; w++) {
            lo = lo < ends[0][w] ? lo : ends[0][w];
            hi = hi > ends[1][w] ? hi : ends[1][w];
        }
        for (;;) {
            const uint32_t range = hi - lo, bits = range ? 32 - __builtin_clz(range) : 0, shift = bits > 11 ? bits - 11 : 0;
            each([&](uint32_t c0, u32x4 k) {
#pragma unroll
                for (int j = 0; j < 4; j++)
                    if (among(c0 + 4 * tid + j) && k[j] >= lo && k[j] <= hi) atomicAdd(&bins[(k[j] - lo) >> shift], 1u);
            });
            __syncthreads();
            // the part that has the left-th largest: two parts to a thread, from the top
            const uint32_t c1 = bins[kBins - 1 - 2 * tid], c0 = bins[kBins - 2 - 2 * tid];
            uint32_t total;
            const uint32_t before = block_prefix(c0 + c1, sh, total) - c0 - c1;
            if (before < left && before + c0 + c1 >= left) {
                const bool upper = before + c1 >= left;
                chosen[0] = kBins - 1 - 2 * tid - !upper;
                chosen[1] = left - before - (upper ? 0 : c1);
                chosen[2] = upper ? c1 : c0;
            }
            bins[tid] = bins[tid + kThreads] = 0;
            __syncthreads();
            lo += chosen[0] << shift;
            left = chosen[1];
            if (shift == 0 || chosen[2] == left) {
                from = lo;
                trim = chosen[2] == left ? 0xFFFFFFFFu : left;
                break;
            }
            hi = hi - lo < (1u << shift) - 1 ? hi : lo + (1u << shift) - 1;
            __syncthreads();                       // (chosen is read before it is written again)
        }
    }
    uint32_t above = 0, equal = 0;                 // of the chunks before
    each([&](uint32_t c0, u32x4 k) {
        uint32_t is_above[4], is_equal[4], mine = 0;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const uint32_t e = c0 + 4 * tid + j;
            const bool in = among(e);
            is_above[j] = e < have && (!in || (trim == 0xFFFFFFFFu ? k[j] >= from : k[j] > from));
            is_equal[j] = trim != 0xFFFFFFFFu && in && k[j] == from;
            mine += is_above[j] | is_equal[j] << 16;
        }
        uint32_t total;
        const uint32_t before = block_prefix(mine, sh, total) - mine;
        uint32_t ab = above + (before & 0xFFFFu), eq = equal + (before >> 16);
#pragma unroll
        for (int j = 0; j < 4; j++) {
            if (is_above[j] || (is_equal[j] && eq < trim)) to[ab + (eq < trim ? eq : trim)] = table[c0 + 4 * tid + j];
            ab += is_above[j];
            eq += is_equal[j];
        }
        above += total & 0xFFFFu;
        equal += total >> 16;
    });
}

template <bool I8>
void bounds(unsigned grid, const KVPool& p, const Renew& a, hipStream_t s) {
    if (p.dim <= 64) k_kv_key_bounds<I8, 8><<<grid, 256, 0, s>>>(p, a);
    else if (p.dim <= 128) k_kv_key_bounds<I8, 16><<<grid, 256, 0, s>>>(p, a);
    else k_kv_key_bounds<I8, 32><<<grid, 256, 0, s>>>(p, a);
}

template <int LR>
void scores(dim3 grid, const KVPool& p, const Pick& a, hipStream_t s) {
    if (a.group <= kHeadsAtOnce) k_kv_scores<LR, true><<<grid, 256, 0, s>>>(p, a);
    else k_kv_scores<LR, false><<<grid, 256, 0, s>>>(p, a);
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
    a.most = (uint32_t)((max_length + c->page_size - 1) / c->page_size + 3) / 4 * 4;
    a.max_length = (uint32_t)max_length;
    a.budget = (uint32_t)budget;
    a.first = (uint32_t)first;
    a.recent = (uint32_t)recent;
    const size_t bh = rows * c->kv_heads;
    if (ws) {
        // As many pages to a lane as leave every CU its waves, up to 16 (the next page's bounds
        // are on their way while one is summed up; 16 rows of 2048 pages 67 us with up to
        // 4, 63 with 8 and 61 with 16).
        const int lr = c->head_dim <= 64 ? 8 : c->head_dim <= 128 ? 16 : 32;
        size_t pages = (size_t)a.most * bh * lr / 64 / (16 * (size_t)cu_count());
        pages = pages < 1 ? 1 : pages > 16 ? 16 : pages;
        const size_t gx = ((size_t)a.most * lr + 256 * pages - 1) / (256 * pages);
        if (gx * bh > 0xffffff) {     // a grid has below 2^32 threads
            snx_set_error("kv_pick: %zu rows of up to %zu tokens are too many", rows, max_length);
            return -1;
        }
        const dim3 grid((unsigned)gx, (unsigned)(bh < 65535 ? bh : 65535), (unsigned)((bh + 65534) / 65535));
        if (lr == 8) scores<8>(grid, p, a, S(st));
        else if (lr == 16) scores<16>(grid, p, a, S(st));
        else scores<32>(grid, p, a, S(st));
        if (snx_launch_check("k_kv_scores")) return -1;
    }
    k_kv_pick<<<(unsigned)bh, kThreads, 0, S(st)>>>(p, a);
    return snx_launch_check("k_kv_pick");
}

}  // extern "C"
