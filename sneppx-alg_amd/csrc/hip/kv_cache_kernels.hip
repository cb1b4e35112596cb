// kv_cache_kernels.hip - writing and cutting the paged key-value cache
// (include/sneppx_kv.h): append and eviction.  The int8 rule has to round as
// quant_kernels.hip does, so this file is built like that one, with IEEE
// divisions and without contraction.
#include <hip/hip_runtime.h>

#include <cfloat>
#include <cstdint>

#include "codec.h"
#include "kv_pool.h"
#include "../snx_internal.h"

using namespace snx;

namespace {

hipStream_t S(void* s) { return reinterpret_cast<hipStream_t>(s); }

// max over non-NaN values, as the reference's `if (a > m) m = a`
__device__ __forceinline__ float nanless_max(float a, float b) { return b > a ? b : a; }

// ------------------------------------------------------------------- append
struct NewRows {
    const uint16_t *k, *v;
    size_t k_stride, v_stride;
    uint16_t *k_stored, *v_stored;
    const int32_t *starts, *lengths, *next_pos;
    uint32_t tokens, rows;
};

// One wave per (token, key or value, head): its head_dim values, up to 4 per
// lane.
template <bool I8>
__global__ void __launch_bounds__(256) k_kv_append(const KVPool p, const NewRows n) {
    const uint64_t item = (uint64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    const uint32_t t = (uint32_t)(item / (2 * p.heads));
    if (t >= n.tokens) return;
    const uint32_t rest = (uint32_t)(item - (uint64_t)t * (2 * p.heads));
    const bool is_v = rest >= p.heads;
    const uint32_t h = is_v ? rest - p.heads : rest;

    // the row of token t: the last one whose tokens start at or before it
    uint32_t b = t;
    int32_t back = 1;
    if (n.starts) {
        uint32_t lo = 0, hi = n.rows;          // starts[lo] <= t < starts[hi], if in any row
        while (hi - lo > 1) {
            const uint32_t mid = (lo + hi) >> 1;
            if (n.starts[mid] <= (int32_t)t) lo = mid;
            else hi = mid;
        }
        b = lo;
        back = n.starts[b + 1] - (int32_t)t;
        if (back <= 0 || n.starts[b] > (int32_t)t) return;
    }
    const int32_t slot = n.lengths[b] - back;
    uint32_t r;
    if (slot < 0 || (uint64_t)slot >= (uint64_t)p.width * p.page_size || !p.row(b, h, (uint32_t)slot, r)) return;

    const uint16_t* x = (is_v ? n.v + t * n.v_stride : n.k + t * n.k_stride) + (size_t)h * p.dim;
    uint8_t* pool = is_v ? p.v : p.k;
    uint16_t* stored = is_v ? n.v_stored : n.k_stored;
    if (stored) stored += ((size_t)t * p.heads + h) * p.dim;
    if (I8) {
        float m = 0.0f;
        for (uint32_t d = lane; d < p.dim; d += 64) m = nanless_max(m, fabsf(bf16_to_f32(x[d])));
        for (int o = 32; o > 0; o >>= 1) m = nanless_max(m, __shfl_xor(m, o));
        const float s = m < FLT_MIN ? 1.0f : m / 127.0f, inv = 1.0f / s;
        for (uint32_t d = lane; d < p.dim; d += 64) {
            const int q = clampi(round_i32(bf16_to_f32(x[d]) * inv), -128, 127);
            reinterpret_cast<int8_t*>(pool)[(size_t)r * p.dim + d] = (int8_t)q;
            if (stored) stored[d] = bf16_out((float)q * s);
        }
        if (lane == 0) (is_v ? p.vs : p.ks)[r] = s;
    } else {
        for (uint32_t d = lane; d < p.dim; d += 64) {
            reinterpret_cast<uint16_t*>(pool)[(size_t)r * p.dim + d] = x[d];
            if (stored) stored[d] = x[d];
        }
    }
    if (lane == 0 && !is_v) {
        if (p.weights) p.weights[r] = 0.0f;
        if (p.positions) p.positions[r] = n.next_pos[b] - back;
    }
}

// ----------------------------------------------------------------- eviction
// What ranks a token: its weight as an unsigned number that orders as the
// floats do (zeros alike, NaN lowest), all ones for a recent one.
__device__ __forceinline__ uint32_t rank_key(float w, int32_t pos, int32_t recent_from) {
    if (pos >= recent_from) return 0xFFFFFFFFu;
    if (w != w) return 0u;
    const uint32_t u = f2u(w == 0.0f ? 0.0f : w);
    return (u >> 31) ? ~u : u | 0x80000000u;
}

constexpr int kCutWaves = 16;
constexpr int kCutThreads = 64 * kCutWaves;

// exclusive prefix over the waves of a per-wave count; *total gets the sum
__device__ __forceinline__ uint32_t wave_prefix(uint32_t count, uint32_t* sh, uint32_t& total) {
    const int w = threadIdx.x >> 6;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh[w] = count;
    __syncthreads();
    uint32_t before = 0, all = 0;
    for (int i = 0; i < kCutWaves; i++) {
        if (i < w) before += sh[i];
        all += sh[i];
    }
    total = all;
    return before;
}

// One workgroup per (row, head): finds the budget-th largest key by its digits
// of 8 bits, from the top (a histogram of the keys that agree with the digits
// found so far), then lists the free slots below the budget and the kept ones
// from it on, both in ascending order, as rows of the pool.
// moves [rows][heads][2][most], counts [rows][heads].
__global__ void __launch_bounds__(kCutThreads) k_kv_cut(const KVPool p, const int32_t* __restrict__ lengths,
                                                        const int32_t* __restrict__ next_pos,
                                                        int32_t* __restrict__ new_lengths, uint32_t max_length,
                                                        uint32_t budget, uint32_t recent, uint32_t most,
                                                        uint32_t* __restrict__ counts, uint32_t* __restrict__ moves) {
    __shared__ uint32_t hist[256], sh[kCutWaves], found[2];
    const uint32_t b = blockIdx.x / p.heads, h = blockIdx.x - b * p.heads;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const uint32_t L = kv_length(lengths, b, max_length);
    uint32_t* const count = counts + blockIdx.x;
    bool gone = false;
    if (L > budget) {
        const uint32_t used = p.page_of(L - 1) + 1;
        for (uint32_t e = tid; e < used; e += kCutThreads)
            gone |= (uint32_t)p.tables[(size_t)b * p.width + e] >= p.pages;
    }
    gone = __syncthreads_or(gone);
    if (tid == 0 && h == 0 && new_lengths) new_lengths[b] = (int32_t)(L > budget && !gone ? budget : L);
    if (L <= budget || gone) {
        if (tid == 0) *count = 0;
        return;
    }
    const int32_t from = (int32_t)((int64_t)next_pos[b] - (int64_t)recent < INT32_MIN
                                       ? INT32_MIN : (int64_t)next_pos[b] - (int64_t)recent);
    auto key = [&](uint32_t t) {
        uint32_t r;
        (void)p.row(b, h, t, r);
        return rank_key(p.weights[r], p.positions[r], from);
    };

    uint32_t prefix = 0, want = budget;      // the want-th largest among the keys that share the prefix
    for (int shift = 24; shift >= 0; shift -= 8) {
        if (tid < 256) hist[tid] = 0;
        __syncthreads();
        const uint32_t mask = shift == 24 ? 0u : 0xFFFFFFFFu << (shift + 8);
        for (uint32_t t = tid; t < L; t += kCutThreads) {
            const uint32_t q = key(t);
            if ((q & mask) == prefix) atomicAdd(&hist[(q >> shift) & 255], 1u);
        }
        __syncthreads();
        if (tid == 0) {
            uint32_t above = 0;
            int d = 255;
            while (above + hist[d] < want) above += hist[d--];
            found[0] = prefix | (uint32_t)d << shift;
            found[1] = want - above;
        }
        __syncthreads();
        prefix = found[0];
        want = found[1];
        __syncthreads();
    }

    // each wave takes consecutive slots, so that order by (wave, step, lane) is
    // order by slot
    const uint32_t per = (L + kCutThreads - 1) / kCutThreads * 64;
    const uint32_t t0 = wave * per, t1 = t0 + per < L ? t0 + per : L;
    const uint64_t below = ((uint64_t)1 << lane) - 1;
    uint32_t n = 0, total;
    for (uint32_t t = t0; t < t1; t += 64)
        n += __popcll(__ballot(t + lane < t1 && key(t + lane) == prefix));
    const uint32_t ties = wave_prefix(n, sh, total);

    uint32_t holes = 0, far = 0, seen = ties;
    for (int pass = 0; pass < 2; pass++) {
        uint32_t hole_at = 0, far_at = 0;
        if (pass == 1) {
            hole_at = wave_prefix(holes, sh, total);
            far_at = wave_prefix(far, sh, total);
            if (tid == 0) *count = total;
            seen = ties;
        }
        for (uint32_t t = t0; t < t1; t += 64) {
            const uint32_t s = t + lane;
            const bool in = s < t1;
            const uint32_t q = in ? key(s) : 0u;
            const bool tie = in && q == prefix;
            const uint64_t tb = __ballot(tie);
            const bool keep = in && (q > prefix || (tie && seen + __popcll(tb & below) < want));
            seen += __popcll(tb);
            const bool hole = in && !keep && s < budget, come = keep && s >= budget;
            const uint64_t hb = __ballot(hole), fb = __ballot(come);
            if (pass == 0) {
                holes += __popcll(hb);
                far += __popcll(fb);
            } else {
                uint32_t r;
                uint32_t* list = moves + (size_t)blockIdx.x * 2 * most;
                if (hole || come) {
                    (void)p.row(b, h, s, r);
                    if (hole) list[hole_at + __popcll(hb & below)] = r;
                    else list[most + far_at + __popcll(fb & below)] = r;
                }
                hole_at += __popcll(hb);
                far_at += __popcll(fb);
            }
        }
    }
}

// The moves, one wave each: rows of k and v and the planes.  Sources lie in
// slots from the budget on and targets below it, so all are independent.
__global__ void __launch_bounds__(256) k_kv_move(const KVPool p, uint32_t row_bytes, uint32_t most,
                                                 const uint32_t* __restrict__ counts,
                                                 const uint32_t* __restrict__ moves) {
    const uint32_t bh = blockIdx.y, n = counts[bh];
    const int lane = threadIdx.x & 63;
    const uint32_t* list = moves + (size_t)bh * 2 * most;
    for (uint32_t i = blockIdx.x * 4 + (threadIdx.x >> 6); i < n; i += gridDim.x * 4) {
        const size_t to = list[i], of = list[most + i];
        for (uint32_t c = lane * 16; c < row_bytes; c += 64 * 16) {
            *reinterpret_cast<uint4*>(p.k + to * row_bytes + c) = *reinterpret_cast<const uint4*>(p.k + of * row_bytes + c);
            *reinterpret_cast<uint4*>(p.v + to * row_bytes + c) = *reinterpret_cast<const uint4*>(p.v + of * row_bytes + c);
        }
        if (lane == 0) {
            p.weights[to] = p.weights[of];
            p.positions[to] = p.positions[of];
            if (p.ks) p.ks[to] = p.ks[of];
            if (p.vs) p.vs[to] = p.vs[of];
        }
    }
}

uint32_t most_moves(size_t max_length, size_t budget) {
    const size_t over = max_length > budget ? max_length - budget : 0;
    return (uint32_t)(over < budget ? over : budget);
}

}  // namespace

extern "C" {

int snx_k_kv_append(const SNEPPXKVCache* c, const uint16_t* k, size_t k_stride, const uint16_t* v, size_t v_stride,
                    size_t tokens, const int32_t* starts, uint16_t* k_stored, uint16_t* v_stored,
                    const int32_t* tables, size_t width, const int32_t* lengths, const int32_t* next_pos,
                    size_t rows, void* st) {
    const KVPool p = kv_pool(c, tables, width);
    const NewRows n{k, v, k_stride, v_stride, k_stored, v_stored, starts, lengths, next_pos, (uint32_t)tokens, (uint32_t)rows};
    const size_t blocks = (tokens * 2 * c->kv_heads + 3) / 4;
    if (blocks > 0x7fffffff) {
        snx_set_error("kv_append: %zu tokens of %zu heads are too many", tokens, c->kv_heads);
        return -1;
    }
    if (c->dtype == SNEPPX_INT8)
        k_kv_append<true><<<(unsigned)blocks, 256, 0, S(st)>>>(p, n);
    else
        k_kv_append<false><<<(unsigned)blocks, 256, 0, S(st)>>>(p, n);
    return snx_launch_check("k_kv_append");
}

size_t snx_kv_evict_ws(const SNEPPXKVCache* c, size_t rows, size_t max_length, size_t budget) {
    return rows * c->kv_heads * (1 + 2 * (size_t)most_moves(max_length, budget)) * sizeof(uint32_t);
}

int snx_k_kv_evict(const SNEPPXKVCache* c, const int32_t* tables, size_t width, const int32_t* lengths,
                   const int32_t* next_pos, int32_t* new_lengths, size_t rows, size_t max_length, size_t budget,
                   size_t recent, void* ws, void* st) {
    const KVPool p = kv_pool(c, tables, width);
    const uint32_t most = most_moves(max_length, budget);
    const size_t bh = rows * c->kv_heads;
    uint32_t* counts = static_cast<uint32_t*>(ws);
    uint32_t* moves = counts + bh;
    k_kv_cut<<<(unsigned)bh, kCutThreads, 0, S(st)>>>(p, lengths, next_pos, new_lengths, (uint32_t)max_length,
                                                      (uint32_t)budget, (uint32_t)(recent < INT32_MAX ? recent : INT32_MAX),
                                                      most, counts, moves);
    if (snx_launch_check("k_kv_cut")) return -1;
    if (!most) return 0;
    const uint32_t row_bytes = (uint32_t)(c->head_dim * (c->dtype == SNEPPX_INT8 ? 1 : 2));
    const uint32_t gx = (most + 3) / 4;
    for (size_t at = 0; at < bh; at += 65535) {
        const size_t n = bh - at < 65535 ? bh - at : 65535;
        k_kv_move<<<dim3(gx < 65536 ? gx : 65536, (unsigned)n), 256, 0, S(st)>>>(p, row_bytes, most, counts + at,
                                                                                moves + at * 2 * most);
        if (snx_launch_check("k_kv_move")) return -1;
    }
    return 0;
}

}  // extern "C"
