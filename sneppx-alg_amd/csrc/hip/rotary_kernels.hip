// rotary_kernels.hip - queries and keys turned to their positions, head by head
// normalised first where that is asked for (include/sneppx_rotary.h), and the same with
// keys and values written to the paged cache (SNEPPX_kv_append_rotated).  Built like
// kv_cache_kernels.hip, whose int8 rule it shares.
//
//   x = x / sqrt(mean(x^2) + eps) norm,  (a, b) = (a cos - b sin, b cos + a sin) m
//
// 8, 16 or 32 lanes have a head, eight of its elements each: of the part that turns
// four pairs, so that nothing is exchanged but the sum of squares (and for int8 the
// maximum).  The work is reading and writing every head once; what stands in its way is
// the angles, four fp64 sines and cosines to a lane, so a lane takes
// up to kMostHeads heads of a token with the angles of the first, all their loads in
// flight over that.  2320 tokens of 40 heads of 128, normalised, take 12.3 us (48 MB read
// and written, 4.9 TB/s behind the launch), into an int8 cache 14.5 (62 MB); 16 tokens 2.3
// in a graph, a chain of position, angle, head and result.
#include <hip/hip_runtime.h>

#include <cstdint>

#include "codec.h"
#include "kv_pool.h"
#include "kv_rows.h"
#include "launch.h"
#include "../snx_internal.h"

using namespace snx;

namespace {

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef double f64x2 __attribute__((ext_vector_type(2)));
typedef u32x2 bf16x4_any __attribute__((aligned(2)));      // of any alignment that elements have

hipStream_t S(void* s) { return reinterpret_cast<hipStream_t>(s); }

struct Heads {
    const uint16_t *q, *k, *v;
    uint16_t *q_out, *k_out, *v_out;
    size_t q_stride, k_stride, v_stride, q_out_stride, k_out_stride;    // (v_out: k_out's)
    const double* freqs;
    const float *q_norm, *k_norm;
    const int32_t *positions, *slots;
    uint32_t tokens, q_heads, kv_heads, heads, dim, turning;    // heads: of all kinds; turning: lanes with pairs
    uint32_t groups;           // lane groups of a token, of which lane group i has heads i, i + groups, ..
    Divider by_groups;
    float magnitude, eps;
    int interleaved;
};

constexpr int kMostHeads = 4;

// Sine and cosine times m, both in fp64 and rounded to fp32 once.  The angle in turns,
// without the whole ones (one rounding, by the product's own), then without the quarters:
// what is left, x of up to pi / 4, goes into the series of Taylor up to x^13 and x^12, whose
// next terms are below 2^-45 and 2^-41.  (An fp32 fraction with sines in fp32 is up to two units
// of 2^-24 further off, which codes of an int8 cache next to a border show, and takes as
// long: 2320 tokens 12.4 us so and 12.3; the library's fp64 sines 12.8, into an int8 cache
// 15.3 against 14.5.)
__device__ __forceinline__ void sine_cosine(double angle, double m, float& s, float& c) {
    constexpr double by_turn = 0.15915494309189533577, turn = 6.28318530717958647693;
    const double part = __builtin_fma(angle, by_turn, -__builtin_rint(angle * by_turn));
    const double quarters = __builtin_rint(4.0 * part), x = turn * __builtin_fma(quarters, -0.25, part), y = x * x;
    constexpr double of_sine[6] = {-1.0 / 6, 1.0 / 120, -1.0 / 5040, 1.0 / 362880, -1.0 / 39916800, 1.0 / 6227020800.0};
    constexpr double of_cosine[6] = {-1.0 / 2, 1.0 / 24, -1.0 / 720, 1.0 / 40320, -1.0 / 3628800, 1.0 / 479001600};
    double a = of_sine[5], b = of_cosine[5];
#pragma unroll
    for (int i = 4; i >= 0; i--) {
        a = __builtin_fma(a, y, of_sine[i]);
        b = __builtin_fma(b, y, of_cosine[i]);
    }
    const float s0 = (float)(__builtin_fma(a * y, x, x) * m), c0 = (float)(__builtin_fma(b, y, 1.0) * m);
    const uint32_t q = (uint32_t)(int)quarters;
    s = u2f(f2u((q & 1u) ? c0 : s0) ^ (q & 2u) << 30);
    c = u2f(f2u((q & 1u) ? s0 : c0) ^ ((q + 1u) & 2u) << 30);
}

template <bool APPEND, bool I8, int LR, int HEADS>
__global__ void __launch_bounds__(256) k_rotate(const KVPool p, const Heads n) {
    const uint32_t number = blockIdx.x * (256 / LR) + threadIdx.x / LR, t = n.by_groups(number);
    if (t >= n.tokens) return;
    const uint32_t j0 = number - t * n.groups, lane = threadIdx.x % LR;
    const bool turns = lane < n.turning, in = 8 * lane < n.dim;
    // this lane's elements: four from `lo` on and four from `hi` on
    const uint32_t lo = turns && !n.interleaved ? 4 * lane : 8 * lane;
    const uint32_t hi = turns && !n.interleaved ? 4 * (n.turning + lane) : 8 * lane + 4;

    u32x2 w[HEADS][2];
#pragma unroll
    for (int i = 0; i < HEADS; i++) {
        const uint32_t j = j0 + i * n.groups, jk = j - n.q_heads, jv = jk - n.kv_heads;
        w[i][0] = w[i][1] = u32x2{0u, 0u};
        if (j >= n.heads || !in) continue;
        const uint16_t* x = j < n.q_heads ? n.q + t * n.q_stride + (size_t)j * n.dim
                            : !APPEND || jk < n.kv_heads ? n.k + t * n.k_stride + (size_t)jk * n.dim
                                                         : n.v + t * n.v_stride + (size_t)jv * n.dim;
        w[i][0] = *reinterpret_cast<const bf16x4_any*>(x + lo);
        w[i][1] = *reinterpret_cast<const bf16x4_any*>(x + hi);
    }
    const int32_t pos = n.positions[t];
    uint32_t slot = 0, page = 0;
    if (APPEND) {
        slot = (uint32_t)n.slots[t];
        page = slot < 0x80000000u ? p.page_of(slot) : 0xFFFFFFFFu;
    }
    const bool there = APPEND && page < p.pages;
    float cs[4], sn[4];
    if (turns && (!APPEND || j0 < n.q_heads + n.kv_heads)) {
        const f64x2 f0 = *reinterpret_cast<const f64x2*>(n.freqs + 4 * lane);
        const f64x2 f1 = *reinterpret_cast<const f64x2*>(n.freqs + 4 * lane + 2);
        const double f[4] = {f0[0], f0[1], f1[0], f1[1]};
#pragma unroll
        for (int e = 0; e < 4; e++) {
            sine_cosine((double)pos * f[e], (double)n.magnitude, sn[e], cs[e]);
        }
    }

#pragma unroll
    for (int i = 0; i < HEADS; i++) {
        const uint32_t j = j0 + i * n.groups;
        if (j >= n.heads) break;
        const bool is_q = j < n.q_heads, is_v = APPEND && j >= n.q_heads + n.kv_heads;
        const uint32_t h = is_q ? j : j - n.q_heads - (is_v ? n.kv_heads : 0);
        float f[8];
#pragma unroll
        for (int e = 0; e < 4; e++) {
            f[2 * e] = u2f(w[i][e >> 1][e & 1] << 16);
            f[2 * e + 1] = u2f(w[i][e >> 1][e & 1] & 0xFFFF0000u);
        }
        const float* const norm = is_v ? nullptr : is_q ? n.q_norm : n.k_norm;
        if (norm) {
            f32x4 g[2] = {};
            if (in) {
                g[0] = *reinterpret_cast<const f32x4*>(norm + lo);
                g[1] = *reinterpret_cast<const f32x4*>(norm + hi);
            }
            float sum = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; e++) sum = __builtin_fmaf(f[e], f[e], sum);
            const float r = 1.0f / __builtin_sqrtf(row_sum<LR>(sum) / (float)n.dim + n.eps);
#pragma unroll
            for (int e = 0; e < 8; e++) f[e] = f[e] * r * g[e >> 2][e & 3];
        }
        auto turn = [](float& a, float& b, float c, float s) {
            const float x = a * c - b * s;
            b = b * c + a * s;
            a = x;
        };
        if (turns && !is_v) {
            if (n.interleaved) {
#pragma unroll
                for (int e = 0; e < 4; e++) turn(f[2 * e], f[2 * e + 1], cs[e], sn[e]);
            } else {
#pragma unroll
                for (int e = 0; e < 4; e++) turn(f[e], f[4 + e], cs[e], sn[e]);
            }
        }
        uint32_t r = 0;
        if (APPEND && !is_q) {
            if (!there) continue;
            r = (page * p.heads + h) * p.page_size + (slot - page * p.page_size);
            uint8_t* const pool = is_v ? p.v : p.k;
            if (I8) {
                uint32_t c[2];
                const float s = quantize_row<LR>(f, c);
                if (in) {
                    *reinterpret_cast<uint32_t*>(pool + (size_t)r * n.dim + lo) = c[0];
                    *reinterpret_cast<uint32_t*>(pool + (size_t)r * n.dim + hi) = c[1];
                }
                if (lane == 0) (is_v ? p.vs : p.ks)[r] = s;
            }
            if (lane == 0 && !is_v) {
                if (p.weights) p.weights[r] = 0.0f;
                if (p.positions) p.positions[r] = pos;
            }
        }
        const u32x2 y0{bf16x2_out(f[0], f[1]), bf16x2_out(f[2], f[3])}, y1{bf16x2_out(f[4], f[5]), bf16x2_out(f[6], f[7])};
        if (!in) continue;
        if (APPEND && !I8 && !is_q) {
            uint16_t* const to = reinterpret_cast<uint16_t*>(is_v ? p.v : p.k) + (size_t)r * n.dim;
            *reinterpret_cast<u32x2*>(to + lo) = y0;
            *reinterpret_cast<u32x2*>(to + hi) = y1;
        }
        uint16_t* const to = is_q ? n.q_out + t * n.q_out_stride
                                  : (is_v ? n.v_out : n.k_out) ? (is_v ? n.v_out : n.k_out) + t * n.k_out_stride : nullptr;
        if (!to) continue;
        *reinterpret_cast<bf16x4_any*>(to + (size_t)h * n.dim + lo) = y0;
        *reinterpret_cast<bf16x4_any*>(to + (size_t)h * n.dim + hi) = y1;
    }
}

template <bool APPEND, bool I8, int LR>
int launch(const KVPool& p, Heads& n, hipStream_t s, const char* who) {
    // Four heads to a lane where that leaves every CU eight waves: in a graph 16 tokens of 40
    // heads take 2.3 us with one and 3.4 with four, 600 of them 4.9 and 4.6, 1200 7.8 and 6.2,
    // 2320 13.0 and 9.9 (8 heads to a lane as 4).
    const size_t waves = (size_t)n.tokens * n.heads * LR / 64;
    const int per = waves >= 2048 * kMostHeads ? kMostHeads : 1;
    n.groups = (n.heads + per - 1) / per;
    n.by_groups = divider(n.groups);
    const size_t numbers = (size_t)n.tokens * n.groups, blocks = (numbers * LR + 255) / 256;
    if (blocks > 0xffffff || numbers >= 0x7ffffff0u) {       // a grid has below 2^32 threads
        snx_set_error("%s: %zu tokens of %zu heads are too many", who, (size_t)n.tokens, (size_t)n.heads);
        return -1;
    }
    if (per == 1) k_rotate<APPEND, I8, LR, 1><<<(unsigned)blocks, 256, 0, s>>>(p, n);
    else k_rotate<APPEND, I8, LR, kMostHeads><<<(unsigned)blocks, 256, 0, s>>>(p, n);
    return snx_launch_check("k_rotate");
}

template <bool APPEND, bool I8>
int launch(const KVPool& p, Heads& n, hipStream_t s, const char* who) {
    if (n.dim <= 64) return launch<APPEND, I8, 8>(p, n, s, who);
    if (n.dim <= 128) return launch<APPEND, I8, 16>(p, n, s, who);
    return launch<APPEND, I8, 32>(p, n, s, who);
}

void rotation(Heads& n, const SNEPPXRotary* r, size_t head_dim, size_t tokens, const int32_t* positions) {
    n.freqs = r->freqs;
    n.q_norm = r->q_norm;
    n.k_norm = r->k_norm;
    n.magnitude = r->magnitude;
    n.eps = r->eps;
    n.interleaved = r->interleaved != 0;
    n.turning = (uint32_t)(r->dims / 8);
    n.dim = (uint32_t)head_dim;
    n.tokens = (uint32_t)tokens;
    n.positions = positions;
}

}  // namespace

extern "C" {

int snx_k_rotary(const SNEPPXRotary* r, const uint16_t* q, size_t q_stride, uint16_t* q_out, size_t q_out_stride,
                 size_t q_heads, const uint16_t* k, size_t k_stride, uint16_t* k_out, size_t k_out_stride,
                 size_t kv_heads, size_t head_dim, const int32_t* positions, size_t tokens, void* st) {
    Heads n = {};
    rotation(n, r, head_dim, tokens, positions);
    n.q = q;
    n.k = k;
    n.q_out = q_out;
    n.k_out = k_out;
    n.q_stride = q_stride;
    n.k_stride = k_stride;
    n.q_out_stride = q_out_stride;
    n.k_out_stride = k_out_stride;
    n.q_heads = (uint32_t)q_heads;
    n.kv_heads = (uint32_t)kv_heads;
    n.heads = (uint32_t)(q_heads + kv_heads);
    return launch<false, false>(KVPool{}, n, S(st), "rotary_apply");
}

int snx_k_kv_append_rotated(const SNEPPXKVCache* c, const SNEPPXRotary* r, const uint16_t* q, size_t q_stride,
                            uint16_t* q_out, size_t q_out_stride, size_t q_heads, const uint16_t* k, size_t k_stride,
                            const uint16_t* v, size_t v_stride, size_t tokens, const int32_t* slots,
                            const int32_t* positions, uint16_t* k_stored, uint16_t* v_stored, void* st) {
    const KVPool p = kv_pool(c, nullptr, 0);
    Heads n = {};
    rotation(n, r, c->head_dim, tokens, positions);
    n.q = q;
    n.k = k;
    n.v = v;
    n.q_out = q_out;
    n.k_out = k_stored;
    n.v_out = v_stored;
    n.q_stride = q_stride;
    n.k_stride = k_stride;
    n.v_stride = v_stride;
    n.q_out_stride = q_out_stride;
    n.k_out_stride = c->kv_heads * c->head_dim;
    n.slots = slots;
    n.q_heads = (uint32_t)q_heads;
    n.kv_heads = (uint32_t)c->kv_heads;
    n.heads = (uint32_t)(q_heads + 2 * c->kv_heads);
    return c->dtype == SNEPPX_INT8 ? launch<true, true>(p, n, S(st), "kv_append_rotated")
                                   : launch<true, false>(p, n, S(st), "kv_append_rotated");
}

}  // extern "C"
