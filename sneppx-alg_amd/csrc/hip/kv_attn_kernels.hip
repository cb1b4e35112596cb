// kv_attn_kernels.hip - attention of one new token per row over the paged
// key-value cache (include/sneppx_kv.h).
//
//   s[t] = scale q . k[t],  p = softmax(s),  out = sum_t p[t] v[t]
//
// for the group of query heads that share a key-value head.  Every key and
// value is used for `group` products only, so reading the cache is what bounds
// it, and the kernel is built around reading it once:
//  * k_kv_attn: a workgroup per (row, key-value head, up to 16 of its query
//    heads, chunk of the length).  Its four waves take tiles of 32 tokens in
//    turn, each wave with its own running maximum, sum and output, and meet
//    once at the end.  Heads are the columns of the matrix cores' tiles (a
//    group of fewer leaves columns empty: even at one head the matrix cores
//    have 8 times the work that the reads allow, so that costs nothing).
//  * k_kv_join: with more than one chunk, the chunks' outputs weighted by
//    their maxima and sums, in the order of the chunks; and the sums of the
//    attention weights, from the logits that the first kernel wrote.
#include <hip/hip_runtime.h>

#include <cstdint>

#include "codec.h"
#include "kv_pool.h"
#include "launch.h"
#include "../snx_internal.h"

using namespace snx;

namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef int i32x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) uint8_t* lds_t;

hipStream_t S(void* s) { return reinterpret_cast<hipStream_t>(s); }

constexpr int TILE = 32;              // tokens of a wave's step
constexpr int WAVES = 4;
constexpr int STEP = TILE * WAVES;    // tokens of a workgroup's step: chunks are multiples of it

struct Attn {
    const uint16_t* q;
    void* out;
    size_t q_stride, out_stride;
    const int32_t* lengths;
    float* part;              // [rows][q_heads][splits][dim]
    float2* ml;               // [rows][q_heads][splits]: maximum, sum
    float* logits;            // [rows][q_heads][logit_stride], or NULL
    uint32_t q_heads, max_length, splits, chunk, tiles, logit_stride, pairs;
    float scale_log2;
    int out_f32, q_aligned, direct;
};

// max / sum over the four lanes that differ in bits 4 and 5
__device__ __forceinline__ float swap32(float x, float& y) {
    const u32x2 r = __builtin_amdgcn_permlane32_swap(f2u(x), f2u(x), false, false);
    y = u2f(r[1]);
    return u2f(r[0]);
}
__device__ __forceinline__ float swap16(float x, float& y) {
    const u32x2 r = __builtin_amdgcn_permlane16_swap(f2u(x), f2u(x), false, false);
    y = u2f(r[1]);
    return u2f(r[0]);
}
__device__ __forceinline__ float quad_max(float x) {
    float y;
    x = swap32(x, y);
    x = fmaxf(x, y);
    x = swap16(x, y);
    return fmaxf(x, y);
}
__device__ __forceinline__ float quad_sum(float x) {
    float y;
    x = swap32(x, y);
    x += y;
    x = swap16(x, y);
    return x + y;
}

// eight int8 as bf16 (exact)
__device__ __forceinline__ bf16x8 bytes_to_bf16(uint32_t a, uint32_t b) {
    u32x4 o;
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const uint32_t w = i ? b : a;
        const float f0 = (float)(int8_t)w, f1 = (float)(int8_t)(w >> 8);
        const float f2 = (float)(int8_t)(w >> 16), f3 = (float)(int8_t)(w >> 24);
        o[2 * i] = __builtin_amdgcn_perm(f2u(f1), f2u(f0), 0x07060302u);
        o[2 * i + 1] = __builtin_amdgcn_perm(f2u(f3), f2u(f2), 0x07060302u);
    }
    return __builtin_bit_cast(bf16x8, o);
}

// Eight fp32 as three bf16 pieces each, exactly (24 significant bits cut into
// 8 + 8 + 8): the products with bf16 values then sum as fp32 ones would.
__device__ __forceinline__ void split3(const float (&x)[8], bf16x8 (&piece)[3]) {
    u32x4 o[3];
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
        float a = x[e], b = x[e + 1];
#pragma unroll
        for (int i = 0; i < 3; i++) {
            o[i][e >> 1] = __builtin_amdgcn_perm(f2u(b), f2u(a), 0x07060302u);
            a -= u2f(f2u(a) & 0xFFFF0000u);
            b -= u2f(f2u(b) & 0xFFFF0000u);
        }
    }
#pragma unroll
    for (int i = 0; i < 3; i++) piece[i] = __builtin_bit_cast(bf16x8, o[i]);
}

// Where 16-byte chunk c of token row r lies in a wave's value tile (rows of
// RB bytes).  The transposed reads take 32 (int8: 16) bytes of the same
// columns from 8 (16) rows at once, the writes one chunk of 16 rows: both
// spread over all banks.
template <int RB, bool I8>
__device__ __forceinline__ int v_chunk(int r, int c) {
    if constexpr (I8) {
        constexpr int per = RB < 256 ? 256 / RB : 1;                   // rows in 256 bytes
        const int f = (r / per) ^ ((r >> 4) << 1);
        return r * (RB / 16) + (c ^ (f & (RB / 16 - 1)));
    } else {
        const int f = RB == 128 ? ((r >> 1) & 1) | ((r >> 3) & 1) << 1 : (r & 3) | ((r >> 3) & 1) << 2;
        return r * (RB / 16) + ((((c >> 1) ^ f) << 1) | ((c & 1) ^ (r >> 4)));
    }
}

template <int DP, bool I8>
struct Lds {
    static constexpr int RB = DP * (I8 ? 1 : 2);                // bytes of a token's row
    static constexpr int V = TILE * RB;                         // a wave's value tile
    static constexpr int WAVE = V + (I8 ? 2 * TILE * 4 : 0);    // and its scales
    static constexpr int OS = DP + 4;                           // floats of a head's row at the end
    static constexpr int END = WAVES * 16 * OS * 4;
    static constexpr int ALL = END > WAVES * WAVE ? END : WAVES * WAVE;
};

// Lane l = 16 g + r.  Keys are the A operand of 16x16x32 products (token rows)
// and the queries the B operand (head r), so that a lane ends up with logits
// of head r for 4 tokens of each product; with product t's row r being token
// 8 (r / 4) + 4 t + r % 4 of the tile these are the tokens 8 g .. 8 g + 7: the
// B operand of the product with the values, with no exchange between lanes.
// That product's A operand is the transposed value tile, which the lanes write
// to LDS by rows and read back transposed; its result has head r in every
// lane, so that a new maximum rescales by the lane's own factor.
// The order of the head's elements in the first product is free: lane group g
// takes 16-byte chunks g, g + 4, .. of the token's row.
// A wave's tile is read while it computes the one before: keys into the
// registers that the first product has just used, values into those that
// went to LDS.
template <int DP, bool I8, bool SAVE>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2)))
k_kv_attn(const KVPool p, const Attn a) {
    typedef Lds<DP, I8> L;
    constexpr int NC = L::RB / 64;        // 16-byte chunks of a row per lane
    constexpr int KS = DP / 32;           // products along the head
    constexpr int DT = DP / 16;           // tiles of 16 output elements
    __shared__ __attribute__((aligned(16))) uint8_t lds[L::ALL];
    __shared__ float2 ends[WAVES][16];

    uint32_t x = blockIdx.x;
    const uint32_t ht = x % a.tiles;
    x /= a.tiles;
    const uint32_t split = x % a.splits, bh = x / a.splits;
    const uint32_t b = bh / p.heads, h = bh - b * p.heads;
    const uint32_t len = kv_length(a.lengths, b, a.max_length);
    const uint32_t first = split * a.chunk, last = first + a.chunk < len ? first + a.chunk : len;
    if (first >= len && !(a.direct && split == 0)) return;

    const int tid = threadIdx.x, lane = tid & 63, r = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t group = a.q_heads / p.heads;
    const uint32_t nh = group - ht * 16 < 16 ? group - ht * 16 : 16;
    const uint32_t hq = h * group + ht * 16;             // the first of the tile's query heads
    const uint32_t row_bytes = p.dim * (I8 ? 1 : 2);
    uint8_t* const vt = lds + wave * L::WAVE;
    float* const sc = reinterpret_cast<float*>(vt + L::V);

    bf16x8 q[KS];
#pragma unroll
    for (int s = 0; s < KS; s++) {
        const uint32_t d = I8 ? 16 * (g + 4 * (s >> 1)) + 8 * (s & 1) : 8 * (g + 4 * s);
        u32x4 w = {0u, 0u, 0u, 0u};
        if ((uint32_t)r < nh && d < p.dim) {
            const uint16_t* src = a.q + b * a.q_stride + (size_t)(hq + r) * p.dim + d;
            if (a.q_aligned) w = *reinterpret_cast<const u32x4*>(src);
            else
#pragma unroll
                for (int e = 0; e < 4; e++) w[e] = src[2 * e] | (uint32_t)src[2 * e + 1] << 16;
        }
        q[s] = __builtin_bit_cast(bf16x8, w);
    }

    f32x4 o[DT] = {};
    float m = -INFINITY, sum = 0.0f;
    bool any = false;

    // this lane's two tokens of a tile: the page table's entries, then their rows
    // of the pool (a token that is not there: row 0, read but not used)
    uint32_t entry[2], row[2];
    bool ok[2], ok_next[2];
    auto look = [&](uint32_t base) {
#pragma unroll
        for (int t = 0; t < 2; t++) {
            const uint32_t tok = base + 8 * (r >> 2) + 4 * t + (r & 3);
            entry[t] = tok < last ? (uint32_t)p.tables[(size_t)b * p.width + p.page_of(tok)] : 0xFFFFFFFFu;
        }
    };
    auto find = [&](uint32_t base) {
#pragma unroll
        for (int t = 0; t < 2; t++) {
            const uint32_t tok = base + 8 * (r >> 2) + 4 * t + (r & 3);
            ok_next[t] = entry[t] < p.pages;
            row[t] = ok_next[t] ? (entry[t] * p.heads + h) * p.page_size + (tok - p.page_of(tok) * p.page_size) : 0;
        }
    };
    u32x4 kc[2][NC], vc[2][NC];
    float ksc[2], vsc[2];
    auto chunk_at = [&](const uint8_t* pool, int t, int i) {
        const uint32_t c = 16 * (g + 4 * i);
        return *reinterpret_cast<const u32x4*>(pool + (size_t)row[t] * row_bytes + (c < row_bytes ? c : 0));
    };
    auto load_k = [&] {
#pragma unroll
        for (int t = 0; t < 2; t++) {
#pragma unroll
            for (int i = 0; i < NC; i++) kc[t][i] = chunk_at(p.k, t, i);
            if (I8) ksc[t] = p.ks[row[t]];
        }
    };
    auto load_v = [&] {
#pragma unroll
        for (int t = 0; t < 2; t++) {
#pragma unroll
            for (int i = 0; i < NC; i++) vc[t][i] = chunk_at(p.v, t, i);
            if (I8) vsc[t] = p.vs[row[t]];
        }
    };

    uint32_t base = first + wave * TILE;
    if (base < last) {
        look(base);
        find(base);
        look(base + STEP);
        load_k();
        load_v();
    }
    while (base < last) {
        const uint32_t next = base + STEP;
        ok[0] = ok_next[0];
        ok[1] = ok_next[1];
        const uint64_t t0 = __ballot(ok[0]), t1 = __ballot(ok[1]);      // lanes whose tokens are there
        const bool whole = (t0 & t1) == ~0ull, more = next < last;
        f32x4 s[2];
#pragma unroll
        for (int t = 0; t < 2; t++) {
            s[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int i = 0; i < KS; i++) {
                const u32x4 w = kc[t][I8 ? i >> 1 : i];
                bf16x8 kf;
                if (I8) kf = (i & 1) ? bytes_to_bf16(w[2], w[3]) : bytes_to_bf16(w[0], w[1]);
                else kf = __builtin_bit_cast(bf16x8, w);
                // past the head's end the lane has other elements, maybe NaN
                if (p.dim != DP && (I8 ? 16 * (g + 4 * (i >> 1)) : 8 * (g + 4 * i)) >= (int)p.dim)
                    kf = __builtin_bit_cast(bf16x8, u32x4{0u, 0u, 0u, 0u});
                s[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, q[i], s[t], 0, 0, 0);
            }
        }
        if (I8 && g == 0)
#pragma unroll
            for (int t = 0; t < 2; t++) sc[8 * (r >> 2) + 4 * t + (r & 3)] = ksc[t];
        if (more) {
            find(next);
            look(next + STEP);
            load_k();
        }
        // values to LDS by rows, those of absent tokens as zeros (0 * NaN)
#pragma unroll
        for (int t = 0; t < 2; t++) {
            const int tok = 8 * (r >> 2) + 4 * t + (r & 3);
#pragma unroll
            for (int i = 0; i < NC; i++) {
                u32x4 w = vc[t][i];
                if (!whole && !ok[t]) w = u32x4{0u, 0u, 0u, 0u};
                *reinterpret_cast<u32x4*>(vt + 16 * v_chunk<L::RB, I8>(tok, g + 4 * i)) = w;
            }
            if (I8 && g == 0) sc[TILE + tok] = ok[t] ? vsc[t] : 0.0f;
        }
        if (more) load_v();
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();

        // softmax of the tile's eight logits of this lane's head
        float e[8];
        float top = -INFINITY;
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
            for (int j = 0; j < 4; j++) {
                float v = s[t][j] * a.scale_log2;
                if (I8) v *= sc[8 * g + 4 * t + j];
                if (!whole && !((t ? t1 : t0) >> (4 * g + j) & 1)) v = -INFINITY;
                e[4 * t + j] = v;
                top = fmaxf(top, v);
            }
        if (SAVE && (uint32_t)r < nh) {
            float* dst = a.logits + ((size_t)b * a.q_heads + hq + r) * a.logit_stride + base + 8 * g;
            *reinterpret_cast<f32x4*>(dst) = f32x4{e[0], e[1], e[2], e[3]};
            *reinterpret_cast<f32x4*>(dst + 4) = f32x4{e[4], e[5], e[6], e[7]};
        }
        any |= (t0 | t1) != 0;
        top = quad_max(top);
        // The reference point moves only when a logit passes it by 8 (weights
        // up to 2^8 are no harm): after the first tile hardly ever.
        if (__any(top > m + 8.0f)) {
            const float to = fmaxf(m, top);
            const float f = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - to);
            m = to;
            sum *= f;
#pragma unroll
            for (int i = 0; i < DT; i++) o[i] *= f;
        }
        const float ref = m == -INFINITY ? 0.0f : m;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            e[i] = __builtin_amdgcn_exp2f(e[i] - ref);
            sum += e[i];
            if (I8) e[i] *= sc[TILE + 8 * g + i];
        }
        bf16x8 pc[3];
        split3(e, pc);
#pragma unroll
        for (int dt = 0; dt < DT; dt++) {
            bf16x8 vf;
            if (I8) {
                const int tok = 8 * g + (r >> 1);
                const lds_t at = (lds_t)(vt + 16 * v_chunk<L::RB, true>(tok, dt) + 8 * (r & 1));
                const i32x2 w = __builtin_amdgcn_ds_read_tr8_b64_v2i32((__attribute__((address_space(3))) i32x2*)at);
                vf = bytes_to_bf16((uint32_t)w[0], (uint32_t)w[1]);
            } else {
                s16x4 w[2];
#pragma unroll
                for (int t = 0; t < 2; t++) {
                    const int tok = 8 * g + 4 * t + (r >> 2), c = 2 * dt + ((r >> 1) & 1);
                    const lds_t at = (lds_t)(vt + 16 * v_chunk<L::RB, false>(tok, c) + 8 * (r & 1));
                    w[t] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)at);
                }
                vf = __builtin_bit_cast(bf16x8, __builtin_shufflevector(w[0], w[1], 0, 1, 2, 3, 4, 5, 6, 7));
            }
#pragma unroll
            for (int i = 0; i < 3; i++) o[dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pc[i], o[dt], 0, 0, 0);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        base = next;
    }

    // the waves meet: a maximum of -inf with tokens there is told from no tokens
    // by a sum of 1 (its outputs are zero)
    sum = quad_sum(sum);
    if (m == -INFINITY && any && sum == 0.0f) sum = 1.0f;
    __syncthreads();
    if (g == 0) ends[wave][r] = make_float2(m, sum);
    float* const ow = reinterpret_cast<float*>(lds) + wave * 16 * L::OS;
    if ((uint32_t)r < nh)
#pragma unroll
        for (int dt = 0; dt < DT; dt++) *reinterpret_cast<f32x4*>(ow + r * L::OS + 16 * dt + 4 * g) = o[dt];
    __syncthreads();
    const uint32_t quads = p.dim / 4;
    for (uint32_t i = tid; i < nh * quads; i += 256) {
        const uint32_t hd = i / quads, d = 4 * (i - hd * quads);
        float top = -INFINITY, total = 0.0f;
#pragma unroll
        for (int w = 0; w < WAVES; w++) top = fmaxf(top, ends[w][hd].x);
        f32x4 v = {};
        float plain = 0.0f;
#pragma unroll
        for (int w = 0; w < WAVES; w++) {
            const float2 e = ends[w][hd];
            const float f = e.x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(e.x - top);
            total += f * e.y;
            plain += e.y;
            v += f * *reinterpret_cast<const f32x4*>(reinterpret_cast<float*>(lds) + (w * 16 + hd) * L::OS + d);
        }
        if (top == -INFINITY) total = plain > 1.0f ? 1.0f : plain;
        if (a.direct) {
            const float inv = top == -INFINITY ? total == 0.0f ? 0.0f : NAN : 1.0f / total;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const size_t at = b * a.out_stride + (size_t)(hq + hd) * p.dim + d + j;
                if (a.out_f32) static_cast<float*>(a.out)[at] = v[j] * inv;
                else static_cast<uint16_t*>(a.out)[at] = bf16_out(v[j] * inv);
            }
        } else {
            const size_t at = ((size_t)b * a.q_heads + hq + hd) * a.splits + split;
            *reinterpret_cast<f32x4*>(a.part + at * p.dim + d) = v;
            if (d == 0) a.ml[at] = make_float2(top, total);
        }
    }
}

// One workgroup per (row, key-value head, x): joins the chunks of the group's
// query heads x, x + gridDim.x, .. and, with logits, adds the attention weights
// of tokens 256 x .., every 256 gridDim.x.
__global__ void __launch_bounds__(256) k_kv_join(const KVPool p, const Attn a) {
    __shared__ float2 stat[256];      // of a head: maximum, 1 / sum
    __shared__ float red[256];
    const uint32_t bh = blockIdx.y + blockIdx.z * 65535u;
    if (bh >= a.pairs) return;
    const uint32_t b = bh / p.heads, h = bh - b * p.heads;
    const uint32_t group = a.q_heads / p.heads;
    const uint32_t len = kv_length(a.lengths, b, a.max_length);
    const uint32_t n = (len + a.chunk - 1) / a.chunk;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;

    // maximum and 1 / sum of a query head over its chunks, by one wave: 0 for
    // no tokens, NaN where there are tokens and every logit is -inf
    auto whole = [&](uint32_t hq) {
        const float2* ml = a.ml + ((size_t)b * a.q_heads + hq) * a.splits;
        float top = -INFINITY, total = 0.0f, plain = 0.0f;
        for (uint32_t i = lane; i < n; i += 64) top = fmaxf(top, ml[i].x);
        for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
        for (uint32_t i = lane; i < n; i += 64) {
            const float2 e = ml[i];
            total += (e.x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(e.x - top)) * e.y;
            plain += e.y;
        }
        for (int o = 32; o > 0; o >>= 1) {
            total += __shfl_xor(total, o);
            plain += __shfl_xor(plain, o);
        }
        return make_float2(top, top == -INFINITY ? plain == 0.0f ? 0.0f : NAN : 1.0f / total);
    };

    const uint32_t threads = p.dim <= 64 ? 64 : p.dim <= 128 ? 128 : 256, ways = 256 / threads;
    const uint32_t d = tid % threads, way = tid / threads;
    for (uint32_t j = blockIdx.x; j < group; j += gridDim.x) {
        const uint32_t hq = h * group + j;
        const float2 st = whole(hq);
        const size_t at = ((size_t)b * a.q_heads + hq) * a.splits;
        float v = 0.0f;
        if (d < p.dim)
#pragma unroll 4
            for (uint32_t i = way; i < n; i += ways) {
                const float mx = a.ml[at + i].x;
                v += (mx == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mx - st.x)) * a.part[(at + i) * p.dim + d];
            }
        red[tid] = v;
        __syncthreads();
        if (way == 0 && d < p.dim) {
            for (uint32_t w = 1; w < ways; w++) v += red[w * threads + d];
            const size_t to = b * a.out_stride + (size_t)hq * p.dim + d;
            if (a.out_f32) static_cast<float*>(a.out)[to] = v * st.y;
            else static_cast<uint16_t*>(a.out)[to] = bf16_out(v * st.y);
        }
        __syncthreads();
    }
    if (!a.logits || !len) return;
    for (uint32_t t0 = blockIdx.x * 256; t0 < len; t0 += gridDim.x * 256) {
        const uint32_t t = t0 + tid;
        uint32_t row = 0;
        const bool ok = t < len && p.row(b, h, t, row);
        float w = 0.0f;
        for (uint32_t j0 = 0; j0 < group; j0 += 256) {
            const uint32_t nj = group - j0 < 256 ? group - j0 : 256;
            __syncthreads();
            for (uint32_t j = wave; j < nj; j += 4) {
                const float2 st = whole(h * group + j0 + j);
                if (lane == 0) stat[j] = make_float2(st.x == -INFINITY ? 0.0f : st.x, st.y);
            }
            __syncthreads();
            if (ok) {
                const float* s = a.logits + ((size_t)b * a.q_heads + h * group + j0) * a.logit_stride + t;
#pragma unroll 4
                for (uint32_t j = 0; j < nj; j++)
                    w += __builtin_amdgcn_exp2f(s[(size_t)j * a.logit_stride] - stat[j].x) * stat[j].y;
            }
        }
        if (ok) p.weights[row] += w;
    }
}

uint32_t div_up(size_t a, size_t b) { return (uint32_t)((a + b - 1) / b); }

// How a call is cut: chunks of the longest row, and its parts of the workspace.
struct Plan {
    uint32_t tiles, chunk, splits, logit_stride;
    size_t part, ml, logits;
    bool direct;
    size_t bytes() const { return part + ml + logits; }
};

Plan plan(const SNEPPXKVCache* c, size_t rows, size_t q_heads, size_t max_length, int accumulate) {
    Plan n;
    const size_t group = q_heads / c->kv_heads;
    n.tiles = div_up(group, 16);
    const size_t units = rows * c->kv_heads * n.tiles;
    const size_t want = (size_t)4 * cu_count();
    size_t splits = (want + units - 1) / units;
    const size_t most = max_length ? div_up(max_length, STEP) : 1;
    if (splits > most) splits = most;
    if (splits > 256) splits = 256;
    n.chunk = max_length ? div_up(div_up(max_length, splits), STEP) * STEP : STEP;
    n.splits = max_length ? div_up(max_length, n.chunk) : 1;
    n.direct = n.splits == 1 && !accumulate;
    n.logit_stride = accumulate ? n.splits * n.chunk : 0;
    n.part = n.direct ? 0 : rows * q_heads * n.splits * c->head_dim * sizeof(float);
    n.ml = n.direct ? 0 : rows * q_heads * n.splits * sizeof(float2);
    n.logits = accumulate ? rows * q_heads * (size_t)n.logit_stride * sizeof(float) : 0;
    return n;
}

template <int DP, bool I8>
void launch(unsigned grid, bool save, const KVPool& p, const Attn& a, hipStream_t s) {
    if (save) k_kv_attn<DP, I8, true><<<grid, 256, 0, s>>>(p, a);
    else k_kv_attn<DP, I8, false><<<grid, 256, 0, s>>>(p, a);
}

template <bool I8>
void launch(unsigned grid, bool save, const KVPool& p, const Attn& a, hipStream_t s) {
    if (p.dim <= 64) launch<64, I8>(grid, save, p, a, s);
    else if (p.dim <= 128) launch<128, I8>(grid, save, p, a, s);
    else launch<256, I8>(grid, save, p, a, s);
}

}  // namespace

extern "C" {

size_t snx_kv_attention_ws(const SNEPPXKVCache* c, size_t rows, size_t q_heads, size_t max_length, int accumulate) {
    return plan(c, rows, q_heads, max_length, accumulate).bytes();
}

int snx_k_kv_attention(const SNEPPXKVCache* c, const uint16_t* q, size_t q_stride, void* out, size_t out_stride,
                       int out_f32, const int32_t* tables, size_t width, const int32_t* lengths, size_t rows,
                       size_t q_heads, size_t max_length, float scale, int accumulate, void* ws, void* st) {
    const KVPool p = kv_pool(c, tables, width);
    const Plan n = plan(c, rows, q_heads, max_length, accumulate);
    const size_t blocks = rows * c->kv_heads * n.tiles * n.splits;
    if (blocks > 0xffffff) {          // a grid has below 2^32 threads
        snx_set_error("kv_attention: %zu rows of up to %zu tokens are too many", rows, max_length);
        return -1;
    }
    Attn a;
    a.q = q;
    a.out = out;
    a.q_stride = q_stride;
    a.out_stride = out_stride;
    a.lengths = lengths;
    uint8_t* w = static_cast<uint8_t*>(ws);
    a.part = reinterpret_cast<float*>(w);
    a.logits = accumulate ? reinterpret_cast<float*>(w + n.part) : nullptr;
    a.ml = reinterpret_cast<float2*>(w + n.part + n.logits);
    a.q_heads = (uint32_t)q_heads;
    a.max_length = (uint32_t)max_length;
    a.splits = n.splits;
    a.chunk = n.chunk;
    a.tiles = n.tiles;
    a.logit_stride = n.logit_stride;
    a.pairs = (uint32_t)(rows * c->kv_heads);
    a.scale_log2 = scale * 1.44269504088896340736f;
    a.out_f32 = out_f32;
    a.q_aligned = ((uintptr_t)q & 15u) == 0 && (rows < 2 || q_stride % 8 == 0);
    a.direct = n.direct;
    if (c->dtype == SNEPPX_INT8) launch<true>((unsigned)blocks, accumulate != 0, p, a, S(st));
    else launch<false>((unsigned)blocks, accumulate != 0, p, a, S(st));
    if (snx_launch_check("k_kv_attn")) return -1;
    if (n.direct) return 0;
    const uint32_t group = (uint32_t)(q_heads / c->kv_heads);
    uint32_t gx = group;
    if (accumulate && div_up(max_length, 256) > gx) gx = div_up(max_length, 256);
    const size_t bh = rows * c->kv_heads;
    k_kv_join<<<dim3(gx < 65536 ? gx : 65536, (unsigned)(bh < 65535 ? bh : 65535), div_up(bh, 65535)), 256, 0, S(st)>>>(p, a);
    return snx_launch_check("k_kv_join");
}

}  // extern "C"
