// kv_shared_kernels.hip - attention of one new token per row, for rows in groups that
// begin with the same pages (SNEPPX_kv_attention_shared, include/sneppx_kv.h).
//
//   s[t] = scale q . k[t],  p = softmax(s),  out = sum_t p[t] v[t]
//
// A group's queries over its prefix are a matrix product: all rows' query heads of a
// key-value head against the same tokens.  So the work is cut into units, each a tile of
// up to 128 queries (rows and heads) and a run of tokens that they have in common: of a
// group's prefix, or of a row's own tokens behind it, for which the queries are the row's
// alone.  A workgroup takes a unit, stages 64 tokens at a time in LDS for its four
// waves, and leaves weighted values, maximum and sum of every query; k_kv_shared_join
// adds up what a query has of its prefix and its own tokens.
#include <hip/hip_runtime.h>

#include <atomic>
#include <cfloat>
#include <cstdint>
#include <type_traits>

#include "codec.h"
#include "kv_pieces.h"
#include "kv_pool.h"
#include "launch.h"
#include "../snx_internal.h"

using namespace snx;

namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef u32x4 bf16x8_any __attribute__((aligned(2)));
typedef u32x2 bf16x4_any __attribute__((aligned(2)));
typedef f32x4 f32x4_any __attribute__((aligned(4)));
typedef __attribute__((address_space(3))) uint8_t* lds_t;
typedef __attribute__((address_space(1))) uint8_t* glb_t;

hipStream_t S(void* s) { return reinterpret_cast<hipStream_t>(s); }

__device__ __forceinline__ __amdgpu_buffer_rsrc_t rsrc(const void* p) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), (short)0, -1, 0x00020000);
}

constexpr int SLOT_KV_SHARED = 10;    // of the stream's workspaces
constexpr uint32_t STEP = 64;         // tokens of a step
constexpr uint32_t TILE = 128;        // queries of a unit
constexpr uint32_t kLeast = 3;        // steps of a unit at least, of long prefixes
constexpr int kLag = 8;               // log2 of how far a logit may pass the maximum that weights refer to

struct Shared {
    const uint16_t* q;
    void* out;
    size_t q_stride, out_stride;
    const int32_t *lengths, *starts, *prefix;
    float *part, *own_part;    // [heads][blocks][columns][dim], [rows][heads][own_tiles][splits][own_columns][dim]
    float2 *ml, *own_ml;       // maximum and sum of the same
    uint32_t rows, q_heads, group, groups, max_length;
    uint32_t about, blocks;    // units of the prefixes of a head: about so many, and so many at most
    uint32_t least;            // steps of one at least
    uint32_t columns, own_columns, own_tiles, splits, own_span;    // own_span: tokens of a split but the last
    float scale_log2;          // not negative: `flip` changes the queries' signs instead
    float room, lift;          // log2 of the most that weights of up to 2^kLag sum up to, and that less kLag
    uint32_t flip;
    int out_f32;
};

// The units of the prefixes, worked out by every wave from what only the device knows:
// one group to a lane, all cut into spans of equal length, the spans of a tile next to
// one another.
struct Prefix {
    uint32_t first, rows, tokens;      // the group's first row and number of rows, tokens of its prefix
    uint32_t base, spans, per;         // its first unit, spans of a tile, steps of a span
};
struct Groups {
    const Shared& a;
    Prefix x0;                 // of group `lane`
    uint32_t most, per;
    __device__ __forceinline__ Groups(const Shared& s, uint32_t slots) : a(s), most(slots < s.max_length ? slots : s.max_length) {
        uint32_t total = 0;
        x0 = at(0);
        for (uint32_t g0 = 0; g0 < a.groups; g0 += 64) {
            const Prefix x = g0 ? at(g0) : x0;
            total += __builtin_amdgcn_readlane(lane_prefix(tiles(x) * steps(x)), 63);
        }
        per = (total + a.about - 1) / (a.about ? a.about : 1);
        per = per > a.least ? per : a.least;
    }
    __device__ __forceinline__ Prefix at(uint32_t g0) const {
        const uint32_t g = g0 + (threadIdx.x & 63);
        Prefix x = {};
        if (g < a.groups) {
            const int32_t r0 = a.starts[g], r1 = a.starts[g + 1];
            const uint32_t from = r0 < 0 ? 0u : (uint32_t)r0 < a.rows ? (uint32_t)r0 : a.rows;
            const uint32_t to = r1 < 0 ? 0u : (uint32_t)r1 < a.rows ? (uint32_t)r1 : a.rows;
            x.first = from;
            x.rows = to > from ? to - from : 0;
            x.tokens = kv_length(a.prefix, g, most);
        }
        return x;
    }
    __device__ __forceinline__ uint32_t steps(const Prefix& x) const { return (x.tokens + STEP - 1) / STEP; }
    __device__ __forceinline__ uint32_t tiles(const Prefix& x) const {
        return x.tokens ? (x.rows * a.group + TILE - 1) / TILE : 0;
    }
    // the group whose unit x is, or (ROW) that row x is in; false if there is none
    template <bool ROW>
    __device__ __forceinline__ bool find(uint32_t i, Prefix& out) const {
        uint32_t base = 0;
        for (uint32_t g0 = 0; g0 < a.groups; g0 += 64) {
            const Prefix x = g0 ? at(g0) : x0;
            const uint32_t spans = (steps(x) + per - 1) / per, n = tiles(x) * spans, upto = lane_prefix(n);
            const uint64_t is = ROW ? __ballot(x.tokens && i >= x.first && i - x.first < x.rows)
                                    : __ballot(n && base + upto > i);
            if (is) {
                const int lane = __builtin_ctzll(is);
                auto of = [&](uint32_t v) { return (uint32_t)__builtin_amdgcn_readlane(v, lane); };
                out = Prefix{of(x.first), of(x.rows), of(x.tokens), base + of(upto - n), of(spans), per};
                return true;
            }
            base += __builtin_amdgcn_readlane(upto, 63);
        }
        return false;
    }
};

// The row of a group whose table its prefix is read by: the first that is as long.  False
// if there is none: rows shorter than the prefix have all their tokens for their own (a
// token that one row has and another has not must not meet the other's weights, not even
// as 0 * NaN).
__device__ __forceinline__ bool row_with(const Shared& a, const Prefix& x, uint32_t& row) {
    row = x.first;
    if (kv_length(a.lengths, x.first, x.tokens) == x.tokens) return true;
    for (uint32_t r0 = 0; r0 < x.rows; r0 += 64) {
        const uint32_t r = r0 + (threadIdx.x & 63);
        const uint64_t is = __ballot(r < x.rows && kv_length(a.lengths, x.first + (r < x.rows ? r : 0), x.tokens) == x.tokens);
        row = x.first + r0 + (is ? __builtin_ctzll(is) : 0);
        if (is) return true;
    }
    return false;
}

// A step's keys and values in LDS, in two buffers: token rows of DP bf16 each, their
// 16-byte pieces in an order that spreads what is read at once over all banks: eight
// rows at one place of the keys, four rows at 64 bytes of the values.
template <int DP>
struct Tiles {
    static constexpr int RB = DP * 2, PIECES = RB / 16, T = STEP * RB, BUF = 2 * T;
    static constexpr int OS = DP + 4;                               // floats of a query's row at the end
    static constexpr int SCALES = 2 * BUF, ENDS = SCALES + 2 * 2 * STEP * 4, ALL = ENDS + 2 * 32 * 8;
    static_assert(4 * (32 * (RB + 32) + 16 + 256) <= ALL, "rows' own tokens take their place");
    static_assert(2 * 32 * OS * 4 <= 2 * BUF, "the queries' rows at the end take the tiles' place");
    static __device__ __forceinline__ int key_piece(int tok, int c) { return c ^ (tok & 7); }
    static __device__ __forceinline__ int value_piece(int tok, int c) {
        return c ^ (PIECES >= 16 ? 4 * (tok & 3) : 4 * ((tok >> 1) & 1));
    }
};

// NEAR: bf16 heads of DP in a pool that 32-bit offsets reach; FAR: other bf16 heads.
enum Form { NEAR, FAR, INT8 };

// a lane's logits: as far as their tokens are there, one bit each in `mine`
template <int N, typename F>
__device__ __forceinline__ float masked_max(float* s, uint32_t mine, bool whole, F bit) {
    if (!whole)
#pragma unroll
        for (int r = 0; r < N; r++)
            if (!(mine >> bit(r) & 1)) s[r] = -INFINITY;
    float top = s[0];
#pragma unroll
    for (int r = 1; r < N; r++) top = fmaxf(top, s[r]);
    return top;
}

// A wave's rows of its own tokens' values in LDS: rows of RB bytes, whose stride and order
// spread the transposed reads (32 bytes of the same columns from eight rows at once) and the
// writes (16 bytes of 16 rows) over all banks.
template <int DP>
struct OwnTile {
    static constexpr int RB = DP * 2, STRIDE = RB + 32, UPPER = 16, V = 32 * STRIDE + UPPER, ALL = V + 2 * 32 * 4;
    static __device__ __forceinline__ int row(int tok) {
        return ((tok & 19) | ((tok >> 1) & 4) | ((tok << 1) & 8)) * STRIDE + (tok >> 4) * UPPER;
    }
};

// The tokens of one row from t0 to t1 for up to 16 of its query heads, by one wave: what a
// wave waits for, the others of the CU make use of.  Lane l = 16 g + r.  Keys are the A
// operand of 16x16x32 products and the queries the B operand (column r); with product t's
// row r being token 8 (r / 4) + 4 t + r % 4 of 32, a lane's weights are those of tokens
// 8 g .. 8 g + 7, the B operand of the product with the values.  Keys and values of the
// next 32 tokens are on their way meanwhile, keys into the registers that the first product
// has used, values into those that went to LDS.  64 rows of 512 tokens and 8 heads (134 MB)
// take 27 us, of 0 to 512 (67 MB) 20: spans are cut by the longest row that the host allows
// for, not by what rows have, so the longest wave has twice an equal share.
template <int DP, bool I8>
__device__ __forceinline__ void own_queries(const KVPool& p, const Shared& a, uint32_t b, uint32_t head0, uint32_t nq,
                                            bf16x8 (&q)[DP / 32]) {
    const uint32_t r = threadIdx.x & 15, g = (threadIdx.x & 63) >> 4;
    const uint16_t* const qh = a.q + b * a.q_stride + (size_t)(head0 + (r < nq ? r : nq - 1)) * p.dim;
#pragma unroll
    for (int s = 0; s < DP / 32; s++) {
        const uint32_t d = I8 ? 16 * (g + 4 * (s >> 1)) + 8 * (s & 1) : 8 * (g + 4 * s);
        u32x4 w = {0u, 0u, 0u, 0u};
        if (d < p.dim) w = *reinterpret_cast<const bf16x8_any*>(qh + d) ^ a.flip;
        q[s] = __builtin_bit_cast(bf16x8, w);
    }
}
template <int DP, bool I8>
__device__ __forceinline__ void own_tokens(const KVPool& p, const Shared& a, uint32_t b, uint32_t h, const bf16x8 (&q)[DP / 32],
                                           uint32_t nq, uint32_t t0, uint32_t t1, size_t slot, uint8_t* vt) {
    typedef OwnTile<DP> L;
    constexpr int NC = DP * (I8 ? 1 : 2) / 64, KS = DP / 32, DT = DP / 16;
    const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    const uint32_t dim = p.dim, row_bytes = dim * (I8 ? 1 : 2);
    const int32_t* const table = p.table(b, h);
    float* const sc = reinterpret_cast<float*>(vt + L::V);

    uint32_t entry[2], row[2];
    bool ok[2];
    auto token = [&](int t) { return 8 * (r >> 2) + 4 * t + (r & 3); };
    auto look = [&](uint32_t base) {
#pragma unroll
        for (int t = 0; t < 2; t++) {
            const uint32_t tok = base + token(t);
            entry[t] = tok < t1 ? (uint32_t)table[p.page_of(tok)] : 0xFFFFFFFFu;
        }
    };
    auto find = [&](uint32_t base) {
#pragma unroll
        for (int t = 0; t < 2; t++) {
            const uint32_t tok = base + token(t);
            ok[t] = entry[t] < p.pages;
            row[t] = ok[t] ? (entry[t] * p.heads + h) * p.page_size + (tok - p.page_of(tok) * p.page_size) : 0;
        }
    };
    u32x4 kc[2][NC], vc[2][NC];
    float ksc[2], vsc[2];
    auto fetch = [&](const uint8_t* pool, const float* scales, u32x4 (&to)[2][NC], float (&s)[2]) {
#pragma unroll
        for (int t = 0; t < 2; t++) {
#pragma unroll
            for (int i = 0; i < NC; i++) {
                const uint32_t x = 16 * (g + 4 * i);
                to[t][i] = *reinterpret_cast<const u32x4*>(pool + (size_t)row[t] * row_bytes + (x < row_bytes ? x : 0));
            }
            if (I8) s[t] = scales[row[t]];
        }
    };
    look(t0);
    f32x4 o[DT] = {};
    float m = -INFINITY, sum = 0.0f;
    bool any = false;
    if (t0 < t1) {
        find(t0);
        look(t0 + 32);
        fetch(p.k, p.ks, kc, ksc);
        fetch(p.v, p.vs, vc, vsc);
    }
    for (uint32_t base = t0; base < t1; base += 32) {
        const uint64_t there[2] = {__ballot(ok[0]), __ballot(ok[1])};      // lanes whose tokens are there
        const bool whole = (there[0] & there[1]) == ~0ull, more = base + 32 < t1;
        const bool is[2] = {ok[0], ok[1]};
        float s[8];
#pragma unroll
        for (int t = 0; t < 2; t++) {
            f32x4 x = {};
#pragma unroll
            for (int i = 0; i < KS; i++) {
                u32x4 w = kc[t][I8 ? i >> 1 : i];
                if (I8) w = (i & 1) ? bytes_to_bf16(w[2], w[3]) : bytes_to_bf16(w[0], w[1]);
                // past the head's end the lane has other elements, maybe NaN
                if ((I8 ? 16 * (g + 4 * (i >> 1)) : 8 * (g + 4 * i)) >= (int)dim) w = u32x4{0u, 0u, 0u, 0u};
                x = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, w), q[i], x, 0, 0, 0);
            }
#pragma unroll
            for (int j = 0; j < 4; j++) s[4 * t + j] = x[j];
            if (I8 && g == 0) sc[token(t)] = ksc[t];
        }
        if (more) {
            find(base + 32);
            look(base + 64);
            fetch(p.k, p.ks, kc, ksc);
        }
#pragma unroll
        for (int t = 0; t < 2; t++) {
            const int tok = token(t);
#pragma unroll
            for (int i = 0; i < NC; i++) {
                if (!is[t]) vc[t][i] = u32x4{0u, 0u, 0u, 0u};        // (0 * NaN)
                uint8_t* const to = vt + L::row(tok) + (I8 ? 32 : 16) * (g + 4 * i);
                if (I8) {
                    *reinterpret_cast<u32x4*>(to) = bytes_to_bf16(vc[t][i][0], vc[t][i][1]);
                    *reinterpret_cast<u32x4*>(to + 16) = bytes_to_bf16(vc[t][i][2], vc[t][i][3]);
                } else {
                    *reinterpret_cast<u32x4*>(to) = vc[t][i];
                }
            }
            if (I8 && g == 0) sc[32 + tok] = is[t] ? vsc[t] : 0.0f;
        }
        if (more) fetch(p.v, p.vs, vc, vsc);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        if (I8)
#pragma unroll
            for (int i = 0; i < 8; i++) s[i] *= sc[8 * g + i];
        // (bits of the lane's tokens 8 g .. 8 g + 7: product t has tokens 4 t .. 4 t + 3 of them in lanes 4 g ..)
        const uint32_t mine = ((uint32_t)(there[0] >> (4 * g)) & 15u) | ((uint32_t)(there[1] >> (4 * g)) & 15u) << 4;
        float top = masked_max<8>(s, mine, whole, [](int i) { return i; });
        any |= mine != 0;
        float other;
        top = swap32(top, other);
        top = fmaxf(top, other);
        top = swap16(top, other);
        top = fmaxf(top, other) * a.scale_log2;
        if (__any(top + a.lift > m)) {
            const float to = fmaxf(m, __builtin_ceilf(top) + a.room);
            const float f = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - to);
            m = to;
            sum *= f;
#pragma unroll
            for (int i = 0; i < DT; i++) o[i] *= f;
        }
        const float ref = m == -INFINITY ? 0.0f : m;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            s[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], a.scale_log2, -ref));
            sum += s[i];
            if (I8) s[i] *= sc[32 + 8 * g + i];
        }
        bf16x8 pc[3];
        split3<I8>(s, pc);
#pragma unroll
        for (int dt = 0; dt < DT; dt++) {
            s16x4 w[2];
#pragma unroll
            for (int t = 0; t < 2; t++) {
                const lds_t at = (lds_t)(vt + L::row(8 * g + 4 * t + (r >> 2)) + 8 * (r & 3) + 32 * dt);
                w[t] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)at);
            }
            const bf16x8 vf = __builtin_bit_cast(bf16x8, __builtin_shufflevector(w[0], w[1], 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
            for (int i = 0; i < 3; i++) o[dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pc[i], o[dt], 0, 0, 0);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
    float other;
    sum = swap32(sum, other);
    sum += other;
    sum = swap16(sum, other);
    sum += other;
    // (a maximum of -inf with tokens there is told from no tokens by a sum of 1)
    any = __any(any);
    if (m == -INFINITY && any && sum == 0.0f) sum = 1.0f;
    if ((uint32_t)r >= nq) return;
    if (g == 0) a.own_ml[slot + r] = make_float2(m, sum);
    float* const to = a.own_part + (slot + r) * dim;
#pragma unroll
    for (int dt = 0; dt < DT; dt++)
        if (16 * dt + 4 * g < (int)dim) *reinterpret_cast<f32x4*>(to + 16 * dt + 4 * g) = o[dt];
}

// Lane l = 32 g + c.  Keys are the A operand of 32x32x16 products (32 token rows), the
// queries the B operand (column c), so a lane ends up with 16 logits of query c: register
// 8 p + 4 t + i is token 16 p + 8 t + 4 g + i.  Those of a p are the lane's eight elements
// of the B operand of the second product as they stand, if its A operand, the values
// transposed (ds_read_tr), has tokens in that order.  Its result has query c in every
// lane, so a new maximum rescales by the lane's own factor.
// With more than 64 queries each wave has 32 of them and all tokens of a step; with
// fewer, waves w and w + 2 have the same 32 and half of the tokens each.
// What bounds it: for many queries the products.  1024 queries of a head over 16384 tokens,
// 8 heads: 145 us, 137 GFLOP with the three pieces of a weight, 0.95 PFLOP/s (a plain
// product reaches 1.29); without the lower two 81, in any order of the instructions.  For
// few the chain of a step (look-up, row, tile, logits, maximum, weights), 3 us, a unit of
// three steps 15.
// (Weights in two pieces for bf16 results, 2^-15 of a weight off, put some results on the
// other side of a rounding: 256 rows behind 16384 tokens take 154 us with three pieces and
// 125 with two, 64 behind 4096 33.4 and 32.7.)
// DIM: the head's elements that products are made of, DP those of a row in LDS (heads of 80,
// 256 rows behind 16384 tokens: 135 us with products of 128 elements, 122 of 96).
template <int DIM, Form FORM>
__global__ void __launch_bounds__(256, DIM <= 128 ? 2 : 1) k_kv_shared(const KVPool p, const Shared a) {
    constexpr int DP = DIM <= 64 ? 64 : DIM <= 128 ? 128 : 256;
    typedef Tiles<DP> L;
    constexpr bool I8 = FORM == INT8;
    constexpr int CH = L::PIECES / (I8 ? 2 : 1);           // 16-byte pieces of a row in the pool
    constexpr int KQ = DIM / 16, DT = DIM / 32;
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    float* const scales = reinterpret_cast<float*>(lds + L::SCALES);       // [buffer][keys, values][STEP]
    float2* const ends = reinterpret_cast<float2*>(lds + L::ENDS);         // [2][32]

    const int tid = threadIdx.x, lane = tid & 63, c = lane & 31, g = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);

    // the unit: a tile of a group's queries and a span of its prefix, or by waves a row's own tokens
    const uint32_t shared_blocks = a.blocks * p.heads;
    if (blockIdx.x >= shared_blocks) {
        const uint32_t i = __builtin_amdgcn_readfirstlane((blockIdx.x - shared_blocks) * 4 + wave);
        // (the rows' first spans, then their second ones, ..: workgroups go to the XCDs in
        // turn, and so every XCD gets spans of all kinds)
        const uint32_t pair = i / p.heads, h = i - pair * p.heads, rest = pair / a.own_tiles, tile = pair - rest * a.own_tiles;
        const uint32_t span = rest / a.rows, b = rest - span * a.rows;
        if (span >= a.splits) return;
        // (asked for before what the groups say, which the rest depends on)
        const uint32_t left = a.group - tile * 16, nq = left < 16 ? left : 16;
        bf16x8 q[DP / 32];
        own_queries<DP, I8>(p, a, b, h * a.group + tile * 16, nq, q);
        uint32_t len = kv_length(a.lengths, b, a.max_length);
        const Groups groups(a, p.width * p.page_size);
        len = len < groups.most ? len : groups.most;
        Prefix x;
        const uint32_t begins = groups.find<true>(b, x) && x.tokens <= len ? x.tokens : 0;
        const uint32_t t0 = begins + span * a.own_span;
        if (span && t0 >= len) return;
        const uint32_t t1 = span + 1 < a.splits && len - t0 > a.own_span ? t0 + a.own_span : len;
        own_tokens<DP, I8>(p, a, b, h, q, nq, t0, t1,
                                   ((((size_t)b * p.heads + h) * a.own_tiles + tile) * a.splits + span) * a.own_columns,
                                   lds + wave * OwnTile<DP>::ALL);
        return;
    }
    const Groups groups(a, p.width * p.page_size);
    const uint32_t unit = blockIdx.x / p.heads, h = blockIdx.x - unit * p.heads;
    Prefix x;
    if (!groups.find<false>(unit, x)) return;
    const uint32_t tile = (unit - x.base) / x.spans, span = unit - x.base - tile * x.spans;
    const uint32_t first = x.first, at = tile * TILE, t0 = span * x.per * STEP;
    const uint32_t t1 = t0 + x.per * STEP < x.tokens ? t0 + x.per * STEP : x.tokens;
    const size_t slot = ((size_t)h * a.blocks + unit) * a.columns;
    const uint32_t left = x.rows * a.group - at, nq = left < TILE ? left : TILE;
    const bool wide = nq > 64;
    const uint32_t q0 = 32 * (wide ? wave : wave & 1);       // this wave's first query
    const bool busy = q0 < nq;
    const int32_t* table = p.table(first, h);
    const uint32_t dim = FORM == NEAR ? DP : p.dim, row_bytes = dim * (I8 ? 1 : 2);

    // this lane's token of a step: the page table's entry, then its row of the pool
    uint32_t entry, row;
    bool ok;
    auto look = [&](uint32_t base) {
        const uint32_t tok = base + lane;
        entry = tok < t1 ? (uint32_t)table[p.page_of(tok)] : 0xFFFFFFFFu;
    };
    auto find = [&](uint32_t base) {
        const uint32_t tok = base + lane;
        ok = entry < p.pages;
        row = ok ? (entry * p.heads + h) * p.page_size + (tok - p.page_of(tok) * p.page_size) : 0;
    };
    look(t0);
    // (columns past the tile's queries repeat its last: nothing reads what they give)
    bf16x8 q[KQ];
    {
        const uint32_t idx = at + (q0 + c < nq ? q0 + c : nq - 1), b = first + idx / a.group;
        const uint16_t* const qh = a.q + b * a.q_stride + (size_t)(h * a.group + idx % a.group) * dim;
#pragma unroll
        for (int s = 0; s < KQ; s++) {
            const uint32_t d = 16 * s + 8 * g;
            u32x4 w = {0u, 0u, 0u, 0u};
            if (d < dim) w = *reinterpret_cast<const bf16x8_any*>(qh + d) ^ a.flip;
            q[s] = __builtin_bit_cast(bf16x8, w);
        }
    }
    // (looked up above by the first row's table, which nearly always has the prefix)
    uint32_t reads;
    if (!row_with(a, x, reads)) return;
    if (reads != first) {
        table = p.table(reads, h);
        look(t0);
    }

    // A step's tiles, each wave 16 tokens: bf16 straight to LDS (a load's 64 pieces lie there
    // one after the other, so each lane fetches what belongs in its place), int8 through
    // registers, as bf16.
    constexpr int OF_LOAD = 64 / CH, LOADS = 16 / OF_LOAD;       // tokens of a wave's load, loads of 16 tokens
    const int in_load = lane / CH, piece = lane % CH;
    u32x4 kc[I8 ? LOADS : 1], vc[I8 ? LOADS : 1];
    float ksc = 0.0f, vsc = 0.0f;
    const __amdgpu_buffer_rsrc_t rk = rsrc(p.k), rv = rsrc(p.v);
    const int tok0 = 16 * wave;
    auto load = [&](uint8_t* kt, uint8_t* vt) {
#pragma unroll
        for (int i = 0; i < LOADS; i++) {
            const int tok = tok0 + i * OF_LOAD + in_load;
            const uint32_t r = __shfl(row, tok);
            if (I8) {
                const size_t x = (size_t)r * row_bytes + (16 * piece < (int)row_bytes ? 16 * piece : 0);
                kc[i] = *reinterpret_cast<const u32x4*>(p.k + x);
                vc[i] = *reinterpret_cast<const u32x4*>(p.v + x);
                continue;
            }
            const uint32_t kp = 16 * L::key_piece(tok, piece), vp = 16 * L::value_piece(tok, piece);
            const lds_t kto = (lds_t)(kt + i * OF_LOAD * L::RB), vto = (lds_t)(vt + i * OF_LOAD * L::RB);
            if (FORM == FAR) {
                const size_t x = (size_t)r * row_bytes;
                if (kp < row_bytes) __builtin_amdgcn_global_load_lds((const glb_t)(p.k + x + kp), kto, 16, 0, 0);
                if (vp < row_bytes) __builtin_amdgcn_global_load_lds((const glb_t)(p.v + x + vp), vto, 16, 0, 0);
            } else {
                const uint32_t x = r * row_bytes;
                __builtin_amdgcn_raw_ptr_buffer_load_lds(rk, kto, 16, x + kp, 0, 0, 0);
                __builtin_amdgcn_raw_ptr_buffer_load_lds(rv, vto, 16, x + vp, 0, 0, 0);
            }
        }
        if (I8 && wave == 0) {
            ksc = p.ks[row];
            vsc = p.vs[row];
        }
    };
    // then: values of absent tokens as zeros (0 * NaN), and int8 rows to LDS
    auto settle = [&](uint8_t* kt, uint8_t* vt, float* sc, uint64_t there) {
        if (I8) {
#pragma unroll
            for (int i = 0; i < LOADS; i++) {
                const int tok = tok0 + i * OF_LOAD + in_load, to = (i * OF_LOAD + in_load) * L::RB;
                const bool in = 16 * piece < (int)row_bytes;
                if (!in) kc[i] = u32x4{0u, 0u, 0u, 0u};
                if (!in || !(there >> tok & 1)) vc[i] = u32x4{0u, 0u, 0u, 0u};
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    *reinterpret_cast<u32x4*>(kt + to + 16 * L::key_piece(tok, 2 * piece + j)) =
                        bytes_to_bf16(kc[i][2 * j], kc[i][2 * j + 1]);
                    *reinterpret_cast<u32x4*>(vt + to + 16 * L::value_piece(tok, 2 * piece + j)) =
                        bytes_to_bf16(vc[i][2 * j], vc[i][2 * j + 1]);
                }
            }
            if (wave == 0) {
                sc[lane] = ksc;
                sc[STEP + lane] = there >> lane & 1 ? vsc : 0.0f;
            }
        } else if (there != ~0ull) {
#pragma unroll
            for (int i = 0; i < LOADS; i++)
                if (!(there >> (tok0 + i * OF_LOAD + in_load) & 1))
                    *reinterpret_cast<u32x4*>(vt + (i * OF_LOAD + in_load) * L::RB + 16 * piece) = u32x4{0u, 0u, 0u, 0u};
        }
    };

    f32x16 o[DT] = {};
    float m = -INFINITY, sum = 0.0f;
    bool any = false;
    // N x 32 tokens, whose rows and scales lie at kt, vt, kscales and vscales
    auto attend = [&](auto n_, const uint8_t* kt, const uint8_t* vt, const float* kscales, const float* vscales, uint64_t there) {
        constexpr int N = decltype(n_)::value;
        f32x16 s[N] = {};
        // (reads ahead of the products: one after the other they would wait for each)
        constexpr int AHEAD = DP <= 64 ? KQ : I8 ? (DP <= 128 ? KQ / 2 : 2) : DP <= 128 ? KQ : 4;
#pragma unroll
        for (int i0 = 0; i0 < KQ; i0 += AHEAD) {
            bf16x8 kf[AHEAD][N];
#pragma unroll
            for (int i = 0; i < AHEAD; i++)
#pragma unroll
                for (int u = 0; u < N; u++)
                    kf[i][u] = *reinterpret_cast<const bf16x8*>(kt + (32 * u + c) * L::RB + 16 * L::key_piece(c, 2 * (i0 + i) + g));
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < AHEAD; i++)
#pragma unroll
                for (int u = 0; u < N; u++) s[u] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[i][u], q[i0 + i], s[u], 0, 0, 0);
            __builtin_amdgcn_sched_barrier(0);
        }
        float top = -INFINITY;
#pragma unroll
        for (int u = 0; u < N; u++) {
            if (I8)
#pragma unroll
                for (int r = 0; r < 16; r += 4) {
                    const f32x4 k4 = *reinterpret_cast<const f32x4*>(kscales + 32 * u + 2 * r + 4 * g);
#pragma unroll
                    for (int i = 0; i < 4; i++) s[u][r + i] *= k4[i];
                }
            const uint32_t mask = (uint32_t)(there >> (32 * u));
            any |= mask != 0;
            if (mask != 0xFFFFFFFFu)
#pragma unroll
                for (int r = 0; r < 16; r++)
                    if (!(mask >> (2 * (r & 12) + (r & 3) + 4 * g) & 1)) s[u][r] = -INFINITY;
#pragma unroll
            for (int r = 0; r < 16; r++) top = fmaxf(top, s[u][r]);
        }
        float other;
        top = swap32(top, other);
        top = fmaxf(top, other) * a.scale_log2;
        // Weights are 2^(logit - m).  The reference m is a whole number, so that changing
        // it rounds nothing, and moves when a logit comes within `lift` of it: after the
        // first steps hardly ever.  It is so far above that weights sum up to 1 at most,
        // however many there are: no sum of weighted values passes the largest value, and
        // results are finite if that is.
        if (__any(top + a.lift > m)) {
            const float to = fmaxf(m, __builtin_ceilf(top) + a.room);
            const float f = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - to);
            m = to;
            sum *= f;
#pragma unroll
            for (int i = 0; i < DT; i++) o[i] *= f;
        }
        const float ref = m == -INFINITY ? 0.0f : m;
        // 16 tokens at a time: the next ones' weights and values while these are multiplied
        bf16x8 pc[2][3], vf[2][DT];
        auto weigh = [&](int k) {
            float e[8];
#pragma unroll
            for (int r = 0; r < 8; r++) {
                e[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[k >> 1][8 * (k & 1) + r], a.scale_log2, -ref));
                sum += e[r];
            }
            if (I8)
#pragma unroll
                for (int r = 0; r < 8; r += 4) {
                    const f32x4 v4 = *reinterpret_cast<const f32x4*>(vscales + 16 * k + 2 * r + 4 * g);
#pragma unroll
                    for (int i = 0; i < 4; i++) e[r + i] *= v4[i];
                }
            split3<I8>(e, pc[k & 1]);
        };
        auto values = [&](int k) {
#pragma unroll
            for (int dt = 0; dt < DT; dt++) {
                s16x4 w[2];
#pragma unroll
                for (int t = 0; t < 2; t++) {
                    const int tok = 16 * k + 8 * t + 4 * g + ((lane & 15) >> 2);
                    const int piece = 4 * dt + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
                    const lds_t at = (lds_t)(vt + tok * L::RB + 16 * L::value_piece(tok, piece) + 8 * (lane & 1));
                    w[t] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)at);
                }
                vf[k & 1][dt] = __builtin_bit_cast(bf16x8, __builtin_shufflevector(w[0], w[1], 0, 1, 2, 3, 4, 5, 6, 7));
            }
        };
        values(0);
        weigh(0);
#pragma unroll
        for (int k = 0; k < 2 * N; k++) {
            __builtin_amdgcn_sched_barrier(0);
            if (k + 1 < 2 * N) {
                values(k + 1);
                weigh(k + 1);
            }
#pragma unroll
            for (int i = 0; i < 3; i++)
#pragma unroll
                for (int dt = 0; dt < DT; dt++)
                    o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[k & 1][dt], pc[k & 1][i], o[dt], 0, 0, 0);
            if (k + 1 < 2 * N) {
                // the reads first, then a few of the weights' instructions behind each product
                __builtin_amdgcn_sched_group_barrier(0x100, 2 * DT, 0);
#pragma unroll
                for (int i = 0; i < 3 * DT; i++) {
                    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                    __builtin_amdgcn_sched_group_barrier(0x402, 8, 0);
                }
            }
        }
        __builtin_amdgcn_sched_barrier(0);
    };

    if (FORM == FAR && row_bytes < L::RB) {      // what loads do not reach: zeros behind the head's end
        for (int i = 16 * tid; i < 2 * L::BUF; i += 16 * 256) *reinterpret_cast<u32x4*>(lds + i) = u32x4{0u, 0u, 0u, 0u};
        __syncthreads();
    }
    find(t0);
    look(t0 + STEP);
    {
        auto steps = [&](auto n, int u0) {
            auto tile = [&](int buf) { return lds + buf * L::BUF + tok0 * L::RB; };
            load(tile(0), tile(0) + L::T);
            int buf = 0;
            for (uint32_t base = t0; base < t1; base += STEP, buf ^= 1) {
                const uint64_t there = __ballot(ok);
                __builtin_amdgcn_s_waitcnt(0x0070);  // this wave's part of the step is there; its reads of the one before are done
                settle(tile(buf), tile(buf) + L::T, scales + 2 * buf * STEP, there);
                __syncthreads();
                if (base + STEP < t1) {
                    find(base + STEP);
                    look(base + 2 * STEP);
                    load(tile(buf ^ 1), tile(buf ^ 1) + L::T);
                }
                const uint8_t* const kt = lds + buf * L::BUF + u0 * 32 * L::RB;
                const float* const sc = scales + 2 * buf * STEP + 32 * u0;
                if (busy) attend(n, kt, kt + L::T, sc, sc + STEP, there >> (32 * u0));
            }
        };
        if (wide) steps(std::integral_constant<int, 2>{}, 0);
        else steps(std::integral_constant<int, 1>{}, wave >> 1);
        __syncthreads();
    }

    // a maximum of -inf with tokens there is told from no tokens by a sum of 1
    {
        float other;
        sum = swap32(sum, other);
        sum += other;
    }
    if (m == -INFINITY && any && sum == 0.0f) sum = 1.0f;
    // waves of the same queries meet
    if (!wide) {
        float* const ow = reinterpret_cast<float*>(lds) + (wave & 1) * 32 * L::OS + c * L::OS;
        if (wave >= 2) {
            if (g == 0) ends[32 * (wave & 1) + c] = make_float2(m, sum);
#pragma unroll
            for (int dt = 0; dt < DT; dt++)
#pragma unroll
                for (int r = 0; r < 16; r += 4)
                    *reinterpret_cast<f32x4*>(ow + 32 * dt + 2 * r + 4 * g) = f32x4{o[dt][r], o[dt][r + 1], o[dt][r + 2], o[dt][r + 3]};
        }
        __syncthreads();
        if (wave >= 2) return;
        const float2 e = ends[32 * (wave & 1) + c];
        const float top = fmaxf(m, e.x);
        const float f0 = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - top);
        const float f1 = e.x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(e.x - top);
        // (without a finite logit in either: 0, 1 or NaN each, of which the sum keeps what the
        // join asks for, no tokens, tokens, and NaN)
        sum = top == -INFINITY ? sum + e.y : f0 * sum + f1 * e.y;
        m = top;
#pragma unroll
        for (int dt = 0; dt < DT; dt++)
#pragma unroll
            for (int r = 0; r < 16; r += 4) {
                const f32x4 x = *reinterpret_cast<const f32x4*>(ow + 32 * dt + 2 * r + 4 * g);
#pragma unroll
                for (int i = 0; i < 4; i++) o[dt][r + i] = f0 * o[dt][r + i] + f1 * x[i];
            }
    }
    if (q0 + c >= nq) return;
    const size_t place = slot + q0 + c;
    if (g == 0) a.ml[place] = make_float2(m, sum);
    float* const to = a.part + place * dim;
#pragma unroll
    for (int dt = 0; dt < DT; dt++)
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
            const uint32_t d = 32 * dt + 2 * r + 4 * g;
            if (d < dim) *reinterpret_cast<f32x4*>(to + d) = f32x4{o[dt][r], o[dt][r + 1], o[dt][r + 2], o[dt][r + 3]};
        }
}

// W waves for each row and query head: what its prefix's spans and its own tokens' left,
// added in that order by every one for its part of them, and then the waves' sums.  What
// bounds it: groups, maxima and parts one after the other, 4 us; 8192 queries of 9 parts 10.8
// (38 MB).
template <int W>
__global__ void __launch_bounds__(256) k_kv_shared_join(const KVPool p, const Shared a) {
    __shared__ f32x4 sums[W > 1 ? W - 1 : 1][64];
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t number = blockIdx.x * (4 / W) + (W > 1 ? 0 : wave);
    if (number >= a.rows * a.q_heads) return;
    const uint32_t b = number / a.q_heads, hq = number - b * a.q_heads, h = hq / a.group, j = hq - h * a.group;
    uint32_t len = kv_length(a.lengths, b, a.max_length);        // (asked for before what the groups say)
    const Groups groups(a, p.width * p.page_size);
    len = len < groups.most ? len : groups.most;
    Prefix x = {};
    const bool shared = groups.find<true>(b, x) && x.tokens <= len;
    const uint32_t idx = shared ? (b - x.first) * a.group + j : 0;
    const uint32_t unit = shared ? x.base + idx / TILE * x.spans : 0;
    // (spans past the workspace: of groups that overlap)
    const uint32_t spans = !shared || unit >= a.blocks ? 0 : x.spans < a.blocks - unit ? x.spans : a.blocks - unit;
    const size_t from = ((size_t)h * a.blocks + unit) * a.columns + idx % TILE;
    const size_t own = ((((size_t)b * p.heads + h) * a.own_tiles + j / 16) * a.splits) * a.own_columns + j % 16;
    const uint32_t begins = shared ? x.tokens : 0;
    const uint32_t splits = len - begins > a.own_span ? (len - begins + a.own_span - 1) / a.own_span : 1;
    const uint32_t n = spans + (splits < a.splits ? splits : a.splits);
    auto place = [&](uint32_t i) { return i < spans ? from + (size_t)i * a.columns : own + (size_t)(i - spans) * a.own_columns; };
    auto end = [&](uint32_t i) { return i >= n ? make_float2(-INFINITY, 0.0f) : i < spans ? a.ml[place(i)] : a.own_ml[place(i)]; };

    const uint32_t span = p.dim <= 64 ? 16 : p.dim <= 128 ? 32 : 64, ways = 64 / span * W;
    const uint32_t d = 4 * (lane & (span - 1)), way = (W > 1 ? wave * (64 / span) : 0) + lane / span;
    const bool in = d < p.dim;
    constexpr int U = 8;              // loads in flight
    f32x4 part[U];
    auto fetch = [&](uint32_t i0, uint32_t k0, uint32_t here) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            const uint32_t k = k0 + u * ways + way, i = i0 + (k < here ? k : here - 1);
            part[u] = *reinterpret_cast<const f32x4*>((i < spans ? a.part : a.own_part) + place(i) * p.dim + (in ? d : 0));
        }
    };
    // (the first values on their way along with the maxima)
    float2 e = end(lane);
    fetch(0, 0, n < 64 ? n : 64);
    float top = e.x;
    for (uint32_t i = lane + 64; i < n; i += 64) top = fmaxf(top, end(i).x);
    top = lane_max(top);
    f32x4 v = {};
    float total = 0.0f, plain = 0.0f;
    for (uint32_t i0 = 0; i0 < n; i0 += 64) {
        if (i0) e = end(i0 + lane);
        const float f = e.x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(e.x - top);
        total += f * e.y;
        plain += e.y;
        const uint32_t here = n - i0 < 64 ? n - i0 : 64;
        for (uint32_t k0 = 0; k0 < here; k0 += U * ways) {
            if (i0 + k0) fetch(i0, k0, here);
#pragma unroll
            for (int u = 0; u < U; u++) {
                const uint32_t k = k0 + u * ways + way;
                const float w = __shfl(f, k & 63);
                if (k < here && w != 0.0f) v += w * part[u];
            }
        }
    }
    total = lane_sum(total);
    plain = lane_sum(plain);
    for (uint32_t o = span; o < 64; o <<= 1)
#pragma unroll
        for (int k = 0; k < 4; k++) v[k] += __shfl_xor(v[k], o);
    if (W > 1) {
        if (wave) sums[wave - 1][lane] = v;
        __syncthreads();
        if (wave) return;
#pragma unroll
        for (int w = 1; w < W; w++) v += sums[w - 1][lane];
    }
    if (way || !in) return;
    v *= top == -INFINITY ? plain == 0.0f ? 0.0f : NAN : 1.0f / total;
    const size_t to = b * a.out_stride + (size_t)hq * p.dim + d;
    if (a.out_f32) *reinterpret_cast<f32x4_any*>(static_cast<float*>(a.out) + to) = v;
    else *reinterpret_cast<bf16x4_any*>(static_cast<uint16_t*>(a.out) + to) = u32x2{bf16x2_out(v[0], v[1]), bf16x2_out(v[2], v[3])};
}

template <int DIM, Form FORM>
int launch(unsigned grid, const KVPool& p, const Shared& a, hipStream_t s) {
    static std::atomic<uint64_t> done{0};
    constexpr int LDS = Tiles<DIM <= 64 ? 64 : DIM <= 128 ? 128 : 256>::ALL;
    const auto fn = k_kv_shared<DIM, FORM>;
    if (LDS > 65536 && lds_optin(reinterpret_cast<const void*>(fn), LDS, done) != hipSuccess) {
        snx_set_error("kv_attention_shared: no %d bytes of LDS", LDS);
        return -1;
    }
    fn<<<grid, 256, LDS, s>>>(p, a);
    return snx_launch_check("k_kv_shared");
}
template <int DIM>
int launch(unsigned grid, bool i8, const KVPool& p, const Shared& a, hipStream_t s) {
    if (i8) return launch<DIM, INT8>(grid, p, a, s);
    // (loads to LDS by 32-bit offsets count apart from LDS reads, those by address do not:
    // 64 rows behind 4096 tokens 32.1 us and 36.7)
    if constexpr (DIM != 96)
        if (p.dim == DIM && (uint64_t)p.pages * p.heads * p.page_size * DIM * 2 <= 0xFFFFFFFFull)
            return launch<DIM, NEAR>(grid, p, a, s);
    return launch<DIM, FAR>(grid, p, a, s);
}
int launch(unsigned grid, bool i8, const KVPool& p, const Shared& a, hipStream_t s) {
    if (p.dim <= 64) return launch<64>(grid, i8, p, a, s);
    if (p.dim <= 96) return launch<96>(grid, i8, p, a, s);
    if (p.dim <= 128) return launch<128>(grid, i8, p, a, s);
    return launch<256>(grid, i8, p, a, s);
}

size_t round16(size_t n) { return (n + 15) / 16 * 16; }

}  // namespace

extern "C" {

int snx_k_kv_attention_shared(const SNEPPXKVCache* c, const uint16_t* q, size_t q_stride, void* out, size_t out_stride,
                              int out_f32, const int32_t* tables, size_t width, const int32_t* lengths, size_t rows,
                              size_t q_heads, size_t max_length, const int32_t* group_starts,
                              const int32_t* prefix_lengths, size_t groups, size_t max_prefix, size_t max_own,
                              float scale, void* st) {
    const KVPool p = kv_pool(c, tables, width);
    const size_t group = q_heads / c->kv_heads;
    const size_t tiles = groups ? rows * group / TILE + groups : 0;      // of a head, at most
    const size_t prefix_steps = groups ? (max_prefix + STEP - 1) / STEP : 0;
    const size_t own_tiles = (group + 15) / 16;
    const size_t places = (size_t)(c->head_dim <= 128 ? 2 : 1) * cu_count();      // of workgroups that run at once
    // Own tokens by about 1024 waves, which all run at once (64 rows behind 4096 tokens with up
    // to 512 of their own 32.1 us so, by 2048 35.4).
    size_t own_span = rows * c->kv_heads * own_tiles * max_own / 1024 / 32 * 32;
    if (own_span < 64) own_span = 64;
    size_t splits = (max_own + own_span - 1) / own_span;
    if (splits < 1) splits = 1;
    // A prefix of up to ten steps a step to each workgroup, of twice that two, of more three:
    // a span's steps follow one another, but all of them are joined (20 rows behind 500
    // tokens 15.3 with spans of three, 13.4 of one; five prefixes of up to 8192 17.6 and 19.4).
    // Steps of heads beyond 128 are twice as long: one of up to 40, else two (2 rows and one
    // key-value head behind 2217 tokens 19.4 with three, 17.7 so; behind 5052 21.0 and 17.4).
    const bool large = c->head_dim > 128;
    size_t least = large ? (prefix_steps + 39) / 40 : (prefix_steps + 9) / 10;
    const size_t most_least = large ? 2 : kLeast;
    least = least < 1 ? 1 : least < most_least ? least : most_least;
    // As many spans of a prefix as make the launch shortest, by a count of what runs one after
    // the other in the CUs' places, in steps (3 us): units of `per` steps and one to begin
    // with, rows' own tokens 40 to a step, in places that units leave free or behind them,
    // and parts, written and read again, at 4.4 TB/s.  (These numbers were chosen among others
    // by timing fifteen calls of 4 to 256 rows.)  Against as many units as places, shared out by the two kinds' work: 112 rows behind 4125 tokens,
    // heads of 256, 77 to 68 us, 64 behind 8192 83 to 61, 32 of 128 behind 2048 with up to
    // 1024 of their own 29.2 to 27.4; what it loses: 20 prefixes of 5 rows 29.8 to 31.0, 64
    // rows behind 4096 31.7 to 32.5.
    const size_t few = groups ? (rows * group + TILE - 1) / TILE : 0;    // tiles of groups that fill them
    const size_t about_tiles = few > groups ? few : groups;
    const size_t own_wgs = (rows * c->kv_heads * own_tiles * splits + 3) / 4;
    const float own_time = max_own ? (float)(own_span < max_own ? own_span : max_own) / 40.0f + 1.0f : 0.0f;
    const float per_place = 1.0f / (float)places;
    auto rounds = [&](size_t wgs) { return __builtin_ceilf((float)wgs * per_place); };
    size_t about = 1;
    float best = FLT_MAX;
    for (size_t per = prefix_steps; per >= least;) {
        const size_t spans = (prefix_steps + per - 1) / per, units = about_tiles * spans * c->kv_heads;
        if (spans > 1 && (units > 4 * places || spans > 128)) break;
        const float unit_time = (float)per + 1.0f, all = rounds(units);
        const float free = all * (float)places - (float)units;       // places of the last round
        float left = (float)own_wgs;
        if (own_time > 0.0f) left -= free * __builtin_floorf(unit_time / own_time);
        const float parts = (float)(rows * q_heads * spans) * (float)c->head_dim * 6e-7f;
        const float time = all * unit_time + (left > 0.0f ? rounds((size_t)left) * own_time : 0.0f) + parts;
        if (time < best) {
            best = time;
            about = about_tiles * spans;
        }
        const size_t next = (prefix_steps + spans) / (spans + 1);        // of one span more
        per = next < per ? next : per - 1;
    }
    const size_t blocks = groups ? about + tiles : 0;
    const size_t columns = rows * group < TILE ? rows * group : TILE, own_columns = group < 16 ? group : 16;
    const size_t slots = blocks * c->kv_heads * columns, own = rows * c->kv_heads * own_tiles * splits * own_columns;
    const size_t grid = blocks * c->kv_heads + (rows * c->kv_heads * own_tiles * splits + 3) / 4;
    // (a grid has below 2^32 threads; steps of all tiles are counted in 32 bits)
    if (grid > 0xffffff || rows * q_heads / 4 > 0xfffffe || tiles * ((max_length + STEP - 1) / STEP) > 0x7fffffff) {
        snx_set_error("kv_attention_shared: %zu rows of up to %zu tokens are too many", rows, max_length);
        return -1;
    }
    const size_t b0 = round16(slots * c->head_dim * sizeof(float)), b1 = round16(own * c->head_dim * sizeof(float));
    const size_t b2 = round16(slots * sizeof(float2)), b3 = round16(own * sizeof(float2));
    uint8_t* ws = static_cast<uint8_t*>(snx_workspace(b0 + b1 + b2 + b3, SLOT_KV_SHARED, st));
    if (!ws) return -1;
    Shared a;
    a.q = q;
    a.out = out;
    a.q_stride = q_stride;
    a.out_stride = out_stride;
    a.lengths = lengths;
    a.starts = group_starts;
    a.prefix = prefix_lengths;
    a.part = reinterpret_cast<float*>(ws);
    a.own_part = reinterpret_cast<float*>(ws + b0);
    a.ml = reinterpret_cast<float2*>(ws + b0 + b1);
    a.own_ml = reinterpret_cast<float2*>(ws + b0 + b1 + b2);
    a.rows = (uint32_t)rows;
    a.q_heads = (uint32_t)q_heads;
    a.group = (uint32_t)group;
    a.groups = (uint32_t)groups;
    a.max_length = (uint32_t)max_length;
    a.about = (uint32_t)about;
    a.blocks = (uint32_t)blocks;
    a.least = (uint32_t)least;
    a.columns = (uint32_t)columns;
    a.own_columns = (uint32_t)own_columns;
    a.own_tiles = (uint32_t)own_tiles;
    a.splits = (uint32_t)splits;
    a.own_span = (uint32_t)own_span;
    // (a scale of zero must not make NaN of a logit of -inf, which is a token that is not there)
    a.flip = scale < 0.0f ? 0x80008000u : 0u;
    a.scale_log2 = (scale < 0.0f ? -scale : scale) * 1.44269504088896340736f;
    if (a.scale_log2 < FLT_MIN) a.scale_log2 = FLT_MIN;
    uint32_t room = kLag;
    while (((size_t)1 << (room - kLag)) < max_length) room++;
    a.room = (float)room;
    a.lift = (float)(room - kLag);
    a.out_f32 = out_f32;
    const bool i8 = c->dtype == SNEPPX_INT8;
    if (launch((unsigned)grid, i8, p, a, S(st))) return -1;
    // Few rows with much to add up: four waves for each query (48 rows of 4 heads and some 55
    // parts 20.0 to 17.7 us, one of 32 heads and 44 17.0 to 15.9; with up to 17 parts one
    // wave is better, 13.5 to 15.1, and with 2048 queries, 32.2 to 36.5).
    const size_t most = (prefix_steps + least - 1) / least, parts = (few && about / few < most ? about / few : most) + splits;
    if (rows * q_heads <= 1024 && parts > 32) k_kv_shared_join<4><<<(unsigned)(rows * q_heads), 256, 0, S(st)>>>(p, a);
    else k_kv_shared_join<1><<<(unsigned)((rows * q_heads + 3) / 4), 256, 0, S(st)>>>(p, a);
    return snx_launch_check("k_kv_shared_join");
}

}  // extern "C"
