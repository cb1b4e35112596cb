// kv_attn_kernels.hip - attention of one new token per row over the paged
// key-value cache (include/sneppx_kv.h).
//
//   s[t] = scale q . k[t],  p = softmax(s),  out = sum_t p[t] v[t]
//
// for the group of query heads that share a key-value head.  Every key and
// value is used for `group` products only, so reading the cache is what bounds
// it, and the kernel is built around reading it once:
//  * k_kv_attn: the tokens of all rows are cut into equal shares, as many as the
//    CUs hold workgroups; a workgroup takes a share of one key-value head and up
//    to 16 of its query heads.  Its four waves take tiles of 32 tokens in turn,
//    each wave with its own running maximum, sum and output, and meet at the
//    row's end.  Heads are the columns of the matrix cores' tiles (a group of
//    fewer leaves columns empty: 16 rows of 4096 tokens take 52, 53 and 57 us at
//    1, 4 and 16 query heads to a key-value head).
//  * A row in several shares is joined, in the order of its shares, by the last of
//    them to arrive, or by k_kv_join after them, which also adds the attention
//    weights, from the logits that the first kernel wrote.
// Reached: 131072 tokens of 8 heads of 128 in bf16 (537 MB) 97 us, 5.5 TB/s, where a
// copy of 256 MB runs at 5.4; 64 rows of 0 to 8192 in int8 (532 MB) 103 us.  A call
// is about 8 us and what it reads at 5.8 TB/s: the look-ups, the first tile, the
// meeting and the join follow one another.
#include <hip/hip_runtime.h>

#include <cstdint>

#include "codec.h"
#include "kv_pieces.h"
#include "kv_pool.h"
#include "launch.h"
#include "../snx_internal.h"

using namespace snx;

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef int i32x2 __attribute__((ext_vector_type(2)));
// of any alignment that their elements have
typedef u32x4 bf16_load8 __attribute__((aligned(2)));
typedef u32x2 bf16_store4 __attribute__((aligned(2)));
typedef f32x4 f32_store4 __attribute__((aligned(4)));
typedef __attribute__((address_space(3))) uint8_t* lds_t;

hipStream_t S(void* s) { return reinterpret_cast<hipStream_t>(s); }

constexpr int SLOT_KV_ATTN = 7;       // of the stream's workspaces
constexpr int TILE = 32;              // tokens of a wave's step
constexpr int WAVES = 4;
constexpr int kLag = 8;               // log2 of how far a logit may pass the maximum that weights refer to
constexpr int STEP = TILE * WAVES;    // tokens of a workgroup's step

// Waves of a SIMD that the registers allow with heads padded to `dim`: of a tile's
// keys, values, queries and outputs.  (bf16 heads of 128 at three spill some:
// 131072 tokens 138 us, 98 at two.  What is taken spills in the forms for heads that
// are no whole 64 or 128: ten registers in bf16 up to 64, two in int8 up to 64 and 128.)
constexpr int resident(int dim, bool i8) { return dim <= 64 ? 4 : dim <= 128 ? (i8 ? 3 : 2) : i8 ? 2 : 1; }
// Workgroups of a CU that a call is divided among, at most: us at 2 / 3 / 4 for
// 131072 tokens of 128 in bf16 98 / 102 / 104, in int8 59 / 63 / 68, 64 rows of 0
// to 8192 in int8 108 / 111 / 123, 16 rows of 4096 of 64 30 / 33 / 31 (all at the
// residency above).
constexpr int shares_of_cu(int dim, bool i8) { return resident(dim, i8) < 2 ? 1 : 2; }
constexpr int padded(size_t dim) { return dim <= 64 ? 64 : dim <= 128 ? 128 : 256; }

struct Attn {
    const uint16_t* q;
    void* out;
    size_t q_stride, out_stride;
    const int32_t* lengths;
    uint32_t* arrivals;       // [rows * kv_heads * tiles], zero, or NULL: k_kv_join follows
    float* part;              // [2 * shares][kv_heads * tiles][heads][dim]
    float2* ml;               // [2 * shares][kv_heads * tiles][heads]: maximum, sum
    float* logits;            // [rows][q_heads][logit_stride], or NULL
    float2* whole;            // with logits, [rows][q_heads] of rows in one share: maximum, 1 / sum (as Parts::whole)
    uint32_t rows, q_heads, max_length, tiles, heads, logit_stride;
    uint32_t shares, about_shares;    // shares, and what is about as many
    Divider by_eights, by_heads, by_shares;      // by 8 tiles, kv_heads and shares
    float scale_log2;
    float room;               // log2 of the most that a row's weights of up to 2^kLag sum up to
    int out_f32;
};

// ------------------------------------------------------------- the division
// All rows' steps (one at least for each row), one row after the other, are cut
// into equal shares; a workgroup takes one, with the end of a row, whole rows
// and the beginning of another in it, and so all end together.  Where a share is
// one or two steps, or rows need about as many shares if each begins one (up to an
// eighth more of three or four steps, for which CUs of two workgroups even out what
// passes a round, no more of longer ones), changing the row costs more than that
// evens out, and every row begins with a new share.  The lengths are known on the
// device alone, so every wave works this out for itself.  (us of shares across rows
// / by rows, 8 heads of 128 in bf16: 16 rows of 0 to 4096 tokens, 4 steps, 66 shares
// for 64, 32 / 28; 38 of 653, 4 steps, 76 shares, 24 / 33; 64 of 0 to 700, 4 steps,
// 80 shares, 28 / 26; 16 of 2049, 5 steps, 64 shares, 33 / 30; 24 of 0 to 4096, 6
// steps, 74 shares, 46 / 54; 64 of 0 to 8192, 16 steps, 100 / 118; heads of 256, one
// workgroup to a CU: 19 of 653, 4 steps, 38 shares for 32, 27 / 45.  A grid for the
// longest row that the host allows for leaves most of it idle: 45 for the first.)
// Between 66 and 80 shares it is not their number alone that decides: the limit is
// below 76, which by rows loses a third, and so gives away a twentieth at 80.  The
// shares that rows need are counted with one row to a lane, so more than 64 rows of
// three and more steps a share are always cut across, which costs some of them: 64 and
// 65 rows of 4000 tokens and one key-value head 24.9 and 27.4 us, of 1000 and two heads
// 16.0 and 21.3.
struct Row {
    uint32_t b, at, len;           // the row, its first step, its length in tokens
    __device__ __forceinline__ uint32_t steps() const { return len > STEP ? (len + STEP - 1) / STEP : 1; }
};

// Division by a number that only the device knows, in fewer instructions than the
// integer one: the reciprocal is good to 40 bits, and (x + 1/2) / d is at least
// 1 / 2d away from the next whole number, which is 2^-33 of it or more.
struct By {
    uint32_t d;
    double inv;
    __device__ __forceinline__ explicit By(uint32_t by) : d(by) {
        const double y = (double)by, r = __builtin_amdgcn_rcp(y);
        inv = __builtin_fma(r, __builtin_fma(-y, r, 1.0), r);
    }
    __device__ __forceinline__ uint32_t operator()(uint32_t x) const { return (uint32_t)(((double)x + 0.5) * inv); }
};

// the shares that a row's steps lie in, and where each left its result
struct Shares {
    uint32_t first, n, inside;     // inside: the row begins within its first share
    __device__ __forceinline__ Shares(const Row& w, const By& per) {
        first = per(w.at);
        n = per(w.at + w.steps() - 1) - first + 1;
        inside = w.at != first * per.d;
    }
    __device__ __forceinline__ uint32_t slot(uint32_t i) const { return 2 * (first + i) + (i == 0 ? inside : 0); }
};
constexpr uint32_t kMostShares = 256;     // of a row

constexpr uint32_t kFewSteps = 2;         // of a share

struct Division {
    const Attn& a;
    uint32_t len0, total, per;     // length of row `lane`; steps of all rows, of a share
    bool by_row;
    By by;
    __device__ __forceinline__ explicit Division(const Attn& attn) : a(attn), by(1) {
        const uint32_t lane = threadIdx.x & 63;
        uint32_t sum = 0, longest = 0;
        len0 = length(lane);
        for (uint32_t r0 = 0; r0 < a.rows; r0 += 64) {
            const uint32_t n = steps(r0 + lane, r0 ? length(r0 + lane) : len0);
            sum += n;
            longest = n > longest ? n : longest;
        }
        total = __builtin_amdgcn_readlane(lane_prefix(sum), 63);
        per = a.by_shares(total + a.shares - 1);
        if (a.shares > kMostShares - 2) {            // a row has part of its first and last share
            const uint32_t least = (lane_max(longest) + kMostShares - 3) / (kMostShares - 2);
            per = per > least ? per : least;
        }
        by = By(per);
        by_row = per <= kFewSteps;
        if (!by_row && a.rows <= 64) {
            const uint32_t n = last_lane(lane_prefix(by(steps(lane, len0) + per - 1)));
            by_row = n <= (per <= 2 * kFewSteps ? a.about_shares : a.shares);
        }
    }
    __device__ __forceinline__ uint32_t length(uint32_t r) const {
        return r < a.rows ? kv_length(a.lengths, r, a.max_length) : 0;
    }
    __device__ __forceinline__ uint32_t steps(uint32_t r, uint32_t len) const {
        return r < a.rows ? Row{r, 0, len}.steps() : 0;
    }
    // what a row takes of the steps: whole shares by row
    __device__ __forceinline__ uint32_t extent(uint32_t steps) const {
        return by_row ? by(steps + per - 1) * per : steps;
    }
    // the row that step `at` belongs to, or row `b`
    template <bool STEPS>
    __device__ __forceinline__ Row find(uint32_t x) const {
        uint32_t base = 0;
        for (uint32_t r0 = 0;; r0 += 64) {
            const uint32_t r = r0 + (threadIdx.x & 63), len = r0 ? length(r) : len0;
            const uint32_t n = extent(steps(r, len)), upto = lane_prefix(n);
            const uint64_t behind = STEPS ? __ballot(base + upto > x) : __ballot(r == x);
            if (behind) {
                const int lane = __builtin_ctzll(behind);
                return Row{r0 + lane, base + (uint32_t)__builtin_amdgcn_readlane(upto - n, lane),
                           (uint32_t)__builtin_amdgcn_readlane(len, lane)};
            }
            base += __builtin_amdgcn_readlane(upto, 63);
            if (r0 + 64 >= a.rows) return Row{a.rows, base, 0};          // no such step
        }
    }
};

// max / sum over the four lanes that differ in bits 4 and 5
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

// A wave's value tile in LDS: token rows of RB bytes.  The transposed reads take
// 32 bytes (int8: 16) of the same columns from 8 (16) rows at once, the writes
// 16 bytes of 16 rows; the row stride and the order of the rows spread both over
// all banks, and leave every address a lane's own base plus a constant.
template <int DP, bool I8>
struct Lds {
    static constexpr int RB = DP * (I8 ? 1 : 2);                // bytes of a token's row
    static constexpr int STRIDE = RB + (I8 ? 16 : 32);
    static constexpr int UPPER = I8 ? 64 : 16;                  // rows from 16 on lie this much further
    static constexpr int V = TILE * STRIDE + UPPER;             // a wave's value tile
    static constexpr int WAVE = V + (I8 ? 2 * TILE * 4 : 0);    // and its scales
    static constexpr int OS = DP + 4;                           // floats of a head's row at the end
    static constexpr int END = WAVES * 16 * OS * 4;
    static constexpr int ALL = END > WAVES * WAVE ? END : WAVES * WAVE;
    // bf16: tokens 0 - 3, 8 - 11, 4 - 7, 12 - 15 (and so the upper half)
    static __device__ __forceinline__ int row(int tok) {
        const int at = I8 ? tok : (tok & 19) | ((tok >> 1) & 4) | ((tok << 1) & 8);
        return at * STRIDE + (tok >> 4) * UPPER;
    }
};

// ------------------------------------------------------ the chunks' results
// Of each chunk and query head the weighted values, maximum and sum.  They are
// stored past the L2s, which the XCDs do not share, and read so, for the
// workgroup that arrives last may join them within the launch.
constexpr int kSysCoherent = 1 | 16;            // buffer cache policy sc0 sc1

__device__ __forceinline__ __amdgpu_buffer_rsrc_t rsrc(const void* p) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), (short)0, -1, 0x00020000);
}

struct Parts {
    const Attn& a;
    __amdgpu_buffer_rsrc_t part, ml;
    uint32_t dim, units, unit;     // unit: key-value head and tile of 16 query heads
    __device__ __forceinline__ Parts(const Attn& attn, uint32_t d, uint32_t n, uint32_t u)
        : a(attn), part(rsrc(attn.part)), ml(rsrc(attn.ml)), dim(d), units(n), unit(u) {}
    __device__ __forceinline__ uint32_t at(uint32_t slot, uint32_t head) const { return (slot * units + unit) * a.heads + head; }
    __device__ __forceinline__ void put(uint32_t slot, uint32_t head, uint32_t d, f32x4 v) const {
        const u32x4 x = __builtin_bit_cast(u32x4, v);
        __builtin_amdgcn_raw_buffer_store_b128(x, part, (at(slot, head) * dim + d) * 4, 0, kSysCoherent);
    }
    __device__ __forceinline__ void put_ml(uint32_t slot, uint32_t head, float m, float l) const {
        __builtin_amdgcn_raw_buffer_store_b64(u32x2{f2u(m), f2u(l)}, ml, at(slot, head) * 8, 0, kSysCoherent);
    }
    __device__ __forceinline__ f32x4 get(uint32_t off) const {
        return __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(part, off, 0, kSysCoherent));
    }
    __device__ __forceinline__ float2 get_ml(uint32_t off) const {
        const u32x2 r = __builtin_amdgcn_raw_buffer_load_b64(ml, off, 0, kSysCoherent);
        return make_float2(u2f(r[0]), u2f(r[1]));
    }

    // maxima and sums of a query head in its row's shares, one per lane and 64
    struct Ends {
        float2 e[kMostShares / 64];
    };
    __device__ __forceinline__ Ends ends(const Shares& w, uint32_t head) const {
        const uint32_t lane = threadIdx.x & 63, slots = units * a.heads * 8, from = at(2 * w.first, head) * 8;
        Ends x;
#pragma unroll
        for (int j = 0; j < (int)kMostShares / 64; j++) {
            x.e[j] = make_float2(-INFINITY, 0.0f);
            if (64 * j < (int)w.n && 64 * j + lane < w.n) x.e[j] = get_ml(from + (64 * j + lane ? 2 * (64 * j + lane) : w.inside) * slots);
        }
        return x;
    }
    // Their maximum and 1 / sum (of weights of 2^-room), by one wave: 0 for no tokens, NaN where there are
    // tokens and every logit is -inf; to `factors` each share's weight.
    __device__ __forceinline__ float2 whole(const Ends& x, const Shares& w, float* factors) const {
        const uint32_t lane = threadIdx.x & 63;
        float top = -INFINITY, total = 0.0f, plain = 0.0f;
#pragma unroll
        for (int j = 0; j < (int)kMostShares / 64; j++) top = fmaxf(top, x.e[j].x);
        top = lane_max(top);
#pragma unroll
        for (int j = 0; j < (int)kMostShares / 64; j++) {
            if (64 * j >= (int)w.n) continue;
            const float f = x.e[j].x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(x.e[j].x - top);
            total += f * x.e[j].y;
            plain += x.e[j].y;
            if (factors) factors[64 * j + lane] = f;
        }
        total = lane_sum(total);
        plain = lane_sum(plain);
        return make_float2(top, top == -INFINITY ? plain == 0.0f ? 0.0f : NAN : 1.0f / total);
    }

    // One wave joins a row's shares of a query head and writes the result: 4
    // elements per lane, the shares in 64 / span turns, added in a fixed order.
    // factors: LDS of the wave, kMostShares floats.
    __device__ __forceinline__ void join(const Shares& w, uint32_t b, uint32_t head, uint32_t hq, float* factors) const {
        constexpr int U = 8;              // loads in flight
        const uint32_t lane = threadIdx.x & 63;
        const uint32_t span = dim <= 64 ? 16 : dim <= 128 ? 32 : 64, ways = 64 / span;
        const uint32_t d = 4 * (lane & (span - 1)), way = lane / span;
        const bool in = d < dim;
        const uint32_t slots = units * a.heads * dim * 4, from = (at(2 * w.first, head) * dim + (in ? d : 0)) * 4;
        const Ends e = ends(w, head);
        f32x4 v = {};
        float2 st = {};
        for (uint32_t i0 = way; i0 < way + (w.n + ways - 1) / ways * ways; i0 += U * ways) {
            f32x4 x[U];
#pragma unroll
            for (int u = 0; u < U; u++) {
                const uint32_t i = i0 + u * ways < w.n ? i0 + u * ways : w.n - 1;     // (not 0: n > 1)
                x[u] = get(from + (u == 0 && i == 0 ? w.inside : 2 * i) * slots);
            }
            if (i0 == way) {
                st = whole(e, w, factors);
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                __builtin_amdgcn_wave_barrier();
            }
#pragma unroll
            for (int u = 0; u < U; u++)
                if (i0 + u * ways < w.n) v += factors[i0 + u * ways] * x[u];
        }
        for (uint32_t o = span; o < 64; o <<= 1)
#pragma unroll
            for (int j = 0; j < 4; j++) v[j] += __shfl_xor(v[j], o);
        if (way == 0 && in) store(b, hq, d, v, st.y);
    }

    __device__ __forceinline__ void store(uint32_t b, uint32_t hq, uint32_t d, f32x4 v, float inv) const {
        const size_t to = b * a.out_stride + (size_t)hq * dim + d;
        v *= inv;
        if (a.out_f32) {
            *reinterpret_cast<f32_store4*>(static_cast<float*>(a.out) + to) = v;
        } else {
            *reinterpret_cast<bf16_store4*>(static_cast<uint16_t*>(a.out) + to) =
                u32x2{bf16x2_out(v[0], v[1]), bf16x2_out(v[2], v[3])};
        }
    }
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
template <int DP, bool I8, bool SAVE, bool FULL>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(resident(DP, I8))))
k_kv_attn(const KVPool p, const Attn a) {
    typedef Lds<DP, I8> L;
    constexpr int NC = L::RB / 64;        // 16-byte chunks of a row per lane
    constexpr int KS = DP / 32;           // products along the head
    constexpr int DT = DP / 16;           // tiles of 16 output elements
    __shared__ __attribute__((aligned(16))) uint8_t lds[L::ALL];
    __shared__ float2 ends[WAVES][16];
    __shared__ uint32_t arrived;

    ask_for(p.tables, p.heads, a.rows, a.scale_log2);
    // The heads of a share, then the next share: workgroups go to the XCDs in turn,
    // and so every XCD gets shares of all rows.  The tiles of one head and share
    // are 8 workgroups apart, on one XCD, whose L2 has their tokens then (16 rows of
    // 4096, 32 query heads to a key-value head: 88 us side by side, 73 so).
    const uint32_t units = p.heads * a.tiles, eights = a.by_eights(blockIdx.x), rest = blockIdx.x - eights * 8 * a.tiles;
    const uint32_t ht = rest / 8, pair = eights * 8 + rest % 8, number = a.by_heads(pair), h = pair - number * p.heads;
    const uint32_t unit = h * a.tiles + ht;
    const Division cut(a);
    if ((uint64_t)number * cut.per >= (cut.by_row ? 0xFFFFFFFFu : cut.total)) return;
    uint32_t at = number * cut.per;
    Row w = cut.find<true>(at);
    if (w.b == a.rows) return;
    const uint32_t row_end = w.at + w.steps(), share_end = at + cut.per;
    const uint32_t most = cut.by_row ? row_end : cut.total, stop = share_end < most ? share_end : most;
    const Parts parts(a, FULL ? DP : p.dim, units, unit);

    for (;;) {
        // (opaque, so that what follows from it is not kept in registers from row to row)
        int tid = threadIdx.x;
        asm volatile("" : "+v"(tid));
        const int lane = tid & 63, r = lane & 15, g = lane >> 4;
        const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
        const uint32_t group = a.q_heads / p.heads;
        const uint32_t nh = group - ht * 16 < 16 ? group - ht * 16 : 16;
        const uint32_t hq = h * group + ht * 16;             // the first of the tile's query heads
        const uint32_t dim = FULL ? DP : p.dim, row_bytes = dim * (I8 ? 1 : 2);
        uint8_t* const vt = lds + wave * L::WAVE;
        float* const sc = reinterpret_cast<float*>(vt + L::V);

        const uint32_t b = w.b, ends_at = w.at + w.steps() < stop ? w.at + w.steps() : stop;
        const uint32_t first = (at - w.at) * STEP, upto = (ends_at - w.at) * STEP, last = upto < w.len ? upto : w.len;
        const Shares shares(w, cut.by);
        const uint32_t next_len = ends_at < stop ? cut.length(b + 1) : 0;

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
                entry[t] = tok < last ? (uint32_t)p.table(b, h)[p.page_of(tok)] : 0xFFFFFFFFu;
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
            return *reinterpret_cast<const u32x4*>(pool + (size_t)row[t] * row_bytes + (FULL || c < row_bytes ? c : 0));
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
        if (base < last) look(base);
        // (columns past the tile's heads repeat its last: nothing reads what they give)
        const uint16_t* const qh = a.q + b * a.q_stride + (size_t)(hq + ((uint32_t)r < nh ? r : nh - 1)) * dim;
        bf16x8 q[KS];
#pragma unroll
        for (int s = 0; s < KS; s++) {
            const uint32_t d = I8 ? 16 * (g + 4 * (s >> 1)) + 8 * (s & 1) : 8 * (g + 4 * s);
            u32x4 w = *reinterpret_cast<const bf16_load8*>(qh + (FULL || d < dim ? d : 0));
            if (!FULL && d >= dim) w = u32x4{0u, 0u, 0u, 0u};
            q[s] = __builtin_bit_cast(bf16x8, w);
        }

        if (base < last) {
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
                    u32x4 w = kc[t][I8 ? i >> 1 : i];
                    // (or the compiler converts when it loads, and keeps twice the registers)
                    if (I8) asm volatile("" : "+v"(w));
                    bf16x8 kf;
                    if (I8) kf = __builtin_bit_cast(bf16x8, (i & 1) ? bytes_to_bf16(w[2], w[3]) : bytes_to_bf16(w[0], w[1]));
                    else kf = __builtin_bit_cast(bf16x8, w);
                    // past the head's end the lane has other elements, maybe NaN
                    if (!FULL && (I8 ? 16 * (g + 4 * (i >> 1)) : 8 * (g + 4 * i)) >= (int)dim)
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
            if (!whole) {
#pragma unroll
                for (int t = 0; t < 2; t++)
#pragma unroll
                    for (int i = 0; i < NC; i++)
                        if (!ok[t]) vc[t][i] = u32x4{0u, 0u, 0u, 0u};
                __builtin_amdgcn_sched_barrier(0);       // (a branch, not a select for each register)
            }
#pragma unroll
            for (int t = 0; t < 2; t++) {
                const int tok = 8 * (r >> 2) + 4 * t + (r & 3);
#pragma unroll
                for (int i = 0; i < NC; i++) *reinterpret_cast<u32x4*>(vt + L::row(tok) + 16 * (g + 4 * i)) = vc[t][i];
                if (I8 && g == 0) sc[TILE + tok] = ok[t] ? vsc[t] : 0.0f;
            }
            if (more) load_v();
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();

            // (the phases are kept apart, which keeps registers few)
            __builtin_amdgcn_sched_barrier(0);
            // softmax of the tile's eight logits of this lane's head
            float e[8];
            float top = -INFINITY;
#pragma unroll
            for (int t = 0; t < 2; t++)
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    float v = s[t][j] * a.scale_log2;
                    if (I8) v *= sc[8 * g + 4 * t + j];
                    e[4 * t + j] = v;
                }
            if (!whole) {
#pragma unroll
                for (int i = 0; i < 8; i++)
                    if (!((i < 4 ? t0 : t1) >> (4 * g + (i & 3)) & 1)) e[i] = -INFINITY;
                __builtin_amdgcn_sched_barrier(0);
            }
#pragma unroll
            for (int i = 0; i < 8; i++) top = fmaxf(top, e[i]);
            if (SAVE && (uint32_t)r < nh) {
                float* dst = a.logits + ((size_t)b * a.q_heads + hq + r) * a.logit_stride + base + 8 * g;
                *reinterpret_cast<f32x4*>(dst) = f32x4{e[0], e[1], e[2], e[3]};
                *reinterpret_cast<f32x4*>(dst + 4) = f32x4{e[4], e[5], e[6], e[7]};
            }
            any |= (t0 | t1) != 0;
            top = quad_max(top);
            // The reference point moves only when a logit passes it by kLag: after the
            // first tile hardly ever.  Weights are taken 2^-room of what they are, so
            // that they sum up to 1 at most, however many are 2^kLag: a sum of weighted
            // values is no larger than the largest value then, and finite if that is.
            // (The joins divide by the sum of the same weights.)
            if (__any(top > m + (float)kLag)) {
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
                e[i] = __builtin_amdgcn_exp2f((e[i] - ref) - a.room);
                sum += e[i];
                if (I8) e[i] *= sc[TILE + 8 * g + i];
            }
            bf16x8 pc[3];
            split3<I8>(e, pc);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int dt = 0; dt < DT; dt++) {
                bf16x8 vf;
                if (I8) {
                    const int tok = 8 * g + (r >> 1);
                    const lds_t at = (lds_t)(vt + L::row(tok) + 8 * (r & 1) + 16 * dt);
                    const i32x2 w = __builtin_amdgcn_ds_read_tr8_b64_v2i32((__attribute__((address_space(3))) i32x2*)at);
                    vf = __builtin_bit_cast(bf16x8, bytes_to_bf16((uint32_t)w[0], (uint32_t)w[1]));
                } else {
                    s16x4 w[2];
#pragma unroll
                    for (int t = 0; t < 2; t++) {
                        const int tok = 8 * g + 4 * t + (r >> 2);
                        const lds_t at = (lds_t)(vt + L::row(tok) + 8 * (r & 3) + 32 * dt);
                        w[t] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)at);
                    }
                    vf = __builtin_bit_cast(bf16x8, __builtin_shufflevector(w[0], w[1], 0, 1, 2, 3, 4, 5, 6, 7));
                }
#pragma unroll
                for (int i = 0; i < 3; i++) o[dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pc[i], o[dt], 0, 0, 0);
                if (dt % 2 == 1) __builtin_amdgcn_sched_barrier(0);
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
        const uint32_t quads = dim / 4;
        for (uint32_t i = tid; i < nh * quads; i += 256) {
            const uint32_t hd = i / quads, d = 4 * (i - hd * quads);
            float top = -INFINITY, total = 0.0f, plain = 0.0f;
#pragma unroll
            for (int w = 0; w < WAVES; w++) top = fmaxf(top, ends[w][hd].x);
            f32x4 v = {};
#pragma unroll
            for (int w = 0; w < WAVES; w++) {
                const float2 e = ends[w][hd];
                const float f = e.x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(e.x - top);
                total += f * e.y;
                plain += e.y;
                v += f * *reinterpret_cast<const f32x4*>(reinterpret_cast<float*>(lds) + (w * 16 + hd) * L::OS + d);
            }
            if (top == -INFINITY) total = plain > 1.0f ? 1.0f : plain;
            if (shares.n == 1) {
                const float inv = top == -INFINITY ? total == 0.0f ? 0.0f : NAN : 1.0f / total;
                parts.store(b, hq + hd, d, v, inv);
                if (SAVE && d == 0) a.whole[(size_t)b * a.q_heads + hq + hd] = make_float2(top, inv);
            } else {
                const uint32_t slot = 2 * number + (at != number * cut.per);
                parts.put(slot, hd, d, v);
                if (d == 0) parts.put_ml(slot, hd, top, total);
            }
        }
        if (!SAVE && shares.n > 1 && a.arrivals) {
            // the last of the row's shares to arrive joins them
            __builtin_amdgcn_s_waitcnt(0x0f70);              // vmcnt(0): this wave's stores are out
            __syncthreads();
            if (tid == 0) {
                uint32_t* const mine = a.arrivals + (size_t)b * units + unit;
                const uint32_t c = atomicAdd(mine, 1u);
                if (c == shares.n - 1) atomicExch(mine, 0u);      // ready for the next call
                arrived = c;
            }
            __syncthreads();
            if (arrived == shares.n - 1)
                for (uint32_t j = wave; j < nh; j += WAVES)
                    parts.join(shares, b, j, hq + j, reinterpret_cast<float*>(lds) + wave * kMostShares);
        }
        at = ends_at;
        if (at >= stop) break;
        w = Row{b + 1, at, next_len};
        __syncthreads();                                     // the next row's tiles reuse the LDS
    }
}

// After k_kv_attn, workgroups x of every (row, key-value head): the first
// `joins` join the shares of four query heads of the group, one a wave, where
// there are several; with logits the others add the attention weights of 256
// tokens each.
__global__ void __launch_bounds__(256) k_kv_join(const KVPool p, const Attn a, uint32_t joins) {
    __shared__ float2 stat[256];      // of a head: maximum, 1 / sum
    __shared__ float factors[4][kMostShares];
    ask_for(p.tables, p.heads, a.rows, a.scale_log2);
    const uint32_t bh = blockIdx.y + blockIdx.z * 65535u;
    if (bh >= a.rows * p.heads) return;
    const uint32_t b = bh / p.heads, h = bh - b * p.heads;
    const uint32_t group = a.q_heads / p.heads;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    auto parts = [&](uint32_t j) { return Parts(a, p.dim, p.heads * a.tiles, h * a.tiles + j / 16); };

    if (blockIdx.x < joins) {
        const Division cut(a);
        const Shares w(cut.find<false>(b), cut.by);
        if (w.n > 1)
            for (uint32_t j = 4 * blockIdx.x + wave; j < group; j += 4 * joins)
                parts(j).join(w, b, j % 16, h * group + j, factors[wave]);
        return;
    }
    // what does not depend on the shares is loaded first
    constexpr int G = 8;
    const uint32_t t = (blockIdx.x - joins) * 256 + tid, len = kv_length(a.lengths, b, a.max_length);
    if ((blockIdx.x - joins) * 256 >= len) return;
    uint32_t row = 0;
    const bool ok = t < len && p.row(b, h, t, row);
    const float* const s = a.logits + ((size_t)b * a.q_heads + h * group) * a.logit_stride + (ok ? t : 0);
    float v[G], before = 0.0f, sum = 0.0f;
#pragma unroll
    for (int j = 0; j < G; j++) v[j] = s[(size_t)((uint32_t)j < group ? j : 0) * a.logit_stride];
    if (ok) before = p.weights[row];
    const Division cut(a);
    const Shares w(cut.find<false>(b), cut.by);
    for (uint32_t j0 = 0; j0 < group; j0 += 256) {
        const uint32_t nj = group - j0 < 256 ? group - j0 : 256;
        __syncthreads();
        for (uint32_t j = wave; j < nj; j += 4) {
            const Parts pt = parts(j0 + j);
            const float2 st = w.n == 1 ? a.whole[(size_t)b * a.q_heads + h * group + j0 + j]
                                       : pt.whole(pt.ends(w, (j0 + j) % 16), w, nullptr);
            // (the sum is of weights of 2^-room)
            if (lane == 0) stat[j] = make_float2(st.x == -INFINITY ? 0.0f : st.x, st.y * __builtin_amdgcn_exp2f(-a.room));
        }
        __syncthreads();
        for (uint32_t j1 = 0; j1 < nj; j1 += G) {
            if (j0 + j1)
#pragma unroll
                for (int j = 0; j < G; j++) v[j] = s[(size_t)(j1 + j < nj ? j0 + j1 + j : 0) * a.logit_stride];
#pragma unroll
            for (int j = 0; j < G; j++)
                if (j1 + j < nj) sum += __builtin_amdgcn_exp2f(v[j] - stat[j1 + j].x) * stat[j1 + j].y;
        }
    }
    if (ok) p.weights[row] = before + sum;
}

uint32_t div_up(size_t a, size_t b) { return (uint32_t)((a + b - 1) / b); }

template <int DP, bool I8>
void launch(unsigned grid, bool save, const KVPool& p, const Attn& a, hipStream_t s) {
    if (p.dim == DP) {
        if (save) k_kv_attn<DP, I8, true, true><<<grid, 256, 0, s>>>(p, a);
        else k_kv_attn<DP, I8, false, true><<<grid, 256, 0, s>>>(p, a);
    } else {
        if (save) k_kv_attn<DP, I8, true, false><<<grid, 256, 0, s>>>(p, a);
        else k_kv_attn<DP, I8, false, false><<<grid, 256, 0, s>>>(p, a);
    }
}

template <bool I8>
void launch(unsigned grid, bool save, const KVPool& p, const Attn& a, hipStream_t s) {
    if (padded(p.dim) == 64) launch<64, I8>(grid, save, p, a, s);
    else if (padded(p.dim) == 128) launch<128, I8>(grid, save, p, a, s);
    else launch<256, I8>(grid, save, p, a, s);
}

}  // namespace

extern "C" {

int snx_k_kv_attention(const SNEPPXKVCache* c, const uint16_t* q, size_t q_stride, void* out, size_t out_stride,
                       int out_f32, const int32_t* tables, size_t width, int of_heads, const int32_t* lengths,
                       size_t rows, size_t q_heads, size_t max_length, float scale, int accumulate, void* st) {
    const KVPool p = kv_pool(c, tables, width, of_heads != 0);
    const size_t group = q_heads / c->kv_heads, tiles = (group + 15) / 16, units = c->kv_heads * tiles;
    const size_t heads = group < 16 ? group : 16;
    // As many shares as the CUs hold workgroups at once; where rows begin shares, one
    // more for each row, but a row has a step at least, and they are up to
    // kFewSteps for each share then.  No more than there are steps.
    const size_t steps = (max_length + STEP - 1) / STEP;
    const int of_cu = shares_of_cu(padded(c->head_dim), c->dtype == SNEPPX_INT8);
    const size_t shares = ((size_t)of_cu * cu_count() + units - 1) / units;
    size_t blocks = shares + rows;
    if (blocks > kFewSteps * shares) blocks = kFewSteps * shares;
    if (blocks > rows * (steps ? steps : 1)) blocks = rows * (steps ? steps : 1);
    blocks = (blocks * c->kv_heads + 7) / 8 * 8 * tiles;
    const size_t part = 2 * blocks * heads * c->head_dim * sizeof(float), ml = 2 * blocks * heads * sizeof(float2);
    const size_t logit_stride = accumulate ? steps * STEP : 0, logits = rows * q_heads * logit_stride * sizeof(float);
    const size_t whole = accumulate ? rows * q_heads * sizeof(float2) : 0;
    // (a grid has below 2^32 threads; offsets of the parts and counts of steps are of 32 bits)
    if (blocks > 0xffffff || part > 0xffffffffu || steps * rows > 0x7fff0000u || steps >= 0x1000000) {
        snx_set_error("kv_attention: %zu rows of up to %zu tokens are too many", rows, max_length);
        return -1;
    }
    // Joined within the launch, unless weights are added (by all CUs, after all
    // maxima are known) or the call is recorded: a graph may be replayed beside
    // other calls, and must not leave arrival counters that they would find.
    void* ws = nullptr;
    uint32_t* arrivals = nullptr;
    if (steps > 1 || accumulate) {
        if (!accumulate && !snx_stream_capturing(st)) {
            if (snx_span_workspaces(part + ml, rows * units * sizeof(uint32_t), st, &ws, &arrivals)) return -1;
        } else {
            ws = snx_workspace(part + ml + logits + whole, SLOT_KV_ATTN, st);
            if (!ws) return -1;
        }
    }
    Attn a;
    a.q = q;
    a.out = out;
    a.q_stride = q_stride;
    a.out_stride = out_stride;
    a.lengths = lengths;
    uint8_t* w = static_cast<uint8_t*>(ws);
    a.arrivals = arrivals;
    a.part = reinterpret_cast<float*>(w);
    a.logits = accumulate ? reinterpret_cast<float*>(w + part) : nullptr;
    a.ml = reinterpret_cast<float2*>(w + part + logits);
    a.whole = reinterpret_cast<float2*>(w + part + logits + ml);
    a.rows = (uint32_t)rows;
    a.q_heads = (uint32_t)q_heads;
    a.max_length = (uint32_t)max_length;
    a.tiles = (uint32_t)tiles;
    a.heads = (uint32_t)heads;
    a.by_eights = divider(8 * tiles);
    a.by_heads = divider(c->kv_heads);
    a.by_shares = divider(shares);
    a.shares = (uint32_t)shares;
    a.about_shares = (uint32_t)(of_cu > 1 ? shares + shares / 8 : shares);
    a.logit_stride = (uint32_t)logit_stride;
    a.scale_log2 = scale * 1.44269504088896340736f;
    uint32_t room = kLag;
    while (((size_t)1 << (room - kLag)) < max_length) room++;
    a.room = (float)room;
    a.out_f32 = out_f32;
    if (c->dtype == SNEPPX_INT8) launch<true>((unsigned)blocks, accumulate != 0, p, a, S(st));
    else launch<false>((unsigned)blocks, accumulate != 0, p, a, S(st));
    if (snx_launch_check("k_kv_attn")) return -1;
    if (!ws || arrivals) return 0;
    const uint32_t joins = div_up(group, 4);
    const size_t gx = joins + (accumulate ? steps * STEP / 256 + 1 : 0);
    const size_t bh = rows * c->kv_heads;
    k_kv_join<<<dim3((unsigned)gx, (unsigned)(bh < 65535 ? bh : 65535), div_up(bh, 65535)), 256, 0, S(st)>>>(p, a, joins);
    return snx_launch_check("k_kv_join");
}

}  // extern "C"
