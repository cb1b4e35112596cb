// kv_cache_kernels.hip - writing and cutting the paged key-value cache
// (include/sneppx_kv.h): append and eviction.  The int8 rule has to round as
// quant_kernels.hip does, so this file is built like that one, with IEEE
// divisions and without contraction.
#include <hip/hip_runtime.h>

#include <atomic>
#include <cfloat>
#include <cstdint>

#include "codec.h"
#include "kv_pool.h"
#include "launch.h"
#include "../snx_internal.h"

using namespace snx;

namespace {

hipStream_t S(void* s) { return reinterpret_cast<hipStream_t>(s); }

// max over non-NaN values, as the reference's `if (a > m) m = a`
__device__ __forceinline__ float nanless_max(float a, float b) { return b > a ? b : a; }

// of LR lanes, to all of them: exchanges of neighbours, pairs, halves of 8, of 16 and
// of 32 lanes
template <int LR>
__device__ __forceinline__ float row_max(float m) {
    m = nanless_max(m, lane_step<0xB1, 0xf>(m, m));
    m = nanless_max(m, lane_step<0x4E, 0xf>(m, m));
    m = nanless_max(m, lane_step<0x141, 0xf>(m, m));
    if (LR >= 16) m = nanless_max(m, lane_step<0x140, 0xf>(m, m));
    if (LR >= 32) m = nanless_max(m, __shfl_xor(m, 16));
    return m;
}

// ------------------------------------------------------------------- append
struct NewRows {
    const uint16_t *k, *v;
    size_t k_stride, v_stride;
    uint16_t *k_stored, *v_stored;
    const int32_t *starts, *lengths, *next_pos;
    uint32_t tokens, rows, slots;
    int aligned, stored_aligned;
};

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

// LR lanes per (token, key or value, head), eight of its values each: one pass
// with the row in registers, 16-byte loads and (int8: 8-byte) stores.  What
// bounds it: at a decode batch the launch (16 tokens of 8 heads of 128: 3 us),
// at a prompt the reads and writes.
template <bool I8, int LR>
__global__ void __launch_bounds__(256) k_kv_append(const KVPool p, const NewRows n) {
    ask_for(p.tables, p.heads, n.starts, n.tokens);
    const uint64_t first = (uint64_t)blockIdx.x * (256 / LR);
    const uint32_t per = 2 * p.heads, t0 = (uint32_t)(first / per);
    const uint32_t rest = (uint32_t)(first - (uint64_t)t0 * per) + threadIdx.x / LR;
    const uint32_t t = t0 + rest / per;
    if (t >= n.tokens) return;
    const uint32_t which = rest % per, d = 8 * (threadIdx.x % LR);
    const bool is_v = which >= p.heads;
    const uint32_t h = is_v ? which - p.heads : which;

    // (loaded ahead of the look-ups, which depend on one another)
    const uint16_t* x = (is_v ? n.v + t * n.v_stride : n.k + t * n.k_stride) + (size_t)h * p.dim + d;
    u32x4 w = {0u, 0u, 0u, 0u};
    const bool in = d < p.dim;
    if (in) {
        if (n.aligned) w = *reinterpret_cast<const u32x4*>(x);
        else
#pragma unroll
            for (int e = 0; e < 4; e++) w[e] = x[2 * e] | (uint32_t)x[2 * e + 1] << 16;
    }

    // the row of token t: the last one whose tokens start at or before it
    uint32_t b = t;
    int32_t back = 1;
    if (n.starts) {
        b = 0;
        uint32_t left = n.rows;
        if (__ballot(t == (uint32_t)__builtin_amdgcn_readfirstlane(t)) == ~0ull) {
            // one token in the wave: 64 rows are asked at once
            const uint32_t lane = threadIdx.x & 63;
            while (left > 1) {
                const uint32_t step = (left + 63) / 64, at = lane * step;
                const uint32_t k = __popcll(__ballot(at < left && n.starts[b + (at < left ? at : 0)] <= (int32_t)t));
                const uint32_t skip = k ? (k - 1) * step : 0;
                b += skip;
                left = left - skip < step ? left - skip : step;
            }
        } else {
            while (left > 1) {
                const uint32_t half = left / 2;
                const bool up = n.starts[b + half] <= (int32_t)t;
                b += up ? half : 0;
                left = up ? left - half : half;
            }
        }
        back = n.starts[b + 1] - (int32_t)t;
        if (back <= 0 || n.starts[b] > (int32_t)t) return;
    }
    const int32_t slot = n.lengths[b] - back;
    uint32_t r;
    if (slot < 0 || (uint32_t)slot >= n.slots || !p.row(b, h, (uint32_t)slot, r)) return;

    if (I8) {
        float f[8], m = 0.0f;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            f[2 * e] = u2f(w[e] << 16);
            f[2 * e + 1] = u2f(w[e] & 0xFFFF0000u);
        }
#pragma unroll
        for (int e = 0; e < 8; e++) m = nanless_max(m, fabsf(f[e]));
        m = row_max<LR>(m);
        const float s = m < FLT_MIN ? 1.0f : m / 127.0f, inv = 1.0f / s;
        // Numbers below 128 round half away by adding the number below 1/2 and
        // cutting; what the rule gives for others (an infinity or NaN in the row, a
        // scale whose reciprocal is infinite) takes the long way.
        float all = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; e++) all += fabsf(f[e]);
        const bool plain = all < INFINITY && m < INFINITY && inv < INFINITY;
        u32x2 q = {0u, 0u};
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const float v = f[e] * inv;
            const int c = plain ? (int)(v + copysignf(0.49999997f, v)) : clampi(round_i32(v), -128, 127);
            q[e >> 2] |= (uint32_t)(c & 0xFF) << (8 * (e & 3));
            f[e] = (float)c * s;
        }
        if (in) *reinterpret_cast<u32x2*>((is_v ? p.v : p.k) + (size_t)r * p.dim + d) = q;
        if (d == 0) (is_v ? p.vs : p.ks)[r] = s;
#pragma unroll
        for (int e = 0; e < 4; e++) w[e] = bf16x2_out(f[2 * e], f[2 * e + 1]);
    } else if (in) {
        *reinterpret_cast<u32x4*>((is_v ? p.v : p.k) + ((size_t)r * p.dim + d) * 2) = w;
    }
    if (n.k_stored && in) {
        uint16_t* to = (is_v ? n.v_stored : n.k_stored) + ((size_t)t * p.heads + h) * p.dim + d;
        if (n.stored_aligned) *reinterpret_cast<u32x4*>(to) = w;
        else
#pragma unroll
            for (int e = 0; e < 8; e++) to[e] = (uint16_t)(w[e >> 1] >> (16 * (e & 1)));
    }
    if (d == 0 && !is_v) {
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
constexpr int kDigit = 11;               // digits of 11, 11 and 10 bits, from the top
constexpr int kBins = 1 << kDigit;
constexpr uint32_t kLogChunk = 12, kMostLog = 15;    // of the slots of a long row that a workgroup has
constexpr size_t kLong = 16384;          // longer rows (half of it in small pages) are cut by several workgroups
constexpr uint32_t kMoveAtOnce = 64;     // moves that the workgroup which finds them makes itself

// a count per wave -> its exclusive prefix over the waves, and the total
__device__ __forceinline__ uint32_t wave_prefix(uint32_t x, uint32_t* sh, uint32_t& total) {
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    __syncthreads();
    if (lane == 0) sh[w] = x;
    __syncthreads();
    const uint32_t upto = lane_prefix(lane < kCutWaves ? sh[lane] : 0u);
    total = __builtin_amdgcn_readlane(upto, kCutWaves - 1);
    return __builtin_amdgcn_readlane(upto, w) - x;
}

// rows of the pool (k, v and the planes) of slots of[i] to those of slots
// to[i], for `n` moves, by `threads` threads of which this is `me`, with U of a
// thread's 16-byte loads in flight
template <int U>
__device__ __forceinline__ void move_rows(const KVPool& p, uint32_t b, uint32_t h, uint32_t row_bytes,
                                          const uint32_t* to, const uint32_t* of, uint32_t n, uint32_t me,
                                          uint32_t threads) {
    const uint32_t per = row_bytes / 16, chunks = n * per;
#pragma unroll 1
    for (uint32_t i0 = me; i0 < chunks; i0 += U * threads) {
        u32x4 x[U], y[U];
        uint32_t src[U], dst[U], c[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const uint32_t i = i0 + u * threads < chunks ? i0 + u * threads : i0, m = i / per;
            c[u] = 16 * (i - m * per);
            src[u] = of[m];
            dst[u] = to[m];
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            (void)p.row(b, h, src[u], src[u]);
            (void)p.row(b, h, dst[u], dst[u]);
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            x[u] = *reinterpret_cast<const u32x4*>(p.k + (size_t)src[u] * row_bytes + c[u]);
            y[u] = *reinterpret_cast<const u32x4*>(p.v + (size_t)src[u] * row_bytes + c[u]);
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (i0 + u * threads >= chunks) continue;
            *reinterpret_cast<u32x4*>(p.k + (size_t)dst[u] * row_bytes + c[u]) = x[u];
            *reinterpret_cast<u32x4*>(p.v + (size_t)dst[u] * row_bytes + c[u]) = y[u];
        }
    }
    for (uint32_t m = me; m < n; m += threads) {
        uint32_t t, f;
        (void)p.row(b, h, to[m], t);
        (void)p.row(b, h, of[m], f);
        const float w = p.weights[f];
        const int32_t pos = p.positions[f];
        if (p.ks) {
            const float x = p.ks[f], y = p.vs[f];
            p.ks[t] = x;
            p.vs[t] = y;
        }
        p.weights[t] = w;
        p.positions[t] = pos;
    }
}

// What the workgroups of a long row find about it, one after the other
struct Chunk {
    uint32_t cands, low_cands;     // its keys with the first digit of the threshold; those below the budget
    uint32_t sure, low_sure;       // its keys above them
};
__host__ __device__ __forceinline__ uint32_t chunks_of(uint32_t slots, uint32_t log) { return (slots + (1u << log) - 1) >> log; }

struct Cut {
    const int32_t *lengths, *next_pos;
    int32_t* new_lengths;
    uint32_t rows, max_length, budget, recent, most, row_bytes;
    uint32_t* counts;          // [rows * heads] moves of each row and head (unless moved at once)
    uint32_t* moves;           // [rows * heads][2][most] slots: targets, then sources
    uint32_t chunks, log;      // the rest of long rows, [rows * heads] of each; log2 of a chunk's slots
    uint32_t* keys;            // [chunks][1 << log]
    uint32_t* cands;           // [chunks][1 << log]: `cands` keys of each chunk, in the order of their slots
    uint32_t* firsts;          // [chunks][kBins / 2]: the chunk's keys by first digit, 16 bits each
    Chunk* found;              // [chunks]
    uint32_t* absent;          // [chunks]: whether a page is not there
    uint2* least;              // [chunks], instead: the lowest key and its slot
};

// The keys of a lane's slots, every 64th from `t` on
struct Ranks {
    const KVPool& p;
    const int32_t* table;
    uint32_t L, t, page, slot, pages64, slots64, last_page, first_row, page_rows;
    int32_t from;
    bool gone = false;
    __device__ __forceinline__ Ranks(const KVPool& pool, const Cut& a, uint32_t b, uint32_t h, uint32_t len, uint32_t start)
        : p(pool), table(pool.tables + (size_t)b * pool.width), L(len), t(start) {
        const int64_t from64 = (int64_t)a.next_pos[b] - (int64_t)a.recent;
        from = (int32_t)(from64 < INT32_MIN ? INT32_MIN : from64);
        pages64 = p.page_of(64);
        slots64 = 64 - pages64 * p.page_size;
        last_page = p.page_of(L - 1);
        first_row = h * p.page_size;
        page_rows = p.heads * p.page_size;
        page = p.page_of(t);
        slot = t - page * p.page_size;
    }
    // G at once (past the length: of its last page), so that their look-ups and
    // loads are in flight together; 0 past the length
    template <int G>
    __device__ __forceinline__ void next(uint32_t (&q)[G]) {
        uint32_t rows[G];
        float w[G];
        int32_t pos[G];
#pragma unroll
        for (int i = 0; i < G; i++) {
            const uint32_t e = (uint32_t)table[page < last_page ? page : last_page];
            const bool there = e < p.pages;
            gone |= !there;
            rows[i] = there ? e * page_rows + first_row + slot : 0;
            page += pages64;
            slot += slots64;
            if (slot >= p.page_size) {
                slot -= p.page_size;
                page++;
            }
        }
#pragma unroll
        for (int i = 0; i < G; i++) {
            w[i] = p.weights[rows[i]];
            pos[i] = p.positions[rows[i]];
        }
#pragma unroll
        for (int i = 0; i < G; i++, t += 64) q[i] = t < L ? rank_key(w[i], pos[i], from) : 0u;
    }
};

__device__ __forceinline__ uint32_t lane_rank(uint64_t m) {
    return __builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0));
}

// The budget-th largest key by its digits from the top: each time a histogram of
// the keys that agree with the digits found so far.
struct Threshold {
    uint32_t prefix = 0, known = 0;      // the digits found so far, their bits
    uint32_t want, tied = 0;             // it is the want-th largest of the `tied` keys that share them
    int shift = 32 - kDigit;             // of the next digit (the last has a known bit in it, alike in all)
    __device__ __forceinline__ explicit Threshold(uint32_t budget) : want(budget) {}

    // counts U keys of each lane
    template <int U>
    __device__ __forceinline__ void tally(uint32_t* hist, const uint32_t (&q)[U], const bool (&there)[U]) const {
        bool mine[U], other = false;
        uint32_t digit[U], n = 0;
#pragma unroll
        for (int u = 0; u < U; u++) {
            mine[u] = there[u] && ((q[u] ^ prefix) & known) == 0;
            digit[u] = (q[u] >> shift) & (kBins - 1);
        }
        // many alike (zeros, recent ones) are counted at once
        const uint32_t first = __builtin_amdgcn_readfirstlane(digit[0]);
#pragma unroll
        for (int u = 0; u < U; u++) {
            other |= mine[u] && digit[u] != first;
            n += __popcll(__ballot(mine[u]));
        }
        if (__ballot(other) == 0) {
            if ((threadIdx.x & 63) == 0 && n) atomicAdd(&hist[first], n);
            return;
        }
#pragma unroll
        for (int u = 0; u < U; u++)
            if (mine[u]) atomicAdd(&hist[digit[u]], 1u);
    }
    // The digit, by all threads: from the top the wave's 128 bins (the first wave has the
    // highest) where the number passes `want`, then, in every wave, the bin of them.
    __device__ __forceinline__ void find(const uint32_t* hist, uint32_t* sh) {
        const int tid = threadIdx.x, lane = tid & 63;
        const u32x2* const pairs = reinterpret_cast<const u32x2*>(hist) + kBins / 2 - 1;
        const u32x2 mine = *(pairs - tid);
        const uint32_t here = last_lane(lane_prefix(mine[0] + mine[1]));
        if (lane == 0) sh[tid >> 6] = here;
        __syncthreads();
        const uint32_t n = lane < kCutWaves ? sh[lane] : 0u, upto = lane_prefix(n);
        const int w = __builtin_ctzll(__ballot(upto >= want));
        const uint32_t before = __builtin_amdgcn_readlane(upto - n, w);
        const u32x2 pair = *(pairs - (64 * w + lane));
        const uint32_t upto2 = before + lane_prefix(pair[0] + pair[1]), upto1 = upto2 - pair[0];
        const int at = __builtin_ctzll(__ballot(upto2 >= want));
        const uint32_t high = __builtin_amdgcn_readlane(upto1, at);       // with the pair's higher bin
        const uint32_t n0 = __builtin_amdgcn_readlane(pair[0], at), n1 = __builtin_amdgcn_readlane(pair[1], at);
        const bool lower = want > high;
        tied = lower ? n0 : n1;
        want -= lower ? high : high - n1;
        prefix |= (uint32_t)(kBins - 1 - 2 * (64 * w + at) - lower) << shift;
        known = ~0u << shift;
        shift = shift > kDigit ? shift - kDigit : 0;
    }
    __device__ __forceinline__ bool done() const { return want == tied || known == ~0u; }
    // Above the prefix all stay, of those equal to it the first `want` in the order of
    // the slots: where all of them do, whatever their other digits are, the prefix
    // goes below them (it is not 0: some key is left out).
    __device__ __forceinline__ void settle() {
        if (want != tied) return;
        prefix -= 1;
        want = 0;
    }
};

// Lists the free slots below the budget and those from it on that stay, both in
// ascending order, of `steps` x 1024 slots from `slot0` on whose keys are in LDS;
// so many ties, free slots and ones to move come before.  Each wave has consecutive
// slots, so that order by (wave, step, lane) is order by slot.  (Slots past the
// length have the lowest key and come after all others.)
__device__ __forceinline__ uint32_t list_slots(const uint32_t* keys, uint32_t slot0, uint32_t steps, uint32_t budget,
                                               const Threshold& at, uint32_t ties, uint32_t holes0, uint32_t fars0,
                                               uint32_t* sh, uint32_t* to, uint32_t* of) {
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t mine = wave * steps * 64, w0 = slot0 + mine;
    const uint32_t* const q = keys + mine + lane;
    uint32_t total, n = 0;
    if (at.want) {
#pragma unroll 1
        for (uint32_t i = 0; i < steps; i++) n += __popcll(__ballot(q[64 * i] == at.prefix));
        ties += wave_prefix(n, sh, total);
    }
    // lane i has step i: the free slots, those that stay, and the numbers of both before
    // them (the latter in the upper half)
    uint32_t lo = 0, hi = 0;
#pragma unroll 1
    for (uint32_t i = 0; i < steps; i++) {
        uint64_t s = __ballot(q[64 * i] > at.prefix);
        if (at.want) {
            const uint64_t tb = __ballot(q[64 * i] == at.prefix);
            s |= __ballot((__builtin_amdgcn_inverse_ballot_w64(tb)) && ties + lane_rank(tb) < at.want);
            ties += __popcll(tb);
        }
        lo = lane == i ? (uint32_t)s : lo;
        hi = lane == i ? (uint32_t)(s >> 32) : hi;
    }
    const uint64_t s = (uint64_t)hi << 32 | lo;
    const uint32_t first = w0 + 64 * lane;
    const uint64_t part = ((uint64_t)1 << ((budget - first) & 63)) - 1;
    const uint64_t low = lane >= steps || first >= budget ? 0 : budget - first >= 64 ? ~0ull : part;
    const uint64_t hole = low & ~s, far = s & ~low;
    const uint32_t own = __popcll(hole) | __popcll(far) << 16, upto = lane_prefix(own), before = upto - own;
    const uint32_t both = __builtin_amdgcn_readlane(upto, 63);
    const uint32_t fars = fars0 + wave_prefix(both >> 16, sh, total) + (before >> 16);
    const uint32_t holes = holes0 + wave_prefix(both & 0xFFFF, sh, total) + (before & 0xFFFF);
#pragma unroll 1
    for (uint32_t i = 0; i < steps; i++) {
        auto write = [&](uint64_t mine, uint32_t first, uint32_t* to) {
            const uint64_t m = (uint64_t)__builtin_amdgcn_readlane((uint32_t)(mine >> 32), i) << 32 |
                               (uint32_t)__builtin_amdgcn_readlane((uint32_t)mine, i);
            const uint32_t at = __builtin_amdgcn_readlane(first, i) + lane_rank(m);
            if (__builtin_amdgcn_inverse_ballot_w64(m)) to[at] = w0 + 64 * i + lane;
        };
        // a step lies below the budget, or from it on, or has it within
        if (w0 + 64 * i < budget) write(hole, holes, to);
        if (w0 + 64 * i + 64 > budget) write(far, fars, of);
    }
    return total;
}

// Of one token too many no threshold is needed: the lowest key goes, of equal ones
// the one in the highest slot, and the last slot's token moves there.
struct Least {
    uint32_t key = ~0u, slot = 0;
    __device__ __forceinline__ void add(uint32_t q, uint32_t t) {       // slots in ascending order
        slot = q <= key ? t : slot;
        key = q <= key ? q : key;
    }
    __device__ __forceinline__ void of_wave() {
        const uint32_t least = ~lane_max(~key);
        slot = lane_max(key == least ? slot : 0u);
        key = least;
    }
    // of `waves` waves, to all of them
    __device__ __forceinline__ void of_group(uint2* sh, uint32_t waves) {
        const uint32_t lane = threadIdx.x & 63;
        of_wave();
        if (lane == 0) sh[threadIdx.x >> 6] = make_uint2(key, slot);
        __syncthreads();
        const uint2 v = sh[lane < waves ? lane : 0];
        key = v.x;
        slot = v.y;
        of_wave();
    }
};

// One workgroup per (row, head) of rows that are not long (see is_long).  A call runs through the code
// about once, and its instructions one after the other are its time: the loops are
// left rolled (the threshold of 16 x 8 of 2049: 8.4 us; unrolled, with keys in
// registers, twice the code, 8.5).
// MOVE: with so few moves that the workgroup makes them at once.
template <bool MOVE>
__global__ void __launch_bounds__(kCutThreads) k_kv_cut(const KVPool p, const Cut a) {
    extern __shared__ __attribute__((aligned(16))) uint32_t keys[];
    __shared__ __attribute__((aligned(16))) uint32_t hist[kBins];
    __shared__ uint32_t sh[kCutWaves];
    __shared__ uint2 sh2[kCutWaves];
    __shared__ uint32_t list[MOVE ? 2 * kMoveAtOnce : 1];
    ask_for(p.tables, p.heads, a.budget, a.counts);
    const uint32_t b = blockIdx.x / p.heads, h = blockIdx.x - b * p.heads;
    const int tid = threadIdx.x;
    const uint32_t L = kv_length(a.lengths, b, a.max_length), budget = a.budget;
    const uint32_t steps = (L + kCutThreads - 1) / kCutThreads;       // slots of a thread
    const uint32_t t0 = (tid & ~63) * steps + (tid & 63);
    u32x2* const bins = reinterpret_cast<u32x2*>(hist) + tid;

    bool gone = false;
    if (L > budget) {
        Ranks ranks(p, a, b, h, L, t0);
        uint32_t i = 0;
#pragma unroll 1
        for (; i + 4 < steps; i += 8) {              // (by fours 8 x 8 of 16000 15.2 us, so 14.2)
            uint32_t q[8];
            ranks.next<8>(q);
#pragma unroll
            for (uint32_t u = 0; u < 8; u++)
                if (i + u < steps) keys[t0 + 64 * (i + u)] = q[u];
        }
        if (i < steps) {
            uint32_t q[4];
            ranks.next<4>(q);
#pragma unroll
            for (uint32_t u = 0; u < 4; u++)
                if (i + u < steps) keys[t0 + 64 * (i + u)] = q[u];
        }
        gone = ranks.gone;
    }
    *bins = u32x2{0u, 0u};
    gone = __syncthreads_or(gone);
    if (tid == 0 && h == 0 && a.new_lengths) a.new_lengths[b] = (int32_t)(L > budget && !gone ? budget : L);
    if (L <= budget || gone) {
        if (!MOVE && tid == 0) a.counts[blockIdx.x] = 0;
        return;
    }
    uint32_t* const to = MOVE ? list : a.moves + (size_t)blockIdx.x * 2 * a.most;
    uint32_t* const of = to + (MOVE ? kMoveAtOnce : a.most);
    uint32_t total;
    if (L - budget == 1) {                           // (16 x 8 of 2049: 5.7 us, 8.4 the other way)
        Least least;
#pragma unroll 1
        for (uint32_t i = 0; i < steps; i++)
            if (t0 + 64 * i < L) least.add(keys[t0 + 64 * i], t0 + 64 * i);
        least.of_group(sh2, kCutWaves);
        total = least.slot != budget;
        if (tid == 0 && total) {
            to[0] = least.slot;
            of[0] = budget;
        }
    } else {
        Threshold at(budget);
#pragma unroll 1
        for (;;) {
#pragma unroll 1
            for (uint32_t i = 0; i < steps; i++) at.tally<1>(hist, {keys[t0 + 64 * i]}, {t0 + 64 * i < L});
            __syncthreads();
            at.find(hist, sh);
            if (at.done()) break;
            __syncthreads();
            *bins = u32x2{0u, 0u};
            __syncthreads();
        }
        at.settle();
        total = list_slots(keys, 0, steps, budget, at, 0, 0, 0, sh, to, of);
    }
    if (MOVE) {
        __syncthreads();
        move_rows<1>(p, b, h, a.row_bytes, to, of, total, tid, kCutThreads);
    } else if (tid == 0) {
        a.counts[blockIdx.x] = total;
    }
}

// ------------------------------------------------------------- of long rows
// A workgroup has 4096 slots, up to 32768 where there are many, in three kernels:
// k_kv_rank counts their keys by first digit; with all chunks' counts k_kv_part
// finds the threshold's and puts the keys that share it apart; k_kv_list finds the
// threshold among these, and where its own slots stand in the lists.  (us of a call
// that cuts so, and with one workgroup for each row and head: 2 rows of 30001 and 8
// heads 32 and 41, 4 of 60000 70 and 113; 1 of 16384 30 and 30, of 12288 29 and 26,
// of 8192 27 and 21.  Every workgroup adds up the counts of all chunks: two tokens
// too many in 8 rows of 131072 take 83 us in chunks for two workgroups a CU, 121 in
// 4096s; in 1 of 1000000 94 and 248.)
__device__ __forceinline__ bool long_row(const KVPool& p, const Cut& a, uint32_t& bh, uint32_t& b, uint32_t& h, uint32_t& L) {
    ask_for(p.tables, p.heads, a.counts, a.absent);
    bh = blockIdx.y + blockIdx.z * 65535u;
    b = bh / p.heads;
    h = bh - b * p.heads;
    if (b >= a.rows) return false;
    L = kv_length(a.lengths, b, a.max_length);
    return L > a.budget && blockIdx.x << a.log < L;
}
// a page of the row that is not there
__device__ __forceinline__ bool row_absent(const Cut& a, uint32_t bh, uint32_t chunks) {
    bool gone = false;
    for (uint32_t c = threadIdx.x; c < chunks; c += kCutThreads) gone |= a.absent[(size_t)bh * a.chunks + c] != 0;
    return __syncthreads_or(gone);
}

// One token too many at most in long rows: the lowest key of each chunk, then of all
// (us of the call, and by the kernels below: 1 row of 30000 11.6 and 25, 8 of 131072
// 45 and 85).
__global__ void __launch_bounds__(kCutThreads) k_kv_least(const KVPool p, const Cut a) {
    __shared__ uint2 sh[kCutWaves];
    const int tid = threadIdx.x;
    uint32_t bh, b, h, L;
    if (!long_row(p, a, bh, b, h, L)) return;
    const size_t chunk = (size_t)bh * a.chunks + blockIdx.x;
    const uint32_t steps = (1u << a.log) / kCutThreads, mine = (tid & ~63) * steps + (tid & 63);
    Ranks ranks(p, a, b, h, L, (blockIdx.x << a.log) + mine);
    Least least;
#pragma unroll 1
    for (uint32_t i = 0; i < steps; i += 4) {
        const uint32_t t = ranks.t;
        uint32_t q[4];
        ranks.next<4>(q);
#pragma unroll
        for (int u = 0; u < 4; u++)
            if (t + 64 * u < L) least.add(q[u], t + 64 * u);
    }
    const bool gone = __syncthreads_or(ranks.gone);
    least.of_group(sh, kCutWaves);
    if (tid == 0) {
        a.least[chunk] = make_uint2(least.key, least.slot);
        a.absent[chunk] = gone;
    }
}
__global__ void __launch_bounds__(kCutThreads) k_kv_drop(const KVPool p, const Cut a) {
    __shared__ uint2 sh[kCutWaves];
    __shared__ uint32_t list[2];
    ask_for(p.tables, p.heads, a.budget, a.absent);
    const uint32_t tid = threadIdx.x, bh = blockIdx.x, b = bh / p.heads, h = bh - b * p.heads;
    const uint32_t L = kv_length(a.lengths, b, a.max_length), chunks = chunks_of(L, a.log);
    const bool gone = L > a.budget && row_absent(a, bh, chunks);
    if (tid == 0 && h == 0 && a.new_lengths) a.new_lengths[b] = (int32_t)(L > a.budget && !gone ? a.budget : L);
    if (L <= a.budget || gone) return;
    Least least;
    for (uint32_t c = tid; c < chunks; c += kCutThreads) {
        const uint2 v = a.least[(size_t)bh * a.chunks + c];
        least.add(v.x, v.y);
    }
    least.of_group(sh, kCutWaves);
    if (least.slot == a.budget) return;
    if (tid == 0) {
        list[0] = least.slot;
        list[1] = a.budget;
    }
    __syncthreads();
    move_rows<1>(p, b, h, a.row_bytes, list, list + 1, 1, tid, kCutThreads);
}

__global__ void __launch_bounds__(kCutThreads) k_kv_rank(const KVPool p, const Cut a) {
    __shared__ __attribute__((aligned(16))) uint32_t hist[kBins];
    const int tid = threadIdx.x;
    uint32_t bh, b, h, L;
    if (!long_row(p, a, bh, b, h, L)) return;
    reinterpret_cast<u32x2*>(hist)[tid] = u32x2{0u, 0u};
    __syncthreads();
    const size_t chunk = (size_t)bh * a.chunks + blockIdx.x;
    const uint32_t steps = (1u << a.log) / kCutThreads, mine = (tid & ~63) * steps + (tid & 63);
    uint32_t* const keys = a.keys + (chunk << a.log) + mine;
    Ranks ranks(p, a, b, h, L, (blockIdx.x << a.log) + mine);
#pragma unroll 1
    for (uint32_t i = 0; i < steps; i += 4) {
        const uint32_t t = ranks.t;
        uint32_t q[4];
        ranks.next<4>(q);
        const bool there[4] = {t < L, t + 64 < L, t + 128 < L, t + 192 < L};
#pragma unroll
        for (int u = 0; u < 4; u++) keys[64 * (i + u)] = q[u];
        Threshold(0).tally<4>(hist, q, there);
    }
    const bool gone = __syncthreads_or(ranks.gone);
    const u32x2 n = reinterpret_cast<const u32x2*>(hist)[tid];
    a.firsts[chunk * (kBins / 2) + tid] = n[0] | n[1] << 16;
    if (tid == 0) a.absent[chunk] = gone;
}

// the threshold's first digit, from the chunks' counts
__device__ __forceinline__ Threshold first_digit(const Cut& a, uint32_t bh, uint32_t chunks, uint32_t* hist, uint32_t* sh) {
    u32x2 bins = {0u, 0u};
    const uint32_t* const firsts = a.firsts + (size_t)bh * a.chunks * (kBins / 2) + threadIdx.x;
#pragma unroll 8
    for (uint32_t c = 0; c < chunks; c++) {
        const uint32_t n = firsts[(size_t)c * (kBins / 2)];
        bins += u32x2{n & 0xFFFF, n >> 16};
    }
    reinterpret_cast<u32x2*>(hist)[threadIdx.x] = bins;
    __syncthreads();
    Threshold at(a.budget);
    at.find(hist, sh);
    return at;
}

__global__ void __launch_bounds__(kCutThreads) k_kv_part(const KVPool p, const Cut a) {
    __shared__ __attribute__((aligned(16))) uint32_t hist[kBins];
    __shared__ uint32_t sh[kCutWaves];
    const uint32_t tid = threadIdx.x, lane = tid & 63;
    uint32_t bh, b, h, L, q[4];
    if (!long_row(p, a, bh, b, h, L)) return;
    const uint32_t chunks = chunks_of(L, a.log);
    const size_t chunk = (size_t)bh * a.chunks + blockIdx.x;
    const uint32_t steps = (1u << a.log) / kCutThreads, mine = (tid & ~63u) * steps + lane;
    const uint32_t t0 = (blockIdx.x << a.log) + mine;
    const uint32_t* const keys = a.keys + (chunk << a.log) + mine;
    uint32_t* const cands_at = a.cands + (chunk << a.log);
    auto four = [&](uint32_t i) {
#pragma unroll
        for (int u = 0; u < 4; u++) q[u] = keys[64 * (i + u)];
    };
    four(0);
    if (row_absent(a, bh, chunks)) return;
    const Threshold at = first_digit(a, bh, chunks, hist, sh);

    uint32_t cands = 0, low_cands = 0, sure = 0, low_sure = 0, total, low_total, to = 0;
    // first the numbers, then the keys
#pragma unroll 1
    for (int listing = 0; listing < 2; listing++) {
#pragma unroll 1
        for (uint32_t i = 0; i < steps; i += 4) {
            if (steps > 4) four(i);
#pragma unroll
            for (int u = 0; u < 4; u++) {
                const uint32_t t = t0 + 64 * (i + u), digit = q[u] & at.known;
                const uint64_t who = __ballot(t < L && digit == at.prefix);
                if (listing) {
                    if (__builtin_amdgcn_inverse_ballot_w64(who)) cands_at[to + lane_rank(who)] = q[u];
                    to += __popcll(who);
                    continue;
                }
                const uint64_t above = __ballot(t < L && digit > at.prefix), below = __ballot(t < a.budget);
                cands += __popcll(who);
                low_cands += __popcll(who & below);
                sure += __popcll(above);
                low_sure += __popcll(above & below);
            }
        }
        if (listing) break;
        to = wave_prefix(cands | low_cands << 16, sh, total) & 0xFFFF;
        (void)wave_prefix(sure | low_sure << 16, sh, low_total);
    }
    if (tid == 0) a.found[chunk] = Chunk{total & 0xFFFF, total >> 16, low_total & 0xFFFF, low_total >> 16};
}

__global__ void __launch_bounds__(kCutThreads) k_kv_list(const KVPool p, const Cut a) {
    extern __shared__ __attribute__((aligned(16))) uint32_t keys[];
    __shared__ __attribute__((aligned(16))) uint32_t hist[kBins];
    __shared__ uint32_t sh[kCutWaves], sums[4][kCutWaves];
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    uint32_t bh, b, h, L;
    const bool cut = long_row(p, a, bh, b, h, L);
    if (b >= a.rows) return;
    const uint32_t chunks = chunks_of(L, a.log), chunk = blockIdx.x, size = 1u << a.log;
    const size_t row = (size_t)bh * a.chunks;
    if (cut)
        for (uint32_t i = tid; i < size / 4; i += kCutThreads)
            reinterpret_cast<u32x4*>(keys)[i] = reinterpret_cast<const u32x4*>(a.keys + ((row + chunk) << a.log))[i];
    const bool gone = L > a.budget && row_absent(a, bh, chunks);
    if (chunk == 0 && tid == 0 && h == 0 && a.new_lengths) a.new_lengths[b] = (int32_t)(L > a.budget && !gone ? a.budget : L);
    if (!cut || gone) {
        if (chunk == 0 && tid == 0) a.counts[bh] = 0;
        return;
    }
    Threshold at = first_digit(a, bh, chunks, hist, sh);
    // each wave has every 16th chunk's, four of a lane at once
    auto each = [&](auto f) {
#pragma unroll 1
        for (uint32_t c = wave; c < chunks; c += kCutWaves) {
            const uint32_t n = a.found[row + c].cands;
            const uint32_t* const cands = a.cands + ((row + c) << a.log);
#pragma unroll 1
            for (uint32_t i = lane; i < n + lane; i += 256) {
                uint32_t q[4];
                bool there[4];
#pragma unroll
                for (uint32_t u = 0; u < 4; u++) {
                    there[u] = i + 64 * u < n;
                    q[u] = cands[there[u] ? i + 64 * u : 0];
                }
                f(c, i, q, there);
            }
        }
    };
#pragma unroll 1
    while (!at.done()) {
        __syncthreads();
        reinterpret_cast<u32x2*>(hist)[tid] = u32x2{0u, 0u};
        __syncthreads();
        each([&](uint32_t, uint32_t, uint32_t (&q)[4], bool (&there)[4]) { at.tally<4>(hist, q, there); });
        __syncthreads();
        at.find(hist, sh);
    }
    at.settle();
    // of the slots before this chunk and of those below the budget: how many keys are
    // above the threshold, how many equal to it
    uint32_t more = 0, ties = 0, low_more = 0, low_ties = 0;
    for (uint32_t c = tid; c < chunks; c += kCutThreads) {
        const Chunk f = a.found[row + c];
        more += c < chunk ? f.sure : 0;
        low_more += f.low_sure;
    }
    each([&](uint32_t c, uint32_t i, uint32_t (&q)[4], bool (&there)[4]) {
        const uint32_t low = a.found[row + c].low_cands;
#pragma unroll
        for (uint32_t u = 0; u < 4; u++) {
            const bool above = there[u] && q[u] > at.prefix, tie = there[u] && q[u] == at.prefix, is_low = i + 64 * u < low;
            more += c < chunk && above;
            ties += c < chunk && tie;
            low_more += is_low && above;
            low_ties += is_low && tie;
        }
    });
    auto sum = [&](uint32_t x, int k) {
        x = last_lane(lane_prefix(x));
        if (lane == 0) sums[k][wave] = x;
    };
    sum(more, 0);
    sum(ties, 1);
    sum(low_more, 2);
    sum(low_ties, 3);
    __syncthreads();
    auto all = [&](int k) { return last_lane(lane_prefix(lane < kCutWaves ? sums[k][lane] : 0u)); };
    ties = all(1);
    low_ties = all(3);
    const uint32_t kept = all(0) + (ties < at.want ? ties : at.want);                      // before this chunk
    const uint32_t low_kept = all(2) + (low_ties < at.want ? low_ties : at.want);          // below the budget
    const uint32_t slot0 = chunk << a.log;
    uint32_t* const to = a.moves + (size_t)bh * 2 * a.most;
    (void)list_slots(keys, slot0, size / kCutThreads, a.budget, at, ties, slot0 < a.budget ? slot0 - kept : 0,
                     slot0 > a.budget ? kept - low_kept : 0, sh, to, to + a.most);
    if (chunk == 0 && tid == 0) a.counts[bh] = a.budget - low_kept;
}

// The moves that k_kv_cut or k_kv_list listed.  Sources lie in slots from the budget
// on and targets below it, so all are independent.  Rows of head_dim values in any
// order bound it: 8 x 8 of 8192 halved, 134 MB read and written, 33 us.  Heads go side
// by side, whose tokens share pages (one after the other: 36 us; 16 x 8 of 2049
// halved 27 and 30.5 us in all), and a workgroup's loads in flight lie far apart in
// the list (54 us in all; side by side 59).
__global__ void __launch_bounds__(256) k_kv_move(const KVPool p, const Cut a) {
    ask_for(p.tables, p.heads, a.budget, a.counts);
    const uint32_t bh = blockIdx.x, b = bh / p.heads, n = a.counts[bh];
    const uint32_t* to = a.moves + (size_t)bh * 2 * a.most;
    constexpr uint32_t most = 1u << 24;          // (16-byte pieces are counted in 32 bits)
    for (uint32_t m = 0; m < n; m += most)
        move_rows<4>(p, b, bh - b * p.heads, a.row_bytes, to + m, to + a.most + m, n - m < most ? n - m : most,
                     blockIdx.y * 256 + threadIdx.x, gridDim.y * 256);
}

template <int LR>
void append(bool i8, unsigned blocks, const KVPool& p, const NewRows& n, hipStream_t s) {
    if (i8) k_kv_append<true, LR><<<blocks, 256, 0, s>>>(p, n);
    else k_kv_append<false, LR><<<blocks, 256, 0, s>>>(p, n);
}

int reserve_lds(const void* kernel, size_t bytes, std::atomic<uint64_t>& done) {
    if (lds_optin(kernel, (int)bytes, done) == hipSuccess) return 0;
    snx_set_error("kv_evict: cannot reserve %zu bytes of LDS", bytes);
    return -1;
}

template <bool MOVE>
int cut(unsigned blocks, const KVPool& p, const Cut& a, hipStream_t s) {
    // (rows that nothing is cut from need no keys)
    const size_t keys = a.most ? ((size_t)a.max_length + kCutThreads - 1) / kCutThreads * kCutThreads : 0;
    static std::atomic<uint64_t> done{0};
    if (reserve_lds(reinterpret_cast<const void*>(&k_kv_cut<MOVE>), kLong * sizeof(uint32_t), done)) return -1;
    k_kv_cut<MOVE><<<blocks, kCutThreads, keys * sizeof(uint32_t), s>>>(p, a);
    return snx_launch_check("k_kv_cut");
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
    NewRows n;
    n.k = k;
    n.v = v;
    n.k_stride = k_stride;
    n.v_stride = v_stride;
    n.k_stored = k_stored;
    n.v_stored = v_stored;
    n.starts = starts;
    n.lengths = lengths;
    n.next_pos = next_pos;
    n.tokens = (uint32_t)tokens;
    n.rows = (uint32_t)rows;
    n.slots = (uint32_t)(width * c->page_size);
    n.aligned = (((uintptr_t)k | (uintptr_t)v) & 15u) == 0 && (tokens < 2 || (k_stride % 8 == 0 && v_stride % 8 == 0));
    n.stored_aligned = (((uintptr_t)k_stored | (uintptr_t)v_stored) & 15u) == 0;
    const int lr = c->head_dim <= 64 ? 8 : c->head_dim <= 128 ? 16 : 32;
    const size_t blocks = (tokens * 2 * c->kv_heads * lr + 255) / 256;
    if (blocks > 0xffffff) {          // a grid has below 2^32 threads
        snx_set_error("kv_append: %zu tokens of %zu heads are too many", tokens, c->kv_heads);
        return -1;
    }
    const bool i8 = c->dtype == SNEPPX_INT8;
    if (lr == 8) append<8>(i8, (unsigned)blocks, p, n, S(st));
    else if (lr == 16) append<16>(i8, (unsigned)blocks, p, n, S(st));
    else append<32>(i8, (unsigned)blocks, p, n, S(st));
    return snx_launch_check("k_kv_append");
}

// Pages of a few tokens scatter a row's keys, which takes a CU longer (us by one
// workgroup a row and head / by several, 3 rows of 14899 and 12 heads cut to 5598:
// pages of 1 87 / 63, of 4 54 / 49, of 8 46 / 46, of 16 40 / 42; 2 of 8000 and 8 heads
// halved, pages of 1: 37 / 38).
static bool is_long(size_t max_length, size_t most, size_t page_size) {
    return most && max_length > (page_size < 8 ? kLong / 2 : kLong);
}
// log2 of a chunk's slots: no more workgroups than two for a CU, if that is few slots
// (for k_kv_part and k_kv_list, which add up all chunks' counts; k_kv_least takes the
// same chunks)
static uint32_t chunk_log(size_t bh, size_t max_length) {
    uint32_t log = kLogChunk;
    while (log < kMostLog && bh * chunks_of((uint32_t)max_length, log) > 2 * (size_t)cu_count()) log++;
    return log;
}

size_t snx_kv_evict_ws(const SNEPPXKVCache* c, size_t rows, size_t max_length, size_t budget) {
    const size_t most = most_moves(max_length, budget), bh = rows * c->kv_heads;
    if (is_long(max_length, most, c->page_size)) {
        const uint32_t log = chunk_log(bh, max_length);
        if (max_length - budget == 1) return bh * chunks_of((uint32_t)max_length, log) * (sizeof(uint2) + sizeof(uint32_t));
        const size_t chunk = ((2u << log) + kBins / 2 + 1) * sizeof(uint32_t) + sizeof(Chunk);
        return bh * (chunks_of((uint32_t)max_length, log) * chunk + (1 + 2 * most) * sizeof(uint32_t));
    }
    return most > kMoveAtOnce ? bh * (1 + 2 * most) * sizeof(uint32_t) : 0;
}

int snx_k_kv_evict(const SNEPPXKVCache* c, const int32_t* tables, size_t width, const int32_t* lengths,
                   const int32_t* next_pos, int32_t* new_lengths, size_t rows, size_t max_length, size_t budget,
                   size_t recent, void* ws, void* st) {
    const KVPool p = kv_pool(c, tables, width);
    const size_t bh = rows * c->kv_heads;
    Cut a = {};
    a.lengths = lengths;
    a.next_pos = next_pos;
    a.new_lengths = new_lengths;
    a.max_length = (uint32_t)max_length;
    a.budget = (uint32_t)budget;
    a.recent = (uint32_t)(recent < INT32_MAX ? recent : INT32_MAX);
    a.most = most_moves(max_length, budget);
    a.row_bytes = (uint32_t)(c->head_dim * (c->dtype == SNEPPX_INT8 ? 1 : 2));
    a.rows = (uint32_t)rows;
    const hipStream_t s = S(st);
    if (is_long(max_length, a.most, c->page_size)) {
        a.log = chunk_log(bh, max_length);
        a.chunks = chunks_of(a.max_length, a.log);
        const size_t all = bh * a.chunks;
        const dim3 grid(a.chunks, (unsigned)(bh < 65535 ? bh : 65535), (unsigned)((bh + 65534) / 65535));
        if (max_length - budget == 1) {
            a.least = static_cast<uint2*>(ws);
            a.absent = reinterpret_cast<uint32_t*>(a.least + all);
            k_kv_least<<<grid, kCutThreads, 0, s>>>(p, a);
            if (snx_launch_check("k_kv_least")) return -1;
            k_kv_drop<<<(unsigned)bh, kCutThreads, 0, s>>>(p, a);
            return snx_launch_check("k_kv_drop");
        }
        a.found = static_cast<Chunk*>(ws);
        a.keys = reinterpret_cast<uint32_t*>(a.found + all);
        a.cands = a.keys + (all << a.log);
        a.firsts = a.cands + (all << a.log);
        a.absent = a.firsts + all * (kBins / 2);
        a.counts = a.absent + all;
        a.moves = a.counts + bh;
        k_kv_rank<<<grid, kCutThreads, 0, s>>>(p, a);
        if (snx_launch_check("k_kv_rank")) return -1;
        k_kv_part<<<grid, kCutThreads, 0, s>>>(p, a);
        if (snx_launch_check("k_kv_part")) return -1;
        static std::atomic<uint64_t> done{0};
        if (reserve_lds(reinterpret_cast<const void*>(&k_kv_list), sizeof(uint32_t) << kMostLog, done)) return -1;
        k_kv_list<<<grid, kCutThreads, sizeof(uint32_t) << a.log, s>>>(p, a);
        if (snx_launch_check("k_kv_list")) return -1;
    } else {
        a.counts = static_cast<uint32_t*>(ws);
        a.moves = a.counts + bh;
        if (a.most <= kMoveAtOnce) return cut<true>((unsigned)bh, p, a, s);
        if (cut<false>((unsigned)bh, p, a, s)) return -1;
    }
    const size_t chunks = (size_t)a.most * (a.row_bytes / 16), gx = (chunks + 1023) / 1024;
    k_kv_move<<<dim3((unsigned)bh, (unsigned)(gx < 65536 ? gx : 65535)), 256, 0, s>>>(p, a);
    return snx_launch_check("k_kv_move");
}

}  // extern "C"
