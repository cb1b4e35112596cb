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
#pragma unroll
        for (int o = LR / 2; o > 0; o >>= 1) m = nanless_max(m, __shfl_xor(m, o));
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
constexpr int kPasses = 4;               // digits of 9, 8, 8 and 7 bits: sign and exponent first
constexpr int kShift[kPasses] = {23, 15, 7, 0}, kBins[kPasses] = {512, 256, 256, 256};
constexpr uint32_t kSome = 4096;         // keys that share the first digit and are kept apart
constexpr uint32_t kMoveAtOnce = 64;     // moves that the workgroup which finds them makes itself

// two counts per wave -> their exclusive prefixes over the waves, and the totals
__device__ __forceinline__ void wave_prefix(uint32_t& x, uint32_t& y, uint2* sh, uint2& total) {
    const int w = threadIdx.x >> 6;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh[w] = make_uint2(x, y);
    __syncthreads();
    x = y = 0;
    total = make_uint2(0, 0);
#pragma unroll
    for (int i = 0; i < kCutWaves; i++) {
        const uint2 v = sh[i];
        if (i < w) {
            x += v.x;
            y += v.y;
        }
        total.x += v.x;
        total.y += v.y;
    }
}

// rows of the pool (k, v and the planes) of slots of[i] to those of slots
// to[i], for `n` moves, by `threads` threads of which this is `me`
__device__ __forceinline__ void move_rows(const KVPool& p, uint32_t b, uint32_t h, uint32_t row_bytes,
                                          const uint32_t* to, const uint32_t* of, uint32_t n, uint32_t me,
                                          uint32_t threads) {
    const uint32_t per = row_bytes / 16, chunks = n * per;
    constexpr int U = 4;
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

struct Cut {
    const int32_t *lengths, *next_pos;
    int32_t* new_lengths;
    uint32_t max_length, budget, recent, most, row_bytes;
    uint32_t* counts;          // [rows * heads] moves of each row and head (unless moved at once)
    uint32_t* moves;           // [rows * heads][2][most] slots: targets, then sources
    uint32_t* keys;            // [rows * heads][max_length] where they do not fit in LDS
};

// One workgroup per (row, head): the budget-th largest key by its digits from
// the top (each time a histogram of the keys that agree with the digits found
// so far, read by every wave for itself), then the free slots below the budget
// and the kept ones from it on, both in ascending order.  Each wave has
// consecutive slots, so that order by (wave, step, lane) is order by slot.
// KEYS: up to 4 of each thread in registers (16 x 8 of 2049 slots: 8.5 us, in LDS
// 10.5), up to 32 in LDS, else in a workspace.  MOVE: with so few moves that the
// workgroup makes them at once.
enum { kRegisters, kLds, kWorkspace };
template <int KEYS, bool MOVE>
__global__ void __launch_bounds__(kCutThreads) k_kv_cut(const KVPool p, const Cut a) {
    // most keys share a few exponents: with many, the first histogram is in copies
    constexpr int kCopies = KEYS == kRegisters ? 1 : 4;
    constexpr int kHist = kCopies * kBins[0] + kBins[1] + kBins[2] + kBins[3];
    extern __shared__ uint32_t near_keys[];
    __shared__ __attribute__((aligned(16))) uint32_t hist[kHist];
    __shared__ uint32_t some[KEYS == kRegisters ? 1 : kSome], some_n;
    __shared__ uint2 sh[kCutWaves];
    __shared__ uint32_t list[MOVE ? 2 * kMoveAtOnce : 1];
    const uint32_t b = blockIdx.x / p.heads, h = blockIdx.x - b * p.heads;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t L = kv_length(a.lengths, b, a.max_length), budget = a.budget;
    const uint32_t steps = (L + 4 * kCutThreads - 1) / (4 * kCutThreads) * 4;       // slots of a thread, by fours
    const uint32_t w0 = wave * steps * 64, t0 = w0 + lane;
    uint32_t* const keys = KEYS == kLds ? near_keys : a.keys + (size_t)blockIdx.x * a.max_length;

    for (int i = tid; i < kHist; i += kCutThreads) hist[i] = 0;
    if (tid == 0) some_n = 0;
    bool gone = false;
    uint32_t own_keys[4];
    if (L > budget) {
        const int64_t from64 = (int64_t)a.next_pos[b] - (int64_t)a.recent;
        const int32_t from = (int32_t)(from64 < INT32_MIN ? INT32_MIN : from64);
        // G slots at once (past the length: its last one), so that their look-ups
        // and loads are in flight together; key 0 past the length
        constexpr int G = KEYS == kRegisters ? 4 : 8;
        for (uint32_t i0 = 0; i0 < (KEYS == kRegisters ? 4 : steps); i0 += G) {
            uint32_t rows[G];
            float w[G];
            int32_t pos[G];
#pragma unroll
            for (int i = 0; i < G; i++) {
                const uint32_t t = t0 + 64 * (i0 + i);
                const bool there = p.row(b, h, t < L ? t : L - 1, rows[i]);
                gone |= !there;
                if (!there) rows[i] = 0;
            }
#pragma unroll
            for (int i = 0; i < G; i++) {
                w[i] = p.weights[rows[i]];
                pos[i] = p.positions[rows[i]];
            }
#pragma unroll
            for (int i = 0; i < G; i++) {
                const uint32_t t = t0 + 64 * (i0 + i), q = t < L ? rank_key(w[i], pos[i], from) : 0u;
                if (KEYS == kRegisters) own_keys[i & 3] = q;
                else if (i0 + i < steps && (KEYS == kLds || t < L)) keys[t] = q;
            }
        }
    }
    gone = __syncthreads_or(gone);
    if (tid == 0 && h == 0 && a.new_lengths) a.new_lengths[b] = (int32_t)(L > budget && !gone ? budget : L);
    if (L <= budget || gone) {
        if (!MOVE && tid == 0) a.counts[blockIdx.x] = 0;
        return;
    }
    // Slots past the length have the lowest key and come after all others: no
    // test keeps them out below.  (Keys are read by the thread that wrote them.)
    auto each_of = [&](uint32_t i0, uint32_t end, auto f) {
        for (uint32_t i = i0; i < (KEYS == kRegisters ? 4 : end); i += 4) {
            uint32_t q[4];
#pragma unroll
            for (int u = 0; u < 4; u++) {
                const uint32_t t = t0 + 64 * (i + u);
                q[u] = KEYS == kRegisters ? own_keys[u] : KEYS == kLds || t < L ? keys[t] : 0u;
            }
#pragma unroll
            for (int u = 0; u < 4; u++) f(i + u, q[u]);
        }
    };
    auto each = [&](auto f) { each_of(0, steps, f); };

    auto lane_rank = [&](uint64_t m) {
        return __builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0));
    };

    uint32_t prefix = 0, want = budget, tied = 0;    // the want-th largest of the `tied` keys that share the prefix
    bool few = false;                                // these are in `some`
    uint32_t* hp = hist;
#pragma unroll
    for (int pass = 0; pass < kPasses; pass++) {
        if (want == tied) break;                     // all of them stay, whatever their other digits are
        const int shift = kShift[pass], bins = kBins[pass], width = pass == 0 ? 9 : pass == 3 ? 7 : 8;
        const uint32_t digits = (1u << width) - 1u, above_shift = (shift + width) & 31;
        // One pass over all keys puts those that are left aside, if there is room
        // (16 of 30001 slots: 39 -> 31 us).
        if (KEYS != kRegisters && pass == 1 && tied <= kSome) {
            few = true;
            uint32_t own = 0;
            each([&](uint32_t, uint32_t q) { own += __popcll(__ballot(q >> above_shift == prefix >> above_shift)); });
            uint32_t at = 0;
            if (lane == 0) at = atomicAdd(&some_n, own);
            at = __builtin_amdgcn_readfirstlane(at);
            each([&](uint32_t, uint32_t q) {
                const uint64_t who = __ballot(q >> above_shift == prefix >> above_shift);
                if (who >> lane & 1) some[at + lane_rank(who)] = q;
                at += __popcll(who);
            });
            __syncthreads();
        }
        if (few) {
            for (uint32_t i = tid; i < kSome && i < some_n; i += kCutThreads) {
                const uint32_t q = some[i];
                if (q >> above_shift == prefix >> above_shift) atomicAdd(&hp[(q >> shift) & digits], 1u);
            }
        } else {
            each([&](uint32_t, uint32_t q) {
                const uint32_t digit = (q >> shift) & digits;
                const uint32_t to = pass == 0 ? digit * kCopies + lane % kCopies : digit;
                const uint64_t who = pass == 0 ? ~0ull : __ballot(q >> above_shift == prefix >> above_shift);
                if (who == 0) return;
                // many alike (zeros, recent ones) are counted at once
                if (who == ~0ull && __ballot(digit != (uint32_t)__builtin_amdgcn_readfirstlane(digit)) == 0) {
                    if (lane == 0) atomicAdd(&hp[to], 64u);
                } else if (who >> lane & 1) {
                    atomicAdd(&hp[to], 1u);
                }
            });
        }
        __syncthreads();
        // from the top: lane i has the i-th bins / 64 of them, the last the highest
        constexpr int most = 8;
        uint32_t n[most];
        const int per = bins / 64;
        uint32_t sum = 0;
        if (pass == 0 && kCopies == 4) {             // a bin's copies at once
#pragma unroll
            for (int j = 0; j < per; j++) {
                const u32x4 v = *reinterpret_cast<const u32x4*>(hp + 4 * (bins - per * (lane + 1) + j));
                n[j] = v[0] + v[1] + v[2] + v[3];
                sum += n[j];
            }
        } else {
#pragma unroll
            for (int j = 0; j < per; j += 4) {
                const u32x4 v = *reinterpret_cast<const u32x4*>(hp + bins - per * (lane + 1) + j);
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    n[j + e] = v[e];
                    sum += v[e];
                }
            }
        }
        const uint32_t upto = lane_prefix(sum);
        uint32_t above = upto - sum, digit = 0, count = 0, rest = 0;
        const uint64_t mine = __ballot(above < want && want <= upto);
#pragma unroll
        for (int j = per - 1; j >= 0; j--) {
            if (above < want && want <= above + n[j]) {
                digit = bins - per * (lane + 1) + j;
                rest = want - above;
                count = n[j];
            }
            above += n[j];
        }
        const int at = __builtin_ctzll(mine);
        prefix |= (uint32_t)__builtin_amdgcn_readlane(digit, at) << shift;
        want = __builtin_amdgcn_readlane(rest, at);
        tied = __builtin_amdgcn_readlane(count, at);
        hp += pass == 0 ? kCopies * bins : bins;
    }

    // of the keys equal to the threshold the first `want` stay
    uint2 total;
    uint32_t ties = 0, none = 0;
    if (want < tied) {
        each([&](uint32_t, uint32_t q) { ties += __popcll(__ballot(q == prefix)); });
        wave_prefix(ties, none, sh, total);
    }
    uint32_t seen = ties;
    // lanes whose slot stays
    const bool ranked = want < tied;
    auto stay = [&](uint32_t q) -> uint64_t {
        if (!ranked) return __ballot(q >= prefix);
        const uint64_t tb = __ballot(q == prefix);
        const uint64_t s = __ballot(q > prefix || (q == prefix && seen + lane_rank(tb) < want));
        seen += __popcll(tb);
        return s;
    };
    // Up to 64 steps from i0 at once, lane i with step i0 + i: the slots below the
    // budget that are left free, those from it on that stay, and the numbers of
    // both before them in the block (the latter in the upper half).
    auto block = [&](uint32_t i0, uint64_t& hole, uint64_t& far) {
        uint32_t lo = 0, hi = 0;
        each_of(i0, i0 + 64 < steps ? i0 + 64 : steps, [&](uint32_t i, uint32_t q) {
            const uint64_t s = stay(q);
            const bool me = (uint32_t)lane == i - i0;
            lo = me ? (uint32_t)s : lo;
            hi = me ? (uint32_t)(s >> 32) : hi;
        });
        const uint64_t s = (uint64_t)hi << 32 | lo;
        const uint32_t at = w0 + 64 * (i0 + lane);
        const uint64_t part = ((uint64_t)1 << ((budget - at) & 63)) - 1;
        const uint64_t low = i0 + lane >= steps || at >= budget ? 0 : budget - at >= 64 ? ~0ull : part;
        hole = low & ~s;
        far = s & ~low;
    };
    uint32_t holes = 0, fars = 0;
    uint64_t hole, far;
    for (uint32_t i0 = 0; i0 < steps; i0 += 64) {
        block(i0, hole, far);
        const uint32_t sum = __builtin_amdgcn_readlane(lane_prefix(__popcll(hole) | __popcll(far) << 16), 63);
        holes += sum & 0xFFFF;
        fars += sum >> 16;
    }
    wave_prefix(holes, fars, sh, total);
    seen = ties;
    uint32_t* const to = MOVE ? list : a.moves + (size_t)blockIdx.x * 2 * a.most;
    uint32_t* const of = to + (MOVE ? kMoveAtOnce : a.most);
    for (uint32_t i0 = 0; i0 < steps; i0 += 64) {
        if (KEYS == kWorkspace && steps > 64) block(i0, hole, far);      // (else it is the one above)
        const uint32_t own = __popcll(hole) | __popcll(far) << 16, upto = lane_prefix(own), before = upto - own;
        const uint32_t end = i0 + 64 < steps ? 64 : steps - i0;
        for (uint32_t i = 0; i < end; i++) {
            const uint32_t t = t0 + 64 * (i0 + i), before_i = __builtin_amdgcn_readlane(before, i);
            auto write = [&](uint64_t mine, uint32_t* to, uint32_t at) {
                const uint64_t m = (uint64_t)__builtin_amdgcn_readlane((uint32_t)(mine >> 32), i) << 32 |
                                   (uint32_t)__builtin_amdgcn_readlane((uint32_t)mine, i);
                if (m >> lane & 1) to[at + lane_rank(m)] = t;
            };
            // a step lies below the budget, or from it on, or has it within
            if (w0 + 64 * (i0 + i) < budget) write(hole, to, holes + (before_i & 0xFFFF));
            if (w0 + 64 * (i0 + i) + 64 > budget) write(far, of, fars + (before_i >> 16));
        }
        const uint32_t sum = __builtin_amdgcn_readlane(upto, 63);
        holes += sum & 0xFFFF;
        fars += sum >> 16;
    }
    if (MOVE) {
        __syncthreads();
        move_rows(p, b, h, a.row_bytes, to, of, total.x, tid, kCutThreads);
    } else if (tid == 0) {
        a.counts[blockIdx.x] = total.x;
    }
}

// The moves that k_kv_cut listed.  Sources lie in slots from the budget on and
// targets below it, so all are independent.
__global__ void __launch_bounds__(256) k_kv_move(const KVPool p, const Cut a, uint32_t first) {
    const uint32_t bh = first + blockIdx.y, b = bh / p.heads, n = a.counts[bh];
    const uint32_t* to = a.moves + (size_t)bh * 2 * a.most;
    move_rows(p, b, bh - b * p.heads, a.row_bytes, to, to + a.most, n, blockIdx.x * 256 + threadIdx.x, gridDim.x * 256);
}

template <int LR>
void append(bool i8, unsigned blocks, const KVPool& p, const NewRows& n, hipStream_t s) {
    if (i8) k_kv_append<true, LR><<<blocks, 256, 0, s>>>(p, n);
    else k_kv_append<false, LR><<<blocks, 256, 0, s>>>(p, n);
}

template <int KEYS, bool MOVE>
int cut(unsigned blocks, const KVPool& p, const Cut& a, hipStream_t s) {
    constexpr uint32_t four = 4 * kCutThreads;
    const int bytes = KEYS == kLds ? (int)((a.max_length + four - 1) / four * four * sizeof(uint32_t)) : 0;
    static std::atomic<uint64_t> done{0};
    const void* fn = reinterpret_cast<const void*>(&k_kv_cut<KEYS, MOVE>);
    if (bytes && lds_optin(fn, 8 * four * sizeof(uint32_t), done) != hipSuccess) {
        snx_set_error("kv_evict: cannot reserve %d bytes of LDS", bytes);
        return -1;
    }
    k_kv_cut<KEYS, MOVE><<<blocks, kCutThreads, bytes, s>>>(p, a);
    return snx_launch_check("k_kv_cut");
}
template <int KEYS>
int cut(bool at_once, unsigned blocks, const KVPool& p, const Cut& a, hipStream_t s) {
    return at_once ? cut<KEYS, true>(blocks, p, a, s) : cut<KEYS, false>(blocks, p, a, s);
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

// keys that do not fit in the LDS of a workgroup
static bool keys_far(size_t max_length) { return max_length > 32 * (size_t)kCutThreads; }

size_t snx_kv_evict_ws(const SNEPPXKVCache* c, size_t rows, size_t max_length, size_t budget) {
    const size_t most = most_moves(max_length, budget), bh = rows * c->kv_heads;
    return bh * sizeof(uint32_t) *
           ((most > kMoveAtOnce ? 1 + 2 * most : 0) + (keys_far(max_length) && most ? max_length : 0));
}

int snx_k_kv_evict(const SNEPPXKVCache* c, const int32_t* tables, size_t width, const int32_t* lengths,
                   const int32_t* next_pos, int32_t* new_lengths, size_t rows, size_t max_length, size_t budget,
                   size_t recent, void* ws, void* st) {
    const KVPool p = kv_pool(c, tables, width);
    const size_t bh = rows * c->kv_heads;
    Cut a;
    a.lengths = lengths;
    a.next_pos = next_pos;
    a.new_lengths = new_lengths;
    a.max_length = (uint32_t)max_length;
    a.budget = (uint32_t)budget;
    a.recent = (uint32_t)(recent < INT32_MAX ? recent : INT32_MAX);
    a.most = most_moves(max_length, budget);
    a.row_bytes = (uint32_t)(c->head_dim * (c->dtype == SNEPPX_INT8 ? 1 : 2));
    const bool at_once = a.most <= kMoveAtOnce;
    a.counts = static_cast<uint32_t*>(ws);
    a.moves = a.counts + bh;
    a.keys = at_once ? a.counts : a.moves + bh * 2 * a.most;
    const int rc = !a.most || max_length <= 4 * (size_t)kCutThreads ? cut<kRegisters>(at_once, (unsigned)bh, p, a, S(st))
                   : !keys_far(max_length)                          ? cut<kLds>(at_once, (unsigned)bh, p, a, S(st))
                                                                    : cut<kWorkspace>(at_once, (unsigned)bh, p, a, S(st));
    if (rc) return -1;
    if (at_once) return 0;
    const size_t chunks = (size_t)a.most * (a.row_bytes / 16), gx = (chunks + 1023) / 1024;
    for (size_t at = 0; at < bh; at += 65535) {
        const size_t n = bh - at < 65535 ? bh - at : 65535;
        k_kv_move<<<dim3((unsigned)(gx < 65536 ? gx : 65536), (unsigned)n), 256, 0, S(st)>>>(p, a, (uint32_t)at);
        if (snx_launch_check("k_kv_move")) return -1;
    }
    return 0;
}

}  // extern "C"
