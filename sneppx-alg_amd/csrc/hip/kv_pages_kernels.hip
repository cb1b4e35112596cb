// kv_pages_kernels.hip - which pages of the key-value cache a row has
// (include/sneppx_kv.h): SNEPPX_kv_reserve, _release and _share over refs, the number
// of rows that hold each page.  Whole numbers throughout: the results do not depend on
// the order in which threads run.
#include <hip/hip_runtime.h>

#include <cstdint>

#include "kv_pool.h"
#include "launch.h"
#include "../snx_internal.h"

using namespace snx;

namespace {

typedef int32_t i32x4 __attribute__((ext_vector_type(4)));
typedef i32x4 i32x4_any __attribute__((aligned(4)));

hipStream_t S(void* s) { return reinterpret_cast<hipStream_t>(s); }

constexpr uint32_t kMost = 0x7FFFFFFFu;              // sums of counts stay here
constexpr uint32_t kEach = 8;                        // refs of a thread in a turn
// tokens that the workgroup which takes pages places itself (16 prompts of up to 256 tokens
// 9.3 us, with a second launch 10.5; 8 of up to 2000 12.3, and 10.9)
constexpr uint32_t kWithin = 4096;

struct Pages {
    int32_t *refs, *tables, *lengths, *next_pos;
    const int32_t* counts;
    int32_t *starts, *granted, *slots, *positions;
    uint32_t pages, page_size, width, rows, tokens;
    Divider page_of;
};

__device__ __forceinline__ uint32_t length_of(const Pages& a, int32_t n) {
    const uint32_t most = a.width * a.page_size;
    return n < 0 ? 0u : (uint32_t)n < most ? (uint32_t)n : most;
}
// pages that n tokens are in
__device__ __forceinline__ uint32_t pages_of(const Pages& a, uint32_t n) { return a.page_of(n + a.page_size - 1); }

__device__ __forceinline__ uint32_t add_cut(uint32_t a, uint32_t b) { return a + b < kMost ? a + b : kMost; }

// Over a workgroup of W waves: inclusive prefixes (sums cut at kMost) of N numbers, and
// their totals.  sh: N * W words, free again after the next barrier.
template <int W, int N>
__device__ __forceinline__ void block_prefix(uint32_t (&x)[N], uint32_t* sh, uint32_t (&total)[N]) {
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
#pragma unroll
    for (int i = 0; i < N; i++) x[i] = lane_scan(x[i], 0u, add_cut);
    __syncthreads();
    if (lane == 63)
#pragma unroll
        for (int i = 0; i < N; i++) sh[i * W + w] = x[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; i++) {
        const uint32_t upto = lane_scan(lane < W ? sh[i * W + lane] : 0u, 0u, add_cut);
        total[i] = __builtin_amdgcn_readlane(upto, W - 1);
        x[i] = add_cut(w ? (uint32_t)__builtin_amdgcn_readlane(upto, w - 1) : 0u, x[i]);
    }
}
template <int W>
__device__ __forceinline__ uint32_t block_prefix(uint32_t x, uint32_t* sh, uint32_t& total) {
    uint32_t a[1] = {x}, t[1];
    block_prefix<W, 1>(a, sh, t);
    total = t[0];
    return a[0];
}

// the last of n ascending numbers (the first at most x) that is at most x: of N x at once
// (looks at LDS, each waiting for the one before)
template <int N>
__device__ __forceinline__ void last_upto(const uint32_t* at, uint32_t n, const uint32_t (&x)[N], uint32_t (&b)[N]) {
#pragma unroll
    for (int i = 0; i < N; i++) b[i] = 0;
    while (n > 1) {
        // (the upper half of an odd number has one more, and the lower is looked through as if
        // it had: what lies behind it is above x)
        const uint32_t half = n / 2;
        uint32_t seen[N];
#pragma unroll
        for (int i = 0; i < N; i++) seen[i] = at[b[i] + half];
#pragma unroll
        for (int i = 0; i < N; i++) b[i] += seen[i] <= x[i] ? half : 0;
        n -= half;
    }
}
__device__ __forceinline__ uint32_t last_upto(const uint32_t* at, uint32_t n, uint32_t x) {
    const uint32_t one[1] = {x};
    uint32_t b[1];
    last_upto<1>(at, n, one, b);
    return b[0];
}

// slot and position of token i of a row's new ones (granted: its length and next
// position before them)
__device__ __forceinline__ void place(const Pages& a, uint32_t t, uint32_t b, uint32_t i, bool ok, uint32_t len, int32_t pos) {
    int32_t slot = -1, at = -1;
    if (ok) {
        const uint32_t s = len + i, e = a.page_of(s);
        const uint32_t page = e < a.width ? (uint32_t)a.tables[(size_t)b * a.width + e] : 0xFFFFFFFFu;
        if (page < a.pages) slot = (int32_t)(page * a.page_size + (s - e * a.page_size));
        at = pos + (int32_t)i;
    }
    a.slots[t] = slot;
    if (a.positions) a.positions[t] = at;
}

// which of the thread's refs from `p` on are free pages
__device__ __forceinline__ uint32_t free_of(const Pages& a, uint32_t p) {
    uint32_t free_bits = 0;
    if (p + kEach <= a.pages) {
        i32x4_any r[kEach / 4];
#pragma unroll
        for (uint32_t k = 0; k < kEach / 4; k++) r[k] = *reinterpret_cast<const i32x4_any*>(a.refs + p + 4 * k);
#pragma unroll
        for (uint32_t k = 0; k < kEach; k++) free_bits |= (uint32_t)(r[k / 4][k % 4] == 0) << k;
    } else {
        for (uint32_t k = 0; k < kEach && p + k < a.pages; k++) free_bits |= (uint32_t)(a.refs[p + k] == 0) << k;
    }
    return free_bits;
}

// One workgroup, a row to a thread (and then the next ones): what each wants and needs, how
// far the free pages go, and then every free page of those to the row and entry that its
// number among them says.  The entries that rows need are numbered one row after the other
// and shared out among the threads, so that a few rows of many pages go as fast as many of
// one.  The first refs are asked for before all else.
// What bounds it: one load after the other (lengths, entries, new entries again) and some
// 14 barriers, 5 us for 64 rows by four waves; 11 for 48 prompts of up to 4096 tokens, of
// which a third is looking for the entries that need pages and a third giving them out.  That
// is where free pages are among the first refs.  Where they are not, as after long use, for
// the lowest free pages are the ones that go out, every call reads the refs up to the last
// page it takes twice on its one CU, first counting and then turn by turn with some five
// barriers each: behind 100000 pages in use 64 rows take 54 us in place of 7, the 48 prompts
// 33 in place of 11; behind 10000 7 and 14.
template <int W>
__global__ void __launch_bounds__(64 * W) k_kv_reserve(const Pages a) {
    constexpr uint32_t THREADS = 64 * W, TURN = kEach * THREADS;
    __shared__ uint32_t sh[3 * W], first[THREADS], entry[THREADS], need[THREADS], upto[THREADS], start[THREADS + 1];
    __shared__ uint32_t length[THREADS], found[TURN];
    __shared__ uint8_t given[THREADS];
    __shared__ int32_t next[THREADS];
    ask_for(a.tables, a.counts, a.positions, a.page_of.mul);
    const uint32_t tid = threadIdx.x, most = a.width * a.page_size;
    uint32_t carry = 0;        // tokens of the rows before
    uint32_t cursor = 0;       // no page before it is free
    bool spent = false;        // a row was left without pages

    for (uint32_t r0 = 0; r0 < a.rows; r0 += THREADS) {
        const uint32_t b = r0 + tid, rows = a.rows - r0 < THREADS ? a.rows - r0 : THREADS;
        uint32_t n = 0, want = 0, e0 = 0, span = 0;
        int32_t pos = 0;
        bool fits = false;
        const uint32_t ahead = free_of(a, cursor + kEach * tid);
        if (b < a.rows) {
            const int32_t c = a.counts ? a.counts[b] : 1;
            n = length_of(a, a.lengths[b]);
            pos = a.next_pos ? a.next_pos[b] : (int32_t)n;
            want = c < 0 ? 0u : (uint32_t)c;
            fits = want <= most - n;
            e0 = pages_of(a, n);
            span = fits ? pages_of(a, n + want) - e0 : 0;
        }
        // (a row's first entry by its own thread: a decode step needs no others)
        uint32_t own = 0xFFFFFFFFu;
        if (span) own = (uint32_t)a.tables[(size_t)b * a.width + e0];
        uint32_t sums[3] = {want, span, span > 1}, totals[3], needed;
        block_prefix<W, 3>(sums, sh, totals);
        const uint32_t tokens = totals[0], entries = totals[1];
        first[tid] = sums[1] - span;
        entry[tid] = e0;
        need[tid] = span - (own < a.pages);
        start[tid + 1] = add_cut(carry, sums[0]);
        if (tid == 0) start[0] = carry;
        length[tid] = n;
        next[tid] = pos;
        __syncthreads();
        if (b < a.rows) a.starts[b] = (int32_t)start[tid];

        // less the entries that name a page (a few, and seldom)
        // (at once, in whole passes that also bring their state back: 48 prompts of up to 600 tokens
        // 10.7 us with one, 11.1 with two, 12.2 with four; of up to 4096, with release, share
        // and the second launch before and behind it, 22.1, 20.3 and 20.3)
        constexpr int U = 2;
        for (uint32_t i0 = tid; totals[2] && i0 < entries; i0 += U * THREADS) {
            uint32_t i[U], r[U], page[U];
#pragma unroll
            for (int u = 0; u < U; u++) i[u] = i0 + u * THREADS < entries ? i0 + u * THREADS : i0;
            last_upto<U>(first, rows, i, r);
#pragma unroll
            for (int u = 0; u < U; u++) {
                const uint32_t j = i[u] - first[r[u]];
                page[u] = 0xFFFFFFFFu;
                if (j) page[u] = (uint32_t)a.tables[(size_t)(r0 + r[u]) * a.width + entry[r[u]] + j];
            }
#pragma unroll
            for (int u = 0; u < U; u++)
                if (i0 + u * THREADS < entries && page[u] < a.pages) atomicSub(&need[r[u]], 1u);
        }
        __syncthreads();
        const uint32_t mine = need[tid];
        // (with them the free pages of the first turn)
        uint32_t pair[2] = {mine, (uint32_t)__popc(ahead)}, pair_totals[2];
        block_prefix<W, 2>(pair, sh, pair_totals);
        needed = pair_totals[0];
        upto[tid] = pair[0] - mine;

        // the free pages, as far as they are needed
        uint32_t have = 0;
        if (needed && !spent) {
            have = pair_totals[1];
            for (uint32_t p0 = cursor + TURN; p0 < a.pages && have < needed; p0 += 2 * TURN) {
                uint32_t sum;
                const uint32_t p = p0 + kEach * tid;
                (void)block_prefix<W>(__popc(free_of(a, p)) + __popc(free_of(a, p + TURN)), sh, sum);
                have += sum;
            }
        }
        const bool ok = b < a.rows && fits && (mine == 0 || pair[0] <= have);
        given[tid] = ok;
        // pages that go to rows: those up to the last row whose pages are there
        uint32_t taken = needed;
        if (have < needed) {
            spent = true;
            uint32_t sum;
            (void)block_prefix<W>(ok ? mine : 0u, sh, sum);
            taken = sum;
        }
        uint32_t bits = ahead, before = pair[1] - __popc(ahead), sum = pair_totals[1];
        bool turned = false;             // beyond the first turn
        for (uint32_t done = 0; done < taken && cursor < a.pages;) {
            const uint32_t p0 = cursor + kEach * tid;
            if (turned) {
                bits = free_of(a, p0);
                before = block_prefix<W>(__popc(bits), sh, sum) - __popc(bits);
            }
            for (uint32_t i = before; bits; bits &= bits - 1) found[i++] = p0 + __builtin_ctz(bits);
            __syncthreads();
            // (all entries are chosen before any is written: of a row whose entries name
            // pages here and there, those that name none are counted)
            const uint32_t n_now = sum < taken - done ? sum : taken - done;
            uint32_t where[kEach];
#pragma unroll
            for (uint32_t q0 = 0; q0 < kEach; q0 += U) {
                if (tid + q0 * THREADS >= n_now) break;
                uint32_t k[U], r[U];
#pragma unroll
                for (uint32_t u = 0; u < U; u++) {
                    const uint32_t i = tid + (q0 + u) * THREADS;
                    k[u] = done + (i < n_now ? i : n_now - 1);
                }
                last_upto<U>(upto, rows, k, r);
#pragma unroll
                for (uint32_t u = 0; u < U; u++) {
                    const uint32_t of = r[u], j = k[u] - upto[of];
                    uint32_t e = entry[of] + j;
                    const uint32_t all = (of + 1 < rows ? first[of + 1] : entries) - first[of];
                    if (all != need[of]) {
                        // (those that earlier turns gave to the row name pages by now)
                        const int32_t* const t = a.tables + (size_t)(r0 + of) * a.width;
                        uint32_t left = done > upto[of] ? k[u] - done : j;
                        for (e = entry[of]; e + 1 < entry[of] + all && ((uint32_t)t[e] < a.pages || left--); e++) {}
                    }
                    where[q0 + u] = (r0 + of) * a.width + e;
                }
            }
            __syncthreads();
#pragma unroll
            for (uint32_t q = 0; q < kEach; q++) {
                if (tid + q * THREADS >= n_now) break;
                const uint32_t page = found[tid + q * THREADS];
                a.tables[where[q]] = (int32_t)page;
                a.refs[page] = 1;
            }
            done += sum;
            if (done > taken) break;
            cursor += TURN;                          // (all of these are taken)
            turned = true;
            __syncthreads();
        }

        if (b < a.rows) {
            const uint32_t count = ok ? want : 0;
            a.granted[b] = (int32_t)count;
            if (count) {
                a.lengths[b] = (int32_t)(n + count);
                if (a.next_pos) a.next_pos[b] = pos + (int32_t)count;
            }
        }
        __syncthreads();
        const uint32_t end = add_cut(carry, tokens);
        if (a.tokens <= kWithin)
            for (uint32_t t = carry + tid; t < end && t < a.tokens; t += THREADS) {
                const uint32_t r = last_upto(start, rows, t);
                place(a, t, r0 + r, t - start[r], given[r], length[r], next[r]);
            }
        carry = end;
        __syncthreads();
    }
    if (tid == 0) a.starts[a.rows] = (int32_t)carry;
    if (a.tokens <= kWithin)
        for (uint32_t t = carry + tid; t < a.tokens; t += THREADS) place(a, t, 0, 0, false, 0, 0);
}

// After it, for more tokens: a thread each (100 000 of them 4 us: search, lengths, entry and
// result one after the other).
__global__ void __launch_bounds__(256) k_kv_slots(const Pages a) {
    const uint32_t t = blockIdx.x * 256 + threadIdx.x;
    if (t >= a.tokens) return;
    const uint32_t* const starts = reinterpret_cast<const uint32_t*>(a.starts);
    const uint32_t b = last_upto(starts, a.rows, t);
    const uint32_t count = (uint32_t)a.granted[b];
    const bool ok = t < starts[a.rows] && count;
    uint32_t n = 0;
    int32_t pos = 0;
    if (ok) {
        n = (uint32_t)a.lengths[b] - count;
        pos = a.next_pos ? a.next_pos[b] - (int32_t)count : (int32_t)n;
    }
    place(a, t, b, t - starts[b], ok, n, pos);
}

// one less row holds a page; a count that is not above 0 stays
__device__ __forceinline__ void give_back(const Pages& a, uint32_t page) {
    if (atomicSub(&a.refs[page], 1) <= 0) atomicAdd(&a.refs[page], 1);
}

// A thread for each entry of the tables (48 rows of 512 2 us: a launch and three loads).
__global__ void __launch_bounds__(256) k_kv_release(const Pages a) {
    const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= (size_t)a.rows * a.width) return;
    const uint32_t b = (uint32_t)(i / a.width), e = (uint32_t)(i - (size_t)b * a.width);
    const uint32_t page = (uint32_t)a.tables[i];
    if (page >= a.pages || e < pages_of(a, length_of(a, a.lengths[b]))) return;
    a.tables[i] = -1;
    give_back(a, page);
}

// A workgroup for each row: its source's entries, unless that row takes some itself (3.2 us:
// sources, lengths and entries one after the other, and the atomics on shared counts).
__global__ void __launch_bounds__(256) k_kv_share(const Pages a, const int32_t* sources) {
    auto takes = [&](uint32_t b) {
        const uint32_t from = (uint32_t)sources[b];
        return from < a.rows && from != b;
    };
    const uint32_t b = blockIdx.x, from = (uint32_t)sources[b];
    if (!takes(b) || takes(from)) return;
    const int32_t c = a.counts[b];
    const uint32_t n = length_of(a, a.lengths[from]), want = c < 0 ? 0u : (uint32_t)c;
    const uint32_t k = a.page_of(want < n ? want : n);
    for (uint32_t e = threadIdx.x; e < k; e += 256) {
        const uint32_t was = (uint32_t)a.tables[(size_t)b * a.width + e];
        const int32_t page = a.tables[(size_t)from * a.width + e];
        a.tables[(size_t)b * a.width + e] = page;
        if ((uint32_t)page < a.pages) atomicAdd(&a.refs[page], 1);
        if (was < a.pages) give_back(a, was);
    }
    if (threadIdx.x == 0) {
        a.lengths[b] = (int32_t)(k * a.page_size);
        if (a.next_pos) a.next_pos[b] = (int32_t)(k * a.page_size);
    }
}

Pages pages_args(int32_t* refs, size_t pages, size_t page_size, int32_t* tables, size_t width, const int32_t* lengths,
                 int32_t* next_pos, const int32_t* counts, size_t rows) {
    Pages a = {};
    a.refs = refs;
    a.tables = tables;
    a.lengths = const_cast<int32_t*>(lengths);
    a.next_pos = next_pos;
    a.counts = counts;
    a.pages = (uint32_t)pages;
    a.page_size = (uint32_t)page_size;
    a.width = (uint32_t)width;
    a.rows = (uint32_t)rows;
    a.page_of = divider(page_size);
    return a;
}

}  // namespace

extern "C" {

int snx_k_kv_reserve(int32_t* refs, size_t pages, size_t page_size, int32_t* tables, size_t width, int32_t* lengths,
                     int32_t* next_pos, const int32_t* counts, size_t rows, int32_t* starts, int32_t* granted,
                     int32_t* slots, int32_t* positions, size_t tokens, void* st) {
    Pages a = pages_args(refs, pages, page_size, tables, width, lengths, next_pos, counts, rows);
    a.starts = starts;
    a.granted = granted;
    a.slots = slots;
    a.positions = positions;
    a.tokens = (uint32_t)tokens;
    // Four waves for what a decode step asks for (their barriers take less: 64 rows 6.7 us,
    // by sixteen 7.6, a copy of their state included), sixteen for more rows, tokens and so
    // pages (512 rows 9.1 and by four 12.4, 16 prompts of up to 256 tokens 9.3 and 11.1).
    if (rows <= 256 && tokens <= 1024) k_kv_reserve<4><<<1, 256, 0, S(st)>>>(a);
    else k_kv_reserve<16><<<1, 1024, 0, S(st)>>>(a);
    if (snx_launch_check("k_kv_reserve")) return -1;
    if (tokens <= kWithin) return 0;
    k_kv_slots<<<(unsigned)((tokens + 255) / 256), 256, 0, S(st)>>>(a);
    return snx_launch_check("k_kv_slots");
}

int snx_k_kv_release(int32_t* refs, size_t pages, size_t page_size, int32_t* tables, size_t width,
                     const int32_t* lengths, size_t rows, void* st) {
    const Pages a = pages_args(refs, pages, page_size, tables, width, lengths, nullptr, nullptr, rows);
    k_kv_release<<<(unsigned)((rows * width + 255) / 256), 256, 0, S(st)>>>(a);
    return snx_launch_check("k_kv_release");
}

int snx_k_kv_share(int32_t* refs, size_t pages, size_t page_size, int32_t* tables, size_t width, int32_t* lengths,
                   int32_t* next_pos, const int32_t* sources, const int32_t* counts, size_t rows, void* st) {
    const Pages a = pages_args(refs, pages, page_size, tables, width, lengths, next_pos, counts, rows);
    if (rows > 0xffffff) {
        snx_set_error("kv_share: %zu rows are too many", rows);
        return -1;
    }
    k_kv_share<<<(unsigned)rows, 256, 0, S(st)>>>(a, sources);
    return snx_launch_check("k_kv_share");
}

}  // extern "C"
