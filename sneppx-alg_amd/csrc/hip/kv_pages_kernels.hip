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

constexpr int kWaves = 16, kThreads = 64 * kWaves;
constexpr uint32_t kMost = 0x7FFFFFFFu;              // sums of counts stay here
constexpr uint32_t kEach = 8, kTurn = kEach * kThreads;       // refs of a thread and of all in a turn
constexpr uint32_t kWithin = 4096;                   // tokens that the workgroup which takes pages places itself

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

// Over the workgroup: inclusive prefixes of x (sums cut at kMost), and the total.
// sh: kWaves words, free again after the next barrier.
__device__ __forceinline__ uint32_t block_prefix(uint32_t x, uint32_t* sh, uint32_t& total) {
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t mine = lane_scan(x, 0u, add_cut);
    __syncthreads();
    if (lane == 63) sh[w] = mine;
    __syncthreads();
    const uint32_t upto = lane_scan(lane < kWaves ? sh[lane] : 0u, 0u, add_cut);
    total = __builtin_amdgcn_readlane(upto, kWaves - 1);
    const uint32_t before = w ? (uint32_t)__builtin_amdgcn_readlane(upto, w - 1) : 0u;
    return add_cut(before, mine);
}

// the last of n ascending numbers (the first at most x) that is at most x
__device__ __forceinline__ uint32_t last_upto(const uint32_t* at, uint32_t n, uint32_t x) {
    uint32_t b = 0;
    while (n > 1) {
        const uint32_t half = n / 2;
        const bool up = at[b + half] <= x;
        b += up ? half : 0;
        n = up ? n - half : half;
    }
    return b;
}

// slot and position of token i of a row's new ones (granted: its length and next
// position before them)
__device__ __forceinline__ void place(const Pages& a, uint32_t t, uint32_t b, uint32_t i, bool ok, uint32_t len, int32_t pos) {
    int32_t slot = -1, at = -1;
    if (ok) {
        const uint32_t s = len + i, e = a.page_of(s);
        const uint32_t page = (uint32_t)a.tables[(size_t)b * a.width + e];
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

// One workgroup, 1024 rows at a time: what each wants and needs, how far the free
// pages go, and then every free page of those to the row and entry that its number
// among them says.  The entries that rows need are numbered one row after the other and
// shared out among the threads, so that a few rows of many pages go as fast as many
// of one.
// What bounds it: one load after the other (lengths, entries, refs), and for pools
// with few free pages the refs up to the last one taken, at the rate of one CU.
__global__ void __launch_bounds__(kThreads) k_kv_reserve(const Pages a) {
    __shared__ uint32_t sh[kWaves], first[kThreads], entry[kThreads], need[kThreads], upto[kThreads], start[kThreads + 1];
    __shared__ uint32_t length[kThreads], found[kTurn];
    __shared__ uint8_t given[kThreads];
    __shared__ int32_t next[kThreads];
    const uint32_t tid = threadIdx.x, most = a.width * a.page_size;
    uint32_t carry = 0;        // tokens of the rows before
    uint32_t cursor = 0;       // no page before it is free
    bool spent = false;        // a row was left without pages

    for (uint32_t r0 = 0; r0 < a.rows; r0 += kThreads) {
        const uint32_t b = r0 + tid, rows = a.rows - r0 < kThreads ? a.rows - r0 : kThreads;
        uint32_t n = 0, want = 0, e0 = 0, span = 0;
        int32_t pos = 0;
        bool fits = false;
        if (b < a.rows) {
            const int32_t c = a.counts ? a.counts[b] : 1;
            n = length_of(a, a.lengths[b]);
            pos = a.next_pos ? a.next_pos[b] : (int32_t)n;
            want = c < 0 ? 0u : (uint32_t)c;
            fits = want <= most - n;
            e0 = pages_of(a, n);
            span = fits ? pages_of(a, n + want) - e0 : 0;
        }
        uint32_t tokens, entries, needed;
        const uint32_t tokens_upto = block_prefix(want, sh, tokens), entries_upto = block_prefix(span, sh, entries);
        first[tid] = entries_upto - span;
        entry[tid] = e0;
        need[tid] = 0;
        start[tid + 1] = add_cut(carry, tokens_upto);
        if (tid == 0) start[0] = carry;
        length[tid] = n;
        next[tid] = pos;
        __syncthreads();
        if (b < a.rows) a.starts[b] = (int32_t)start[tid];

        // entries that name no page
        for (uint32_t i = tid; i < entries; i += kThreads) {
            const uint32_t r = last_upto(first, rows, i);
            const uint32_t page = (uint32_t)a.tables[(size_t)(r0 + r) * a.width + entry[r] + (i - first[r])];
            if (page >= a.pages) atomicAdd(&need[r], 1u);
        }
        __syncthreads();
        const uint32_t mine = need[tid], mine_upto = block_prefix(mine, sh, needed);
        upto[tid] = mine_upto - mine;

        // the free pages, as far as they are needed
        uint32_t have = 0;
        if (needed && !spent)
            for (uint32_t p0 = cursor; p0 < a.pages && have < needed; p0 += 2 * kTurn) {
                uint32_t sum;
                const uint32_t p = p0 + kEach * tid;
                (void)block_prefix(__popc(free_of(a, p)) + __popc(free_of(a, p + kTurn)), sh, sum);
                have += sum;
            }
        const bool ok = b < a.rows && fits && (mine == 0 || mine_upto <= have);
        given[tid] = ok;
        __syncthreads();
        // pages that go to rows: those up to the last row whose pages are there
        uint32_t taken = needed;
        if (have < needed) {
            spent = true;
            uint32_t sum;
            (void)block_prefix(ok ? mine : 0u, sh, sum);
            taken = sum;
        }
        for (uint32_t done = 0; done < taken && cursor < a.pages;) {
            const uint32_t p0 = cursor + kEach * tid;
            uint32_t bits = free_of(a, p0), sum;
            uint32_t i = block_prefix(__popc(bits), sh, sum) - __popc(bits);
            for (; bits; bits &= bits - 1) found[i++] = p0 + __builtin_ctz(bits);
            __syncthreads();
            // (all entries are chosen before any is written: of a row whose entries name
            // pages here and there, those that name none are counted)
            const uint32_t n_now = sum < taken - done ? sum : taken - done;
            uint32_t where[kEach];
#pragma unroll
            for (uint32_t q = 0; q < kEach; q++) {
                const uint32_t k = done + tid + q * kThreads;
                if (tid + q * kThreads >= n_now) break;
                const uint32_t r = last_upto(upto, rows, k), j = k - upto[r];
                uint32_t e = entry[r] + j;
                const uint32_t all = (r + 1 < rows ? first[r + 1] : entries) - first[r];
                if (all != need[r]) {
                    // (those that earlier turns gave to the row name pages by now)
                    const int32_t* const t = a.tables + (size_t)(r0 + r) * a.width;
                    uint32_t left = done > upto[r] ? k - done : j;
                    for (e = entry[r]; e + 1 < entry[r] + all && ((uint32_t)t[e] < a.pages || left--); e++) {}
                }
                where[q] = (r0 + r) * a.width + e;
            }
            __syncthreads();
#pragma unroll
            for (uint32_t q = 0; q < kEach; q++) {
                if (tid + q * kThreads >= n_now) break;
                const uint32_t page = found[tid + q * kThreads];
                a.tables[where[q]] = (int32_t)page;
                a.refs[page] = 1;
            }
            done += sum;
            if (done <= taken) cursor += kTurn;      // (all of these are taken)
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
        const uint32_t end = add_cut(carry, tokens);
        if (a.tokens <= kWithin)
            for (uint32_t t = carry + tid; t < end && t < a.tokens; t += kThreads) {
                const uint32_t r = last_upto(start, rows, t);
                place(a, t, r0 + r, t - start[r], given[r], length[r], next[r]);
            }
        carry = end;
        __syncthreads();
    }
    if (tid == 0) a.starts[a.rows] = (int32_t)carry;
    if (a.tokens <= kWithin)
        for (uint32_t t = carry + tid; t < a.tokens; t += kThreads) place(a, t, 0, 0, false, 0, 0);
}

// After it, for more tokens: a thread each.
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

// A thread for each entry of the tables.
__global__ void __launch_bounds__(256) k_kv_release(const Pages a) {
    const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= (size_t)a.rows * a.width) return;
    const uint32_t b = (uint32_t)(i / a.width), e = (uint32_t)(i - (size_t)b * a.width);
    const uint32_t page = (uint32_t)a.tables[i];
    if (page >= a.pages || e < pages_of(a, length_of(a, a.lengths[b]))) return;
    a.tables[i] = -1;
    give_back(a, page);
}

// A workgroup for each row: its source's entries, unless that row takes some itself.
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
    k_kv_reserve<<<1, kThreads, 0, S(st)>>>(a);
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
