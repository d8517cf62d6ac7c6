// Paged KV cache (sm_100a): storing rows, and the calls that change which
// sequence has which pages. The attention is in paged_attn.cu.
//
// The reference keeps one region of its whole context per process
// (src/brain_runtime.c:2019-2020). Here sequences of different lengths share a
// pool of pages, and one page may be part of several of them.
#include <algorithm>
#include <atomic>
#include <utility>
#include <cuda.h>
#include "../../include/atlas_cuda.h"
#include "paged.cuh"

namespace atlas {

int api_fail(int code, const char *fmt, ...);
int api_device(int device, int *sms);

namespace paged {

using k8::launch;
using k8::wait_predecessor;

// paged_attn.cu
cudaError_t launch_few(const AttnArgs &a, const CUtensorMap &kmap, const CUtensorMap &vmap, bool bf, int nt, int dev, int sms,
                       cudaStream_t stream);
// paged_prompt.cu
cudaError_t launch_prompt(const AttnArgs &a, const CUtensorMap &kmap, const CUtensorMap &vmap, const CUtensorMap &qmap, bool bf, uint32_t tiles, int dev,
                          int sms, cudaStream_t stream);

namespace {

// --------------------------------------------------------------- append ----
//
// Rows of 256 bytes from [seq][token][kv_head] to their places: sixteen threads
// a row, one thread for 16 bytes of K and of V. Nothing is computed; bound by
// HBM and the reads of L2 before the first store for prompts (1024 bytes per token
// and KV head; 8192 tokens of 8 heads 13.8 us, 4.9 TB/s), by the launch for single
// tokens (1.7 us).

struct AppendArgs {
    Cache c;
    Rows r;
    const uint16_t *k, *v;    // [seq][tokens][kv_heads][128], ld elements between tokens
    uint64_t ld;
    uint32_t layer, early;
};

// Rows (token, head) of a sequence that 16 threads take: 8192 tokens of 8 heads take 13.8 us; with 1 or 4 rows 16.4 or 16.2
constexpr uint32_t kAppendThreads = 256, kAppendRows = 2;

// Through L2, whose lines of it go first: a row is read once, and the pages should stay (without that 14.7 us instead of 13.8)
__device__ __forceinline__ uint4 load_once(const uint4 *p, uint64_t policy)
{
    uint4 x;
    asm volatile("ld.global.cg.L2::cache_hint.v4.u32 {%0, %1, %2, %3}, [%4], %5;"
                 : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w)
                 : "l"(p), "l"(policy)
                 : "memory");
    return x;
}

__global__ void __launch_bounds__(kAppendThreads) append_kernel(const __grid_constant__ AppendArgs a)
{
    const uint32_t s = blockIdx.y, part = threadIdx.x & 15u;
    wait_predecessor(a.early);
    const uint64_t p0 = __ldcg(a.r.pos0 + s);
    const uint64_t rows = (uint64_t)row_count(a.r, s) * a.c.kv_heads;
    const uint64_t row0 = (uint64_t)blockIdx.x * (kAppendThreads / 16u * kAppendRows) + (threadIdx.x >> 4);
    uint4 k[kAppendRows], v[kAppendRows];
    uint64_t to[kAppendRows];
    uint32_t e[kAppendRows];
    const uint64_t once = policy_evict_first();
    // the rows are on their way while their pages are looked up
#pragma unroll
    for (uint32_t i = 0; i < kAppendRows; ++i) {
        const uint64_t row = row0 + i * (kAppendThreads / 16u);
        e[i] = ~0u;
        to[i] = 0u;
        if (row >= rows) continue;
        const uint32_t t = (uint32_t)(row / a.c.kv_heads), h = (uint32_t)(row - (uint64_t)t * a.c.kv_heads);
        const size_t from = ((size_t)s * a.r.tokens + t) * a.ld + (size_t)h * kDim;
        k[i] = load_once(reinterpret_cast<const uint4 *>(a.k + from) + part, once);
        v[i] = load_once(reinterpret_cast<const uint4 *>(a.v + from) + part, once);
        const uint64_t p = p0 + t;
        if (p >= a.c.limit) continue;
        e[i] = (uint32_t)__ldcg(a.c.table + (size_t)s * a.c.max_pages + (p >> a.c.page_log2));
        to[i] = ((((uint64_t)a.layer * a.c.pages * a.c.kv_heads + h) << a.c.page_log2) + (p & ((1u << a.c.page_log2) - 1u))) * 16u + part;
    }
#pragma unroll
    for (uint32_t i = 0; i < kAppendRows; ++i) {
        // a page that other sequences have too is not written to
        if (e[i] < a.c.pages && __ldcg(a.c.refs + e[i]) <= 1) to[i] += ((uint64_t)e[i] * a.c.kv_heads << a.c.page_log2) * 16u;
        else to[i] = ~0ull;
    }
#pragma unroll
    for (uint32_t i = 0; i < kAppendRows; ++i)
        if (to[i] != ~0ull) {
            reinterpret_cast<uint4 *>(a.c.k)[to[i]] = k[i];
            reinterpret_cast<uint4 *>(a.c.v)[to[i]] = v[i];
        }
}

// ----------------------------------------------------------------- fork ----
//
// New entry (s, j) is the old entry (parent[s], j): column j of the table needs
// nothing but itself, so a CTA reads its columns whole before it writes them,
// and one launch suffices. The counts change by atomic additions of integers:
// their order does not show. Bound by
// latency: two dependent reads of L2.

struct ForkArgs {
    Cache c;
    const int32_t *parent;
    const uint32_t *length, *first;
    uint32_t early;
};

constexpr uint32_t kForkColumns = 8, kForkThreads = 256;

__global__ void __launch_bounds__(kForkThreads) fork_kernel(const __grid_constant__ ForkArgs a)
{
    extern __shared__ uint32_t was[];   // [nseq][kForkColumns]
    wait_predecessor(a.early);
    const uint32_t j = blockIdx.x * kForkColumns + threadIdx.x % kForkColumns, s0 = threadIdx.x / kForkColumns;
    const bool there = j < a.c.max_pages;
    for (uint32_t s = s0; s < a.c.nseq; s += kForkThreads / kForkColumns)
        was[s * kForkColumns + threadIdx.x % kForkColumns] = there ? (uint32_t)__ldcg(a.c.table + (size_t)s * a.c.max_pages + j) : ~0u;
    __syncthreads();
    if (!there) return;
    for (uint32_t s = s0; s < a.c.nseq; s += kForkThreads / kForkColumns) {
        const uint32_t parent = (uint32_t)__ldcg(a.parent + s), old = was[s * kForkColumns + threadIdx.x % kForkColumns];
        const uint64_t begin = (uint64_t)j << a.c.page_log2, end = begin + (1u << a.c.page_log2);
        uint32_t now = ~0u;
        if (parent < a.c.nseq && begin < __ldcg(a.length + s) && (!a.first || end > __ldcg(a.first + s)))
            now = was[parent * kForkColumns + threadIdx.x % kForkColumns];
        if (now >= a.c.pages) now = ~0u;
        if (now == old) continue;
        a.c.table[(size_t)s * a.c.max_pages + j] = (int32_t)now;
        if (old < a.c.pages) atomicSub(a.c.refs + old, 1);
        if (now < a.c.pages) atomicAdd(a.c.refs + now, 1);
    }
}

// ---------------------------------------------- which pages: one CTA plans ----

constexpr uint32_t kPlanThreads = 1024, kPlanWarps = kPlanThreads / 32;

struct PlanArgs {
    Cache c;
    Rows r;
    uint32_t *out;                        // pages lacking (reserve), pages in use (compact)
    uint32_t early;
};

__device__ __forceinline__ WorkHead *head_of(const Cache &c) { return reinterpret_cast<WorkHead *>(c.work); }
__device__ __forceinline__ uint32_t *array_of(const Cache &c, WorkArray i)
{
    return c.work + sizeof(WorkHead) / 4u + (size_t)i * c.pages;
}

struct Scan {
    uint32_t warp[2][kPlanWarps];
};

// The sum of x over the threads before this one; `all`: over all threads. `turn` alternates between two calls.
__device__ __forceinline__ uint32_t scan_all(Scan &sm, uint32_t &turn, uint32_t x, uint32_t &all)
{
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
    uint32_t inc = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t up = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= (uint32_t)o) inc += up;
    }
    turn ^= 1u;
    if (lane == 31u) sm.warp[turn][warp] = inc;
    __syncthreads();
    uint32_t w = sm.warp[turn][lane];     // 32 warps
    all = __reduce_add_sync(0xffffffffu, w);
    w = lane < warp ? w : 0u;
    return inc - x + __reduce_add_sync(0xffffffffu, w);
}

constexpr uint32_t kPlanPages = 16;       // pages that a thread looks at at a time

// Bit i: page p0 + i is in use (i < kPlanPages); pages behind the last one are neither
__device__ __forceinline__ uint32_t used_mask(const Cache &c, uint32_t p0, uint32_t &exist)
{
    uint32_t m = 0u;
    exist = p0 >= c.pages ? 0u : c.pages - p0 >= kPlanPages ? (1u << kPlanPages) - 1u : (1u << (c.pages - p0)) - 1u;
#pragma unroll
    for (uint32_t i = 0; i < kPlanPages; i += 4u) {
        if (p0 + i + 4u <= c.pages) {
            const int4 x = __ldcg(reinterpret_cast<const int4 *>(c.refs + p0 + i));
            m |= ((x.x > 0 ? 1u : 0u) | (x.y > 0 ? 2u : 0u) | (x.z > 0 ? 4u : 0u) | (x.w > 0 ? 8u : 0u)) << i;
        } else {
            for (uint32_t k = i; k < i + 4u; ++k)
                if (p0 + k < c.pages && __ldcg(c.refs + p0 + k) > 0) m |= 1u << k;
        }
    }
    return m;
}

// The first `want` free pages, ascending, into `list`; how many there are (up to want). All threads. `free0`: this thread's
// of the first kPlanThreads * kPlanPages pages.
__device__ __forceinline__ uint32_t find_free(const Cache &c, Scan &sm, uint32_t &turn, uint32_t free0, uint32_t want, uint32_t *list)
{
    uint32_t found = 0u;
    for (uint32_t b = 0; b < c.pages && found < want; b += kPlanThreads * kPlanPages) {
        const uint32_t p0 = b + threadIdx.x * kPlanPages;
        uint32_t exist, all, m = free0;
        if (b) {
            m = used_mask(c, p0, exist);
            m = exist & ~m;
        }
        uint32_t at = found + scan_all(sm, turn, __popc(m), all);
        for (; m && at < want; m &= m - 1u) list[at++] = p0 + (uint32_t)__ffs((int)m) - 1u;
        found += all;
    }
    __syncthreads();                      // the list is there
    return min(found, want);
}

struct ReserveSmem {
    Scan scan;
    uint32_t copies;
    // The entries that the call's tokens are written to, in order: sequence by sequence, position by position
    uint32_t before[kMaxSeqs + 1];        // entries of the sequences before
    uint32_t j0[kMaxSeqs];                // the first entry's column
    uint8_t r0[kMaxSeqs];                 // the rows before the first position in its page
    alignas(16) uint32_t page[kPlanThreads];
    uint32_t fresh[kPlanThreads];   // few entries: the shared pages; the new ones
};

// The sequence that entry `e` is of
__device__ __forceinline__ uint32_t sequence_of(const ReserveSmem &sm, uint32_t nseq, uint32_t e)
{
    uint32_t lo = 0u, hi = nseq;          // before[lo] <= e < before[hi]
    while (hi - lo > 1u) {
        const uint32_t mid = (lo + hi) >> 1;
        if (sm.before[mid] <= e) lo = mid;
        else hi = mid;
    }
    return lo;
}

// Who gets which page. An entry of the call needs a new page if it has none, or
// one that is named elsewhere too; but of a page that only entries of this call
// name, the last one keeps it. (One entry after the other: whoever finds its
// page named by others leaves it, until one is left.) New pages are the lowest
// free ones, in the entries' order; all or nothing. One CTA: the orders are
// those of scans over entries and pages. Up to a thread's entry each, the entries
// are looked at once, and those of one page find each other in shared memory;
// more go through arrays in the workspace, in several passes.
// Bound by latency: three dependent reads of L2 and three scans of some hundred
// cycles for few entries.
__device__ __forceinline__ void plan_reserve(const PlanArgs &a, ReserveSmem &sm)
{
    uint32_t turn = 0u, exist;
    if (threadIdx.x == 0) sm.copies = 0u;
    // on its way with the positions: what will be free
    const uint32_t used0 = used_mask(a.c, threadIdx.x * kPlanPages, exist), free0 = exist & ~used0;
    uint32_t total = 0u;
    for (uint32_t b = 0; b < a.c.nseq; b += kPlanThreads) {
        const uint32_t s = b + threadIdx.x;
        uint32_t n = 0u, all;
        if (s < a.c.nseq) {
            const uint32_t m = row_count(a.r, s);
            const uint64_t p0 = __ldcg(a.r.pos0 + s), p1 = min(p0 + m, (uint64_t)a.c.limit);
            const uint32_t j0 = (uint32_t)(p0 >> a.c.page_log2);
            if (p0 < p1) n = (uint32_t)((p1 - 1u) >> a.c.page_log2) - j0 + 1u;
            sm.j0[s] = j0;
            sm.r0[s] = (uint8_t)(p0 & ((1u << a.c.page_log2) - 1u));
        }
        const uint32_t at = total + scan_all(sm.scan, turn, n, all);
        if (s < a.c.nseq) sm.before[s] = at;
        total += all;
    }
    if (threadIdx.x == 0) sm.before[a.c.nseq] = total;
    __syncthreads();
    uint32_t *const writers = array_of(a.c, kWriters), *const last = array_of(a.c, kLastWriter);
    uint32_t *const from = array_of(a.c, kCopyFrom), *const to_page = array_of(a.c, kCopyTo), *const rows = array_of(a.c, kCopyRows);
    // page and place of entry e
    uint32_t s;
    size_t at;
    auto entry = [&](uint32_t e) {
        s = sequence_of(sm, a.c.nseq, e);
        at = (size_t)s * a.c.max_pages + sm.j0[s] + (e - sm.before[s]);
        return (uint32_t)__ldcg(a.c.table + at);
    };
    auto names_of = [&](uint32_t p) { return p < a.c.pages ? (uint32_t)max(__ldcg(a.c.refs + p), 0) : 0u; };
    // entry e of sequence s, at `at`, leaves page p for page `to`
    auto give = [&](uint32_t e, uint32_t p, uint32_t to) {
        a.c.table[at] = (int32_t)to;
        a.c.refs[to] = 1;
        const uint32_t r = e == sm.before[s] ? sm.r0[s] : 0u;
        if (p < a.c.pages && r) {
            const uint32_t i = atomicAdd(&sm.copies, 1u);
            from[i] = p;
            to_page[i] = to;
            rows[i] = r;
        }
    };
    uint32_t need;
    if (total <= kPlanThreads) {
        const uint32_t e = threadIdx.x;
        const bool mine = e < total;
        uint32_t p = ~0u, names = 0u;
        if (mine) {
            p = entry(e);
            names = names_of(p);
        }
        const bool shared = names > 1u;
        sm.page[e] = shared ? p : ~0u;
        uint32_t written = 0u, behind = 0u;       // entries of the call that name the page, and such ones behind this one
        if (__syncthreads_or(shared) && shared)
            for (uint32_t k = 0; k < total; k += 4u) {   // those behind the last one name none
                const uint4 x = *reinterpret_cast<const uint4 *>(sm.page + k);
                const uint32_t same = (x.x == p ? 1u : 0u) | (x.y == p ? 2u : 0u) | (x.z == p ? 4u : 0u) | (x.w == p ? 8u : 0u);
                written += __popc(same);
                behind += k + 4u <= e ? 0u : k > e ? __popc(same) : __popc(same >> (e - k) >> 1);
            }
        const bool is_last = shared && behind == 0u, keeps = mine && (names == 1u || (p < a.c.pages && names == 0u) || (is_last && written >= names));
        const bool want = mine && !keeps;
        const uint32_t rank = scan_all(sm.scan, turn, want ? 1u : 0u, need);
        const uint32_t found = need ? find_free(a.c, sm.scan, turn, free0, need, sm.fresh) : 0u;
        if (threadIdx.x == 0) *a.out = need - found;
        if (found == need) {
            if (is_last) a.c.refs[p] = (int32_t)(written >= names ? 1u : names - written);
            if (want) give(e, p, sm.fresh[rank]);
        }
    } else {
        // how many entries of the call name each page that has several names, and which of them is last
        bool shares = false;
        for (uint32_t e = threadIdx.x; e < total; e += kPlanThreads) {
            const uint32_t p = entry(e);
            if (names_of(p) > 1u) {
                writers[p] = 0u;
                last[p] = 0u;
                shares = true;
            }
        }
        if (__syncthreads_or(shares)) {
            for (uint32_t e = threadIdx.x; e < total; e += kPlanThreads) {
                const uint32_t p = entry(e);
                if (names_of(p) > 1u) {
                    atomicAdd(writers + p, 1u);
                    atomicMax(last + p, e);
                }
            }
            __syncthreads();
        }
        auto needs = [&](uint32_t e, uint32_t p) {
            if (p >= a.c.pages) return true;
            const uint32_t names = names_of(p);
            return names > 1u && (__ldcg(last + p) != e || __ldcg(writers + p) < names);
        };
        uint32_t mine = 0u;
        for (uint32_t e = threadIdx.x; e < total; e += kPlanThreads) mine += needs(e, entry(e)) ? 1u : 0u;
        scan_all(sm.scan, turn, mine, need);
        uint32_t *const fresh = array_of(a.c, kFresh);
        const uint32_t found = need ? find_free(a.c, sm.scan, turn, free0, need, fresh) : 0u;
        if (threadIdx.x == 0) *a.out = need - found;
        if (found == need) {
            uint32_t given = 0u;
            for (uint32_t b = 0; b < total; b += kPlanThreads) {
                const uint32_t e = b + threadIdx.x;
                uint32_t p = ~0u, all, names = 0u, written = 0u;
                bool want = false;
                if (e < total) {
                    p = entry(e);
                    want = needs(e, p);
                    if ((names = names_of(p)) > 1u) written = __ldcg(writers + p);
                }
                const uint32_t rank = given + scan_all(sm.scan, turn, want ? 1u : 0u, all);
                given += all;
                // the entry that is the page's last writer comes last: nobody after it looks at the page's count
                if (names > 1u && __ldcg(last + p) == e) a.c.refs[p] = (int32_t)(written >= names ? 1u : names - written);
                if (want) give(e, p, __ldcg(fresh + rank));
            }
        }
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        head_of(a.c)->copies = sm.copies;
        head_of(a.c)->from = ~0u;
    }
}

// U pages are in use. The i-th used page from number U on goes to the i-th free
// one below U, so that the first U are the used ones, and as few move as can be.
// One CTA, two passes over the counts (1027 pages: 6.9 us, cold and alone).
__device__ __forceinline__ void plan_compact(const PlanArgs &a, Scan &sm)
{
    uint32_t turn = 0u, exist0, exist, used;
    const uint32_t mask0 = used_mask(a.c, threadIdx.x * kPlanPages, exist0);   // the first pages' are kept for the second pass
    uint32_t mine = __popc(mask0);
    for (uint32_t b = kPlanThreads * kPlanPages; b < a.c.pages; b += kPlanThreads * kPlanPages) mine += __popc(used_mask(a.c, b + threadIdx.x * kPlanPages, exist));
    scan_all(sm, turn, mine, used);
    uint32_t *const from = array_of(a.c, kCopyFrom), *const to = array_of(a.c, kCopyTo), *const rows = array_of(a.c, kCopyRows);
    uint32_t *const moved = array_of(a.c, (WorkArray)kMovedTo);
    uint32_t holes = 0u, high = 0u;
    for (uint32_t b = 0; b < a.c.pages; b += kPlanThreads * kPlanPages) {
        const uint32_t p0 = b + threadIdx.x * kPlanPages;
        uint32_t m = mask0;
        exist = exist0;
        if (b) m = used_mask(a.c, p0, exist);
        const uint32_t low = used <= p0 ? 0u : used - p0 >= kPlanPages ? (1u << kPlanPages) - 1u : (1u << (used - p0)) - 1u;
        uint32_t free = exist & ~m & low, over = m & ~low, all;
        // both counts in one scan: at most 2^14 each
        const uint32_t before = scan_all(sm, turn, __popc(free) | (uint32_t)__popc(over) << 16, all);
        for (uint32_t i = holes + (before & 0xffffu); free; free &= free - 1u) to[i++] = p0 + (uint32_t)__ffs((int)free) - 1u;
        for (uint32_t i = high + (before >> 16); over; over &= over - 1u) from[i++] = p0 + (uint32_t)__ffs((int)over) - 1u;
        holes += all & 0xffffu;
        high += all >> 16;
    }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < high; i += kPlanThreads) {
        const uint32_t p = from[i], q = to[i];
        a.c.refs[q] = __ldcg(a.c.refs + p);
        a.c.refs[p] = 0;
        moved[p] = q;
        rows[i] = 1u << a.c.page_log2;
    }
    if (threadIdx.x == 0) {
        head_of(a.c)->copies = high;
        head_of(a.c)->from = used;
        *a.out = used;
    }
}

// Carries out a plan: the first rows of pages, in every layer, K and V, to other
// pages, and the table's new numbers. No target is a source. Rows that follow one
// another in both pages go 64 at a time (16 KB): pieces of whole pages, whose KV
// heads follow one another too, or of a head's first rows. One lane of each of a
// CTA's moving warps brings pieces into shared memory and out again by bulk copies,
// four buffers a warp, so that 192 KB an SM are on their way without a register.
// Bound by HBM (268 MB to another place 82.7 us, 6.5 TB/s, 99 % of the copy rate;
// 16-byte loads and stores by all threads, four on their way each: 154 us).
struct MoveArgs {
    Cache c;
    uint32_t early;
};

constexpr uint32_t kMoveWarps = 3, kMoveThreads = kMoveWarps * 32, kMoveStages = 4, kMoveRows = 64;

struct MovePiece {
    uint8_t *src, *dst;
    uint32_t bytes;
};

struct alignas(128) MoveSmem {
    uint8_t buffer[kMoveWarps][kMoveStages][kMoveRows * kRowBytes];
    uint64_t full[kMoveWarps][kMoveStages];
    MovePiece piece[kMoveWarps][kMoveStages];
    uint32_t err;
};

// The barriers; before a barrier of the CTA
__device__ __forceinline__ void init_move(MoveSmem &sm)
{
    const uint32_t warp = threadIdx.x >> 5;
    if ((threadIdx.x & 31u) == 0u && warp < kMoveWarps) {
        for (uint32_t i = 0; i < kMoveStages; ++i) mbar_init(&sm.full[warp][i], 1u);
        fence_mbar_init();
    }
    if (threadIdx.x == 0u) sm.err = kStatusOk;
}

// By CTA `cta` of `ctas`
__device__ __forceinline__ void move_pages(const Cache &ca, MoveSmem &sm, uint32_t cta, uint32_t ctas)
{
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
    const uint32_t copies = __ldcg(&head_of(ca)->copies), moved_from = __ldcg(&head_of(ca)->from);
    if (warp < kMoveWarps && copies) {
        const uint32_t *from = array_of(ca, kCopyFrom), *to = array_of(ca, kCopyTo), *rows = array_of(ca, kCopyRows);
        const bool whole = moved_from != ~0u;
        const uint32_t page = 1u << ca.page_log2;
        // runs of a page that lie together, and pieces of a run
        const uint32_t runs = whole ? 1u : ca.kv_heads, run_rows = whole ? ca.kv_heads << ca.page_log2 : page;
        const uint32_t subs = (run_rows + kMoveRows - 1u) / kMoveRows, per_page = runs * subs;
        const uint32_t pieces = copies * ca.layers * 2u * per_page, step = ctas * kMoveWarps;
        MovePiece *const slot = sm.piece[warp];
        uint64_t *const full = sm.full[warp];
        uint32_t loaded = 0u;
        bool ok = true;
        // lane 0: piece n, which was loaded, goes out
        auto store = [&](uint32_t n) {
            const MovePiece p = slot[n % kMoveStages];
            uint8_t *const buffer = sm.buffer[warp][n % kMoveStages];
            ok = ok && mbar_wait(full + n % kMoveStages, n / kMoveStages & 1u, &sm.err);
            if (ok) {
                asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(p.dst), "r"(smem_addr(buffer)), "r"(p.bytes) : "memory");
                asm volatile("cp.async.bulk.commit_group;" ::: "memory");
            } else {   // a wait that ran out: by hand
                for (uint32_t b = 0; b < p.bytes; b += 16u) *reinterpret_cast<uint4 *>(p.dst + b) = __ldcg(reinterpret_cast<const uint4 *>(p.src + b));
            }
        };
        // every lane looks a piece up, 32 at a time; lane 0 then copies them
        for (uint32_t x0 = cta * kMoveWarps + warp; x0 < pieces; x0 += 32u * step) {
            const uint32_t x = x0 + lane * step;
            MovePiece mine{nullptr, nullptr, 0u};
            if (x < pieces) {
                const uint32_t at = x / per_page, in = x - at * per_page, run = in / subs, row = (in - run * subs) * kMoveRows;
                const uint32_t i = at / (2u * ca.layers), layer2 = at - i * 2u * ca.layers;
                uint8_t *pool = reinterpret_cast<uint8_t *>(layer2 & 1u ? ca.v : ca.k);
                const uint32_t have = whole ? run_rows : __ldcg(rows + i), p = __ldcg(from + i), q = __ldcg(to + i);
                auto place = [&](uint32_t number) {
                    return pool + (((((uint64_t)(layer2 >> 1) * ca.pages + number) * ca.kv_heads + run) << ca.page_log2) + row) * kRowBytes;
                };
                if (row < have) mine = MovePiece{place(p), place(q), min(have - row, kMoveRows) * kRowBytes};
            }
            for (uint32_t there = __ballot_sync(0xffffffffu, mine.bytes != 0u); there; there &= there - 1u) {
                const int l = __ffs((int)there) - 1;
                MovePiece p;
                p.src = reinterpret_cast<uint8_t *>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(mine.src), l));
                p.dst = reinterpret_cast<uint8_t *>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(mine.dst), l));
                p.bytes = __shfl_sync(0xffffffffu, mine.bytes, l);
                if (lane == 0u) {
                    // loads are kMoveStages - 1 ahead of the stores; a buffer is free once its last store has read it
                    if (loaded >= kMoveStages - 1u) store(loaded - (kMoveStages - 1u));
                    asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
                    slot[loaded % kMoveStages] = p;
                    mbar_arrive_expect_tx(full + loaded % kMoveStages, p.bytes);
                    bulk_g2s(sm.buffer[warp][loaded % kMoveStages], p.src, p.bytes, full + loaded % kMoveStages);
                }
                ++loaded;
            }
        }
        if (lane == 0u) {
            for (uint32_t n = loaded - min(loaded, kMoveStages - 1u); n < loaded; ++n) store(n);
            asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
        }
    }
    if (moved_from == ~0u) return;
    const uint32_t *moved = array_of(ca, (WorkArray)kMovedTo);
    const size_t entries = (size_t)ca.nseq * ca.max_pages;
    for (size_t i = (size_t)cta * blockDim.x + threadIdx.x; i < entries; i += (size_t)ctas * blockDim.x) {
        const uint32_t p = (uint32_t)__ldcg(ca.table + i);
        if (p >= moved_from && p < ca.pages) ca.table[i] = (int32_t)__ldcg(moved + p);
    }
}

__global__ void __launch_bounds__(kMoveThreads) move_kernel(const __grid_constant__ MoveArgs a)
{
    extern __shared__ __align__(128) uint8_t move_smem[];
    MoveSmem &sm = *reinterpret_cast<MoveSmem *>(move_smem);
    init_move(sm);
    __syncthreads();
    wait_predecessor(a.early);
    move_pages(a.c, sm, blockIdx.x, gridDim.x);
}

// The plan, by one CTA; in a cluster, all its CTAs then carry it out.
template <bool COMPACT>
__global__ void __launch_bounds__(kPlanThreads) plan_kernel(const __grid_constant__ PlanArgs a)
{
    extern __shared__ __align__(128) uint8_t plan_smem[];
    const uint32_t ctas = k8::cluster_size();
    MoveSmem &move = *reinterpret_cast<MoveSmem *>(plan_smem);
    if (ctas > 1u) init_move(move);
    // the plan's own memory lies in the buffers
    static_assert(sizeof(ReserveSmem) <= sizeof(move.buffer), "the plan exceeds the buffers' memory");
    wait_predecessor(a.early);
    if (k8::cluster_rank() == 0u) {
        if (COMPACT) plan_compact(a, reinterpret_cast<ReserveSmem *>(plan_smem)->scan);
        else plan_reserve(a, *reinterpret_cast<ReserveSmem *>(plan_smem));
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (ctas == 1u) return;
    k8::cluster_sync();
    move_pages(a.c, move, k8::cluster_rank(), ctas);
}

// ------------------------------------------------------------- host side ----

bool on_device(const void *p, int dev)
{
    cudaPointerAttributes at{};
    if (cudaPointerGetAttributes(&at, p) != cudaSuccess) {
        cudaGetLastError();
        return false;
    }
    return at.type == cudaMemoryTypeManaged || (at.type == cudaMemoryTypeDevice && at.device == dev);
}

bool aligned(const void *p, uintptr_t n) { return ((uintptr_t)p & (n - 1)) == 0; }

constexpr uint32_t kMaxRecordRows = 256;

// What a call may have: query heads, values from token to token, tokens of all sequences
constexpr uint32_t kMaxHeads = 32768u;
constexpr uint64_t kMaxStep = 0xffffffffull, kMaxRows = 0x7fffffffull;

size_t parts_offset(uint32_t pages)
{
    return (sizeof(WorkHead) + (size_t)kWorkArrays * pages * 4u + 255u) & ~(size_t)255u;
}

size_t work_bytes(uint32_t pages) { return parts_offset(pages) + kPartsBytes + 2u * kMaxCtas * (size_t)record_floats(kMaxRecordRows) * 4u; }

int check_shape(const char *who, const AtlasPaged *c)
{
    if (c->type != ATLAS_PAGED_FP16 && c->type != ATLAS_PAGED_BF16)
        return api_fail(ATLAS_EINVAL, "%s: type %u is neither ATLAS_PAGED_FP16 nor ATLAS_PAGED_BF16", who, c->type);
    if (c->page != 16 && c->page != 32 && c->page != 64 && c->page != 128)
        return api_fail(ATLAS_EINVAL, "%s: pages of 16, 32, 64 or 128 positions, not %u", who, c->page);
    if (!c->layers || !c->pages || !c->kv_heads || c->kv_heads > 16384u || c->pages > 0x0fffffffu ||
        (uint64_t)c->pages * c->kv_heads * c->page > 0x7fffffffull / c->layers)
        return api_fail(ATLAS_EINVAL, "%s: bad pool (%u layers, %u pages of %u positions, %u KV heads): at most 2^31 - 1 rows", who,
                        c->layers, c->pages, c->page, c->kv_heads);
    if (!c->nseq || c->nseq > kMaxSeqs || !c->max_pages || (uint64_t)c->max_pages * c->page > 0x7fffff00ull ||
        (uint64_t)c->nseq * c->max_pages > 0x7fffffffull)
        return api_fail(ATLAS_EINVAL, "%s: bad table (%u sequences of %u pages)", who, c->nseq, c->max_pages);
    return ATLAS_OK;
}

// The checks that all calls share; fills the kernels' view of the cache.
int open_cache(const char *who, const AtlasPaged *c, Cache &out, int &dev, int &sms)
{
    if (!c || !c->k || !c->v || !c->table || !c->refs || !c->work) return api_fail(ATLAS_EINVAL, "%s: null argument", who);
    const int rc = check_shape(who, c);
    if (rc != ATLAS_OK) return rc;
    if (!aligned(c->k, 16) || !aligned(c->v, 16) || !aligned(c->refs, 16) || !aligned(c->table, 4) || !aligned(c->work, 256))
        return api_fail(ATLAS_EINVAL, "%s: the pool and refs must be 16-byte aligned, the table 4-byte, the workspace 256-byte", who);
    if (c->work_bytes < work_bytes(c->pages))
        return api_fail(ATLAS_EINVAL, "%s: a workspace of %llu bytes, not %llu", who, (unsigned long long)work_bytes(c->pages),
                        (unsigned long long)c->work_bytes);
    dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || api_device(dev, &sms) != ATLAS_OK)
        return api_fail(ATLAS_ENODEV, "%s: no sm_100 device", who);
    const void *need[] = {c->k, c->v, c->table, c->refs, c->work};
    for (const void *p : need)
        if (!on_device(p, dev)) return api_fail(ATLAS_EINVAL, "%s: the cache must be memory of the current device", who);
    out.k = static_cast<uint16_t *>(c->k);
    out.v = static_cast<uint16_t *>(c->v);
    out.table = c->table;
    out.refs = c->refs;
    out.work = static_cast<uint32_t *>(c->work);
    out.layers = c->layers;
    out.pages = c->pages;
    out.kv_heads = c->kv_heads;
    out.page_log2 = c->page == 16 ? 4 : c->page == 32 ? 5 : c->page == 64 ? 6 : 7;
    out.nseq = c->nseq;
    out.max_pages = c->max_pages;
    out.limit = c->max_pages << out.page_log2;
    return ATLAS_OK;
}

// Device integers of a call; null where `optional`
int check_ints(const char *who, const char *name, const void *p, int dev, bool optional = false)
{
    if (!p && optional) return ATLAS_OK;
    if (!p) return api_fail(ATLAS_EINVAL, "%s: null argument", who);
    if (!aligned(p, 4) || !on_device(p, dev))
        return api_fail(ATLAS_EINVAL, "%s: %s must be 4-byte aligned memory of the current device", who, name);
    return ATLAS_OK;
}

int check_tokens(const char *who, uint32_t tokens, const uint32_t *pos0, const uint32_t *n_tok, Rows &rows, int dev)
{
    if (tokens > 0x00ffffffu) return api_fail(ATLAS_EINVAL, "%s: at most 2^24 - 1 tokens, not %u", who, tokens);
    int rc = check_ints(who, "pos0", pos0, dev);
    if (rc == ATLAS_OK) rc = check_ints(who, "n_tok", n_tok, dev, true);
    rows = Rows{pos0, n_tok, tokens};
    return rc;
}

// Token rows of `heads` x 128 values, ld values apart (0: dense).
int check_rows(const char *who, const void *p, uint32_t heads, uint64_t &ld, int dev)
{
    if (!p) return api_fail(ATLAS_EINVAL, "%s: null argument", who);
    if (!ld) ld = (uint64_t)heads * kDim;
    if (ld < (uint64_t)heads * kDim || ld % 8 || ld > kMaxStep)
        return api_fail(ATLAS_EINVAL, "%s: token rows %llu values apart: at least heads x 128, a multiple of 8", who, (unsigned long long)ld);
    if (!aligned(p, 16)) return api_fail(ATLAS_EINVAL, "%s: token rows must be 16-byte aligned", who);
    if (!on_device(p, dev)) return api_fail(ATLAS_EINVAL, "%s: token rows must be memory of the current device", who);
    return ATLAS_OK;
}

// Whether `n` rows of `width` values from a on, lda values apart, share memory with rows of b, ldb apart (at least `width` each).
// Rows the same distance apart may lie beside one another, as in a buffer of both; others share it where their ranges do.
bool rows_overlap(const void *a, uint64_t lda, const void *b, uint64_t ldb, uint64_t width, uint64_t n)
{
    if ((uintptr_t)a > (uintptr_t)b) {
        std::swap(a, b);
        std::swap(lda, ldb);
    }
    const uint64_t ahead = (uintptr_t)b - (uintptr_t)a, bytes = 2 * width, step = 2 * lda;   // b's first row lies `ahead` behind a's
    if (ahead >= (n - 1) * step + bytes) return false;
    if (lda != ldb || n == 1) return true;
    // b's first row begins in the step of a's row `ahead` / `step`; the next of a's, if there is one, may reach into its end
    const uint64_t row = ahead / step, in = ahead - row * step;
    return in < bytes || (row + 1 < n && step - in < bytes);
}

using Encode = decltype(&cuTensorMapEncodeTiled);

int find_encode(const char *who, Encode &encode)
{
    static std::atomic<Encode> known{nullptr};
    encode = known.load(std::memory_order_acquire);
    if (!encode) {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult found{};
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &found) != cudaSuccess ||
            found != cudaDriverEntryPointSuccess || !p) {
            cudaGetLastError();
            return api_fail(ATLAS_ECUDA, "%s: the driver has no cuTensorMapEncodeTiled", who);
        }
        encode = reinterpret_cast<Encode>(p);
        known.store(encode, std::memory_order_release);
    }
    return ATLAS_OK;
}

// A pool as [2 halves of 64 dimensions][rows][64], for copies of `box` rows of both halves
int map_pool(const char *who, Encode encode, const Cache &c, bool bf, void *pool, uint32_t box, uint32_t halves, CUtensorMap &map)
{
    const cuuint64_t rows = ((cuuint64_t)c.layers * c.pages * c.kv_heads) << c.page_log2;
    const cuuint64_t dims[3] = {kDim / 2, rows, 2}, strides[2] = {kRowBytes, kRowBytes / 2};
    const cuuint32_t boxes[3] = {kDim / 2, box, halves}, steps[3] = {1, 1, 1};
    if (!k8::in_context([&] {
            return encode(&map, bf ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, pool, dims, strides, boxes, steps,
                          CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
        }))
        return api_fail(ATLAS_ECUDA, "%s: the pool cannot be described to the copy engine", who);
    return ATLAS_OK;
}

int done(const char *who, cudaError_t e)
{
    if (e == cudaSuccess) return ATLAS_OK;
    cudaGetLastError();
    return api_fail(ATLAS_ECUDA, "%s: %s", who, cudaGetErrorString(e));
}

// Plans, and copies at most `copies` pages: in one launch of a cluster where that is little (16 SMs copy 1.5 TB/s or so; a second
// launch costs 2.4 us on the host and 2 on the device), in two where it may be much
constexpr uint64_t kLittle = 8u << 20;
constexpr uint32_t kPlanCluster = 16;

template <bool COMPACT>
cudaError_t launch_plan(const PlanArgs &p, uint64_t copies, int dev, int sms, cudaStream_t stream)
{
    const Cache &c = p.c;
    cudaError_t e = k8::allow<plan_kernel<COMPACT>>(dev, (int)sizeof(MoveSmem));
    if (e != cudaSuccess) return e;
    const uint64_t bytes = copies * c.layers * 2 * ((uint64_t)c.kv_heads << c.page_log2) * kRowBytes;
    if (bytes <= kLittle && k8::clusters_at_once<plan_kernel<COMPACT>>(dev, kPlanCluster, kPlanThreads, sizeof(MoveSmem)))
        return launch(plan_kernel<COMPACT>, dim3(kPlanCluster), kPlanThreads, sizeof(MoveSmem), kPlanCluster, p, sms, stream);
    if ((e = launch(plan_kernel<COMPACT>, dim3(1), kPlanThreads, sizeof(ReserveSmem), 1, p, sms, stream)) != cudaSuccess) return e;
    if ((e = k8::allow<move_kernel>(dev, (int)sizeof(MoveSmem))) != cudaSuccess) return e;
    MoveArgs a{};
    a.c = c;
    const uint64_t entries = COMPACT ? (uint64_t)c.nseq * c.max_pages : 0;
    const uint64_t ctas = std::max(bytes / (kMoveWarps * kMoveRows * kRowBytes), entries / kMoveThreads) + 1;
    return launch(move_kernel, dim3((uint32_t)std::min<uint64_t>(ctas, (uint64_t)sms)), kMoveThreads, sizeof(MoveSmem), 1, a, sms, stream);
}

}  // namespace
}  // namespace paged
}  // namespace atlas

using namespace atlas;
using namespace atlas::paged;

extern "C" int atlas_cuda_paged_work(const AtlasPaged *cache, uint64_t *bytes)
{
    const char *who = "paged_work";
    if (!cache || !bytes) return api_fail(ATLAS_EINVAL, "%s: null argument", who);
    const int rc = check_shape(who, cache);
    if (rc == ATLAS_OK) *bytes = work_bytes(cache->pages);
    return rc;
}

extern "C" int atlas_cuda_paged_append(const AtlasPaged *cache, uint32_t layer, uint32_t tokens, const uint32_t *d_pos0,
                                       const uint32_t *d_ntok, const void *d_k, const void *d_v, uint64_t ld, void *stream)
{
    const char *who = "paged_append";
    AppendArgs a{};
    int dev, sms, rc = open_cache(who, cache, a.c, dev, sms);
    if (rc == ATLAS_OK) rc = check_tokens(who, tokens, d_pos0, d_ntok, a.r, dev);
    if (rc == ATLAS_OK && layer >= cache->layers) rc = api_fail(ATLAS_EINVAL, "%s: layer %u of %u", who, layer, cache->layers);
    if (rc != ATLAS_OK || !tokens) return rc;   // no rows need no memory
    if ((rc = check_rows(who, d_k, cache->kv_heads, ld, dev)) != ATLAS_OK) return rc;
    if ((rc = check_rows(who, d_v, cache->kv_heads, ld, dev)) != ATLAS_OK) return rc;
    a.k = static_cast<const uint16_t *>(d_k);
    a.v = static_cast<const uint16_t *>(d_v);
    a.ld = ld;
    a.layer = layer;
    constexpr uint64_t per = kAppendThreads / 16u * kAppendRows;
    const uint64_t ctas = ((uint64_t)tokens * cache->kv_heads + per - 1) / per;
    if (ctas > 0x7fffffffull) return api_fail(ATLAS_EINVAL, "%s: too many rows", who);
    return done(who, launch(append_kernel, dim3((uint32_t)ctas, cache->nseq), kAppendThreads, 0, 1, a, sms, (cudaStream_t)stream));
}

extern "C" int atlas_cuda_paged_fork(const AtlasPaged *cache, const int32_t *d_parent, const uint32_t *d_length, const uint32_t *d_first,
                                     void *stream)
{
    const char *who = "paged_fork";
    ForkArgs a{};
    int dev, sms, rc = open_cache(who, cache, a.c, dev, sms);
    if (rc == ATLAS_OK) rc = check_ints(who, "parent", d_parent, dev);
    if (rc == ATLAS_OK) rc = check_ints(who, "length", d_length, dev);
    if (rc == ATLAS_OK) rc = check_ints(who, "first", d_first, dev, true);
    if (rc != ATLAS_OK) return rc;
    a.parent = d_parent;
    a.length = d_length;
    a.first = d_first;
    const cudaError_t e = k8::allow<fork_kernel>(dev, (int)(kMaxSeqs * kForkColumns * 4u));
    if (e != cudaSuccess) return done(who, e);
    return done(who, launch(fork_kernel, dim3((cache->max_pages + kForkColumns - 1) / kForkColumns), kForkThreads,
                            (size_t)cache->nseq * kForkColumns * 4u, 1, a, sms, (cudaStream_t)stream));
}

extern "C" int atlas_cuda_paged_reserve(const AtlasPaged *cache, uint32_t tokens, const uint32_t *d_pos0, const uint32_t *d_ntok,
                                        uint32_t *d_short, void *stream)
{
    const char *who = "paged_reserve";
    PlanArgs a{};
    int dev, sms, rc = open_cache(who, cache, a.c, dev, sms);
    if (rc == ATLAS_OK) rc = check_tokens(who, tokens, d_pos0, d_ntok, a.r, dev);
    if (rc == ATLAS_OK) rc = check_ints(who, "short", d_short, dev);
    if (rc != ATLAS_OK) return rc;
    a.out = d_short;
    // a sequence's first page at most is copied
    return done(who, launch_plan<false>(a, std::min(cache->nseq, cache->pages), dev, sms, (cudaStream_t)stream));
}

extern "C" int atlas_cuda_paged_compact(const AtlasPaged *cache, uint32_t *d_used, void *stream)
{
    const char *who = "paged_compact";
    PlanArgs a{};
    int dev, sms, rc = open_cache(who, cache, a.c, dev, sms);
    if (rc == ATLAS_OK) rc = check_ints(who, "used", d_used, dev);
    if (rc != ATLAS_OK) return rc;
    a.out = d_used;
    return done(who, launch_plan<true>(a, cache->pages / 2u, dev, sms, (cudaStream_t)stream));
}

namespace {

// The query rows of a KV head that a CTA takes at a time: 8 or 16 (the form for few rows), 128 or 256. Measured, us in a row
// of calls, all with the build as it is, in turn. Up to 16 rows in the form for few, or units of 128: 2 and 3 tokens of 8
// sequences over 2303, 40 heads on 8, 22.0 and 26.7, 22.2 and 27.4; 3 over 8447 15.8 and 18.0; 2 of 4 sequences over 640, 28
// on 4, 9.3 and 13.4. 128 or 256, where 128 leave no CTA a second unit: 7 tokens of 4 sequences over 8001 27.8 and 31.5, 333
// of 16 on 2 over 5001 42 to 44 and 46, 512 of 28 on 4 16 and 19; where they do: 1000 of 40 on 8 44 and 41, 8 x 2048 652 and
// 509, 8192 704 to 712 and 669 to 697.
constexpr uint32_t kFewRows = 16;

uint32_t attn_rows(const Cache &c, uint32_t group, uint32_t tokens, int sms)
{
    const uint64_t rows = (uint64_t)tokens * group;
    if (rows <= kFewRows || group > 128) return rows <= 8 ? 8 : 16;
    const uint32_t per = 128 / group;
    return (uint64_t)c.nseq * c.kv_heads * ((tokens + per - 1) / per) <= (uint64_t)sms ? 128 : 256;
}

// The token rows of q as [2 halves of 64 dimensions][token][head][64], for copies of a KV head's group of heads of `tokens` tokens
int map_queries(const char *who, Encode encode, const AttnArgs &a, bool bf, uint32_t tokens, CUtensorMap &map)
{
    const cuuint64_t dims[4] = {kDim / 2, a.q_heads, (cuuint64_t)a.c.nseq * a.r.tokens, 2}, strides[3] = {kRowBytes, a.ldq * 2, kRowBytes / 2};
    const cuuint32_t boxes[4] = {kDim / 2, a.group, tokens, 1}, steps[4] = {1, 1, 1, 1};
    if (!k8::in_context([&] {
            return encode(&map, bf ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<uint16_t *>(a.q), dims, strides,
                          boxes, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
        }))
        return api_fail(ATLAS_ECUDA, "%s: the token rows cannot be described to the copy engine", who);
    return ATLAS_OK;
}

int check_heads(const char *who, const AtlasPaged *cache, uint32_t q_heads, uint32_t tokens)
{
    if (!q_heads || q_heads % cache->kv_heads || q_heads > kMaxHeads || (uint64_t)q_heads * tokens > 0x3fffffffull ||
        (uint64_t)tokens * cache->nseq > kMaxRows)
        return api_fail(ATLAS_EINVAL, "%s: %u query heads over %u KV heads, %u tokens", who, q_heads, cache->kv_heads, tokens);
    return ATLAS_OK;
}

}  // namespace

extern "C" int atlas_cuda_paged_attn_form(const AtlasPaged *cache, uint32_t q_heads, uint32_t tokens, uint32_t *rows)
{
    const char *who = "paged_attn_form";
    if (!cache || !rows) return api_fail(ATLAS_EINVAL, "%s: null argument", who);
    Cache c;
    int dev, sms, rc = open_cache(who, cache, c, dev, sms);
    if (rc == ATLAS_OK) rc = check_heads(who, cache, q_heads, tokens);
    if (rc == ATLAS_OK && !tokens) rc = api_fail(ATLAS_EINVAL, "%s: no tokens", who);
    if (rc == ATLAS_OK) *rows = attn_rows(c, q_heads / cache->kv_heads, tokens, sms);
    return rc;
}

extern "C" int atlas_cuda_paged_attn(const AtlasPaged *cache, uint32_t layer, uint32_t q_heads, uint32_t tokens, const uint32_t *d_pos0,
                                     const uint32_t *d_ntok, const void *d_q, uint64_t ldq, void *d_out, uint64_t ldo, void *stream)
{
    const char *who = "paged_attn";
    AttnArgs a{};
    int dev, sms, rc = cache ? check_shape(who, cache) : ATLAS_OK;
    if (rc != ATLAS_OK) return rc;
    // a row of `out` may be written before another CTA has read its neighbours in `q`
    if (cache && d_q && d_out && tokens && q_heads && q_heads <= kMaxHeads) {   // sizes past the limits are refused below
        const uint64_t width = (uint64_t)q_heads * kDim, lq = ldq ? ldq : width, lo = ldo ? ldo : width, n = (uint64_t)cache->nseq * tokens;
        if (lq >= width && lo >= width && lq <= kMaxStep && lo <= kMaxStep && n <= kMaxRows && rows_overlap(d_q, lq, d_out, lo, width, n))
            return api_fail(ATLAS_EINVAL, "%s: q and out must not overlap", who);
    }
    rc = open_cache(who, cache, a.c, dev, sms);
    if (rc == ATLAS_OK) rc = check_tokens(who, tokens, d_pos0, d_ntok, a.r, dev);
    if (rc != ATLAS_OK) return rc;
    if ((rc = check_heads(who, cache, q_heads, tokens)) != ATLAS_OK) return rc;
    if (layer >= cache->layers) return api_fail(ATLAS_EINVAL, "%s: layer %u of %u", who, layer, cache->layers);
    if (!tokens) return ATLAS_OK;               // no rows need no memory
    if ((rc = check_rows(who, d_q, q_heads, ldq, dev)) != ATLAS_OK) return rc;
    if ((rc = check_rows(who, d_out, q_heads, ldo, dev)) != ATLAS_OK) return rc;
    a.q = static_cast<const uint16_t *>(d_q);
    a.out = static_cast<uint16_t *>(d_out);
    a.ldq = ldq;
    a.ldo = ldo;
    a.q_heads = q_heads;
    a.group = q_heads / cache->kv_heads;
    a.by_group = divisor(a.group);
    a.layer = layer;
    a.parts = reinterpret_cast<float *>(static_cast<char *>(cache->work) + parts_offset(cache->pages));
    const bool bf = cache->type == ATLAS_PAGED_BF16;
    const uint32_t rows = attn_rows(a.c, a.group, tokens, sms);
    const bool prompt = rows >= 128;
    Encode encode;
    if ((rc = find_encode(who, encode)) != ATLAS_OK) return rc;
    CUtensorMap kmap, vmap, qmap;
    // 16 rows of all dimensions at a time, or a page's of half of them
    const uint32_t box = prompt ? cache->page : 16, halves = prompt ? 1 : 2;
    if ((rc = map_pool(who, encode, a.c, bf, cache->k, box, halves, kmap)) != ATLAS_OK) return rc;
    if ((rc = map_pool(who, encode, a.c, bf, cache->v, box, halves, vmap)) != ATLAS_OK) return rc;
    if (!prompt) return done(who, launch_few(a, kmap, vmap, bf, (int)rows / 8, dev, sms, (cudaStream_t)stream));
    if ((rc = map_queries(who, encode, a, bf, 128 / a.group, qmap)) != ATLAS_OK) return rc;
    return done(who, launch_prompt(a, kmap, vmap, qmap, bf, rows / 128, dev, sms, (cudaStream_t)stream));
}
