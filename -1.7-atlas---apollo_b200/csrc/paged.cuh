// What the attention kernels over pages share: how a call's work is dealt out
// over the CTAs, the partial sums' places, 16-bit types.
//
// A unit is a tile of a sequence's query rows and a KV head; its work is the
// tiles of keys (of KEYS positions) that its last row sees. All units' tiles of
// keys, in the order sequence, head, rows, make one line, of which each CTA
// takes an equal piece: whole units inside it are finished by the CTA; of those
// that its ends cut, it leaves partial sums (Part), which part_merge_kernel
// joins. So every SM has the same to read and compute whatever the lengths,
// which only the device knows, and the pieces do not depend on timing.
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>
#include "kv8.cuh"
#include "paged.h"

namespace atlas {
namespace paged {

// Of each CTA: two records of partial sums, that of the unit that its piece
// begins in, and that of the one it ends in. A record: [rows][128] sums, then
// [rows] (maximum, sum of weights), for `rows` = the form's rows per unit.
// In front of all, a Part per CTA.
struct Part {
    uint32_t first;       // the record that the unit begins in; ~0: no unit that others began ends in this CTA's piece
    uint32_t count;       // records of the unit: `first`, then 2 x its CTA's following numbers
    uint32_t s, h, row0, rows;
    uint32_t pad[2];
};

constexpr size_t kPartsBytes = kMaxCtas * sizeof(Part);
constexpr uint32_t record_floats(uint32_t rows) { return rows * (kDim + 2u); }

namespace {

using k8::ex2;
using k8::TileRows;

// Two floats as a pair of 16-bit values, `lo` in the lower half
template <bool BF>
__device__ __forceinline__ uint32_t pack(float lo, float hi)
{
    uint32_t d;
    if (BF) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
    else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
    return d;
}

// One 16-bit value as a float
template <bool BF>
__device__ __forceinline__ float unpack1(uint32_t x)
{
    return BF ? __uint_as_float(x << 16) : __half2float(__ushort_as_half((unsigned short)x));
}

// Bits of the halves of x that are infinite or NaN: 0xffff each
template <bool BF>
__device__ __forceinline__ uint32_t nonfinite2(uint32_t x)
{
    constexpr uint32_t e = BF ? 0x7f80u : 0x7c00u;
    return ((x & e) == e ? 0xffffu : 0u) | ((x >> 16 & e) == e ? 0xffff0000u : 0u);
}

// Dividing 64-bit numbers that mostly have 32 bits
__device__ __forceinline__ uint64_t quotient(uint64_t a, uint64_t b)
{
    return ((a | b) >> 32) == 0u ? (uint64_t)((uint32_t)a / (uint32_t)b) : a / b;
}

// A sequence as its units see it: tiles of keys [k0, ..), k0 behind the pages that are gone at its start
struct Seq {
    uint32_t p0, rows, k0;
};

// Up to this many sequences, each lane of a warp keeps one's Seq (where the line has less than 2^31 tiles of keys)
constexpr uint32_t kKeptSeqs = 32;

// How a call's rows are cut into tiles of `tile` rows. Beginning and ending a unit takes as long as EXTRA tiles of keys: in the
// line, each unit has that many places before its tiles of keys.
template <uint32_t KEYS, uint32_t EXTRA>
struct Cut {
    const AttnArgs &a;
    const uint32_t tile;  // query rows of a unit
    const Divisor by_tile;

    // the tiles of keys that rows before `row1` see, from the front
    __device__ __forceinline__ uint32_t keys(const Seq &q, uint32_t row1) const
    {
        const uint64_t last = min((uint64_t)q.p0 + divide(row1 - 1u, a.by_group) + 1u, (uint64_t)a.c.limit);
        return (uint32_t)((last + KEYS - 1u) / KEYS);
    }
    __device__ __forceinline__ uint32_t units(const Seq &q) const { return divide(q.rows + tile - 1u, by_tile); }
    // work of a unit: at least one tile of keys, so that its rows are written
    __device__ __forceinline__ uint32_t cost(const Seq &q, uint32_t i) const
    {
        const uint32_t k = keys(q, min((i + 1u) * tile, q.rows));
        return k > q.k0 ? k - q.k0 : 1u;
    }
    // The first tile of keys behind the pages that are gone at a sequence's start: its leading entries that name none are
    // passed over, 128 at a time. The whole warp.
    __device__ __forceinline__ uint32_t begin(uint32_t s, uint32_t p0, uint32_t rows) const
    {
        const int32_t *entries = a.c.table + (size_t)s * a.c.max_pages;
        const uint32_t lane = threadIdx.x & 31u;
        const uint32_t seen = (uint32_t)min((uint64_t)p0 + divide(rows - 1u, a.by_group) + 1u, (uint64_t)a.c.limit);
        const uint32_t pages = (seen + (1u << a.c.page_log2) - 1u) >> a.c.page_log2;
        uint32_t page = pages;
        for (uint32_t b = 0; b < pages && page == pages; b += 128u) {
            uint32_t x[4];
#pragma unroll
            for (uint32_t i = 0; i < 4u; ++i) x[i] = b + 32u * i + lane < pages ? (uint32_t)__ldcg(entries + b + 32u * i + lane) : ~0u;
#pragma unroll
            for (uint32_t i = 0; i < 4u; ++i) {
                const uint32_t have = __ballot_sync(0xffffffffu, x[i] < a.c.pages);
                if (have && page == pages) page = b + 32u * i + (uint32_t)__ffs((int)have) - 1u;
            }
        }
        return (uint32_t)(((uint64_t)page << a.c.page_log2) / KEYS);
    }
    // the whole warp
    __device__ __forceinline__ Seq open(uint32_t s) const
    {
        const uint32_t e0 = (uint32_t)__ldcg(a.c.table + (size_t)s * a.c.max_pages);
        Seq q;
        q.p0 = __ldcg(a.r.pos0 + s);
        q.rows = row_count(a.r, s) * a.group;
        q.k0 = q.rows && e0 >= a.c.pages ? begin(s, q.p0, q.rows) : 0u;
        return q;
    }
    // `kept`: this lane's, where lanes keep them
    __device__ __forceinline__ Seq open(uint32_t s, const Seq &kept) const { return a.keep ? open_each(s, kept) : open(s); }
    // the same for a sequence of each lane's own, where lanes keep them
    __device__ __forceinline__ Seq open_each(uint32_t s, const Seq &kept) const
    {
        Seq q;
        q.p0 = __shfl_sync(0xffffffffu, kept.p0, (int)s);
        q.rows = __shfl_sync(0xffffffffu, kept.rows, (int)s);
        q.k0 = __shfl_sync(0xffffffffu, kept.k0, (int)s);
        return q;
    }
    // a sequence's work, and its largest unit's; the whole warp
    __device__ __forceinline__ uint64_t all(const Seq &q, uint32_t &most) const
    {
        const uint32_t lane = threadIdx.x & 31u, n = q.rows ? units(q) : 0u;
        uint64_t sum = 0u;
        uint32_t m = 0u;
        for (uint32_t i = lane; i < n; i += 32u) {
            const uint32_t c = cost(q, i);
            sum += c + EXTRA;
            m = max(m, c);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        most = max(most, __reduce_max_sync(0xffffffffu, m));
        return sum;
    }
};

// The piece of a CTA: it begins in unit (s, h, i), `skip` tiles of keys behind the unit's first one, and has `left` of them
struct Piece {
    uint64_t begin, each; // in the line of all; a CTA's share, or 0: pieces are of one unit, and
    uint32_t behind;      // so many pieces of it come before this one
    uint32_t shared;      // CTAs of a cluster that have the piece together: one unit, whole
    uint32_t s, h, i, skip;
    uint64_t left;
    Seq kept;             // lane s has sequence s, where lanes keep them
};

struct PieceSmem {
    uint64_t work[kMaxSeqs + 1];          // a sequence's tiles of keys; then those of the sequences up to it
    uint32_t units[kMaxSeqs + 1];         // its units, likewise
    uint32_t most[32];                    // the largest unit that a warp has seen
    uint32_t all_units;
};

__device__ __forceinline__ uint64_t up_to(uint64_t x)   // the sum of the lanes' x up to this one
{
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint64_t y = __shfl_up_sync(0xffffffffu, x, o);
        if ((threadIdx.x & 31u) >= (uint32_t)o) x += y;
    }
    return x;
}
__device__ __forceinline__ uint32_t up_to(uint32_t x)
{
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t y = __shfl_up_sync(0xffffffffu, x, o);
        if ((threadIdx.x & 31u) >= (uint32_t)o) x += y;
    }
    return x;
}

// The unit of sequence p.s that place `rest` of a KV head's units is in, from its place in the line
template <class T, uint32_t KEYS, uint32_t EXTRA>
__device__ __forceinline__ void enter_unit(const Cut<KEYS, EXTRA> &cut, Piece &p, T rest)
{
    const uint32_t lane = threadIdx.x & 31u;
    const Seq q = cut.open(p.s, p.kept);
    const uint32_t units = cut.units(q);
    for (uint32_t b = 0; units > 1u; b += 32u) {
        const uint32_t c = b + lane < units ? cut.cost(q, b + lane) + EXTRA : 0u;
        const T x = up_to((T)c);
        const uint32_t past = __ballot_sync(0xffffffffu, x > rest);
        if (past || b + 32u >= units) {
            const uint32_t at = past ? (uint32_t)__ffs((int)past) - 1u : 31u;
            p.i = min(b + at, units - 1u);
            rest -= __shfl_sync(0xffffffffu, x - c, (int)at);
            break;
        }
        rest -= __shfl_sync(0xffffffffu, x, 31);
    }
    // what lies before the first tile of keys is not work
    const uint32_t place = (uint32_t)rest;
    p.skip = place > EXTRA ? place - EXTRA : 0u;
    if (place < EXTRA) p.left -= min(p.left, (uint64_t)(EXTRA - place));
}

// This CTA's piece where a warp's lanes keep the sequences; by each warp that wants it, for itself. The line is cut into equal
// pieces of `least` tiles of keys at least; but units that are no more than CTAs (and 32 of a KV head) are cut one by one
// if no piece gets longer than that, and left whole if none gets more than `worth` tiles longer (what joining partial
// sums costs). In clusters, if there are enough of them, each has a unit together. (Short code on purpose: its first run after
// a launch waits for its instructions; in an earlier build, with up to 128 units of a KV head in four registers a lane, a
// prompt's calls took 2 to 4 us longer.)
template <uint32_t KEYS, uint32_t EXTRA>
__device__ __forceinline__ Piece find_kept(const Cut<KEYS, EXTRA> &cut, uint32_t least, uint32_t worth, uint32_t cluster = 1u)
{
    const AttnArgs &a = cut.a;
    const uint32_t lane = threadIdx.x & 31u, n = a.c.nseq;
    Piece p;
    p.s = p.h = p.i = p.skip = 0u;
    p.begin = p.each = 0u;
    p.behind = 0u;
    p.shared = 1u;
    p.left = 0u;
    uint32_t most = 0u;
    const bool there = lane < n;
    const uint32_t e0 = there ? (uint32_t)__ldcg(a.c.table + (size_t)lane * a.c.max_pages) : 0u;
    p.kept.p0 = there ? __ldcg(a.r.pos0 + lane) : 0u;
    p.kept.rows = there ? row_count(a.r, lane) * a.group : 0u;
    p.kept.k0 = 0u;
    for (uint32_t gone = __ballot_sync(0xffffffffu, p.kept.rows && e0 >= a.c.pages); gone; gone &= gone - 1u) {
        const uint32_t s = (uint32_t)__ffs((int)gone) - 1u;
        const uint32_t k0 = cut.begin(s, __shfl_sync(0xffffffffu, p.kept.p0, (int)s), __shfl_sync(0xffffffffu, p.kept.rows, (int)s));
        if (lane == s) p.kept.k0 = k0;
    }
    // lane s: its sequence's units and work per KV head
    const uint32_t units = p.kept.rows ? cut.units(p.kept) : 0u;
    uint32_t work = 0u;
    if (__all_sync(0xffffffffu, units <= 4u)) {
        for (uint32_t i = 0; i < units; ++i) {
            const uint32_t c = cut.cost(p.kept, i);
            work += c + EXTRA;
            most = max(most, c);
        }
        most = __reduce_max_sync(0xffffffffu, most);
    } else {
        for (uint32_t s = 0; s < n; ++s) {
            const uint32_t sum = (uint32_t)cut.all(cut.open(s, p.kept), most);
            if (lane == s) work = sum;
        }
    }
    // the line up to the end of each sequence
    const uint32_t all_units = __reduce_add_sync(0xffffffffu, units) * a.c.kv_heads;
    const uint32_t line = n == 1u ? work * a.c.kv_heads : up_to(work * a.c.kv_heads);
    const uint32_t total = __shfl_sync(0xffffffffu, line, (int)n - 1);
    if (!total) return p;
    const uint32_t each = max((total + gridDim.x - 1u) / gridDim.x, least);
    if (cluster > 1u && all_units * cluster <= gridDim.x && (most + cluster - 1u) / cluster <= each + worth) {
        const uint32_t u = blockIdx.x / cluster;
        if (u >= all_units) return p;
        const uint32_t ends = n == 1u ? all_units : up_to(units * a.c.kv_heads);
        uint32_t before = 0u;
        if (n > 1u) {
            p.s = (uint32_t)__ffs((int)__ballot_sync(0xffffffffu, lane < n && ends > u)) - 1u;
            before = __shfl_sync(0xffffffffu, ends, p.s ? (int)p.s - 1 : 0);
            if (p.s == 0u) before = 0u;
        }
        const uint32_t own = __shfl_sync(0xffffffffu, units, (int)p.s);
        p.h = (u - before) / own;
        p.i = u - before - p.h * own;
        p.left = cut.cost(cut.open(p.s, p.kept), p.i);
        p.shared = cluster;
        return p;
    }
    if (all_units <= gridDim.x && all_units <= 32u * a.c.kv_heads) {
        // Units cut into pieces of their own. Lane l has tile number l of all sequences' tiles of rows: its sequence, its number
        // there and its work.
        uint32_t seq = lane, tile = 0u, cost = units ? work - EXTRA : 0u;
        if (!__all_sync(0xffffffffu, units <= 1u)) {
            const uint32_t tiles_to = up_to(units), all_tiles = __shfl_sync(0xffffffffu, tiles_to, 31);
            seq = 0u;
#pragma unroll
            for (uint32_t step = 16u; step; step >>= 1)
                if (__shfl_sync(0xffffffffu, tiles_to, (int)(seq + step - 1u)) <= lane) seq += step;
            tile = lane - (__shfl_sync(0xffffffffu, tiles_to, (int)seq) - __shfl_sync(0xffffffffu, units, (int)seq));
            const Seq q = cut.open_each(seq, p.kept);
            cost = lane < all_tiles ? cut.cost(q, tile) : 0u;
        }
        // The pieces' size: sum ceil(work / size) <= CTAs holds where size >= total / (CTAs - units), as rounding up adds
        // less than one a unit, and where every unit gets as many pieces as the largest one
        uint32_t size = most;
        if (most > each + worth) {
            size = (most + gridDim.x / all_units - 1u) / (gridDim.x / all_units);
            if (all_units < gridDim.x) size = min(size, (total - all_units * EXTRA) / (gridDim.x - all_units) + 1u);
            size = max(size, least);
            if (size + worth >= most) size = most;
        }
        if (size == most ? most <= each + worth : size <= each) {
            const uint32_t cuts = (cost + size - 1u) / size, ends = up_to(cuts * a.c.kv_heads);
            const uint32_t mine = __ballot_sync(0xffffffffu, ends > blockIdx.x);
            if (!mine) return p;
            const int l = __ffs((int)mine) - 1;
            const uint32_t own_cuts = __shfl_sync(0xffffffffu, cuts, l), c = __shfl_sync(0xffffffffu, cost, l);
            const uint32_t at = blockIdx.x - (__shfl_sync(0xffffffffu, ends, l) - own_cuts * a.c.kv_heads);
            p.s = __shfl_sync(0xffffffffu, seq, l);
            p.i = __shfl_sync(0xffffffffu, tile, l);
            p.h = at / own_cuts;
            p.behind = at - p.h * own_cuts;
            // as even as can be
            const uint32_t even = c / own_cuts, more = c - even * own_cuts;
            p.skip = p.behind * even + min(p.behind, more);
            p.left = even + (p.behind < more ? 1u : 0u);
            return p;
        }
    }
    p.each = each;
    const uint32_t at = each * blockIdx.x;
    if (at >= total) return p;
    uint32_t before = 0u;
    if (n > 1u) {
        p.s = (uint32_t)__ffs((int)__ballot_sync(0xffffffffu, lane < n && line > at)) - 1u;
        before = __shfl_sync(0xffffffffu, line, p.s ? (int)p.s - 1 : 0);
        if (p.s == 0u) before = 0u;
    }
    const uint32_t of_head = __shfl_sync(0xffffffffu, work, (int)p.s);
    p.h = (at - before) / of_head;
    p.begin = at;
    p.left = min(each, total - at);
    enter_unit(cut, p, at - before - of_head * p.h);
    return p;
}

// The same for any number of sequences; by all WARPS warps together through `sm`, which is free again behind the call. Units are
// pieces of their own, or the line is cut.
template <uint32_t WARPS, uint32_t KEYS, uint32_t EXTRA>
__device__ __forceinline__ Piece find_together(const Cut<KEYS, EXTRA> &cut, PieceSmem &sm, uint32_t least, uint32_t worth)
{
    const AttnArgs &a = cut.a;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u, n = a.c.nseq;
    Piece p;
    p.s = p.h = p.i = p.skip = 0u;
    p.begin = p.each = 0u;
    p.behind = 0u;
    p.shared = 1u;
    p.left = 0u;
    uint32_t most = 0u;
    for (uint32_t s = warp; s < n; s += WARPS) {
        const Seq q = cut.open(s);
        const uint64_t sum = cut.all(q, most);
        if (lane == 0u) {
            sm.work[s] = sum;
            sm.units[s] = q.rows ? cut.units(q) : 0u;
        }
    }
    if (lane == 0u) sm.most[warp] = most;
    __syncthreads();
    most = __reduce_max_sync(0xffffffffu, lane < WARPS ? sm.most[lane] : 0u);
    if (warp == 0u) {
        uint64_t work = 0u, units = 0u;
        for (uint32_t b = 0u; b < n; b += 32u) {
            const uint64_t w = up_to(b + lane < n ? sm.work[b + lane] * a.c.kv_heads : 0u), u = up_to((uint64_t)(b + lane < n ? sm.units[b + lane] : 0u) * a.c.kv_heads);
            if (b + lane < n) {
                sm.work[b + lane] = work + w;
                sm.units[b + lane] = (uint32_t)(units + u);
            }
            work += __shfl_sync(0xffffffffu, w, 31);
            units += __shfl_sync(0xffffffffu, u, 31);
        }
        if (lane == 0u) sm.all_units = units >> 32 ? ~0u : (uint32_t)units;
    }
    __syncthreads();
    const uint64_t total = sm.work[n - 1u];
    const uint32_t all_units = sm.all_units;
    p.each = quotient(total + gridDim.x - 1u, gridDim.x);
    const bool whole = all_units <= gridDim.x && most <= p.each + worth;
    // the sequence that place `at` is in, by the sums up to each one
    auto find = [&](auto at, const auto *sums) {
        uint32_t lo = 0u, hi = n - 1u;   // sums[hi] > at
        while (lo < hi) {
            const uint32_t mid = (lo + hi) >> 1;
            if (sums[mid] > at) hi = mid;
            else lo = mid + 1u;
        }
        return lo;
    };
    uint64_t before = 0u, of_head = 1u;
    uint32_t before_units = 0u;
    if (whole) {
        if (blockIdx.x < all_units) {
            p.s = find(blockIdx.x, sm.units);
            before_units = p.s ? sm.units[p.s - 1u] : 0u;
        }
    } else {
        p.each = max(p.each, (uint64_t)least);
        p.begin = p.each * blockIdx.x;
        if (p.begin < total) {
            p.left = min(p.each, total - p.begin);
            p.s = find(p.begin, sm.work);
            before = p.s ? sm.work[p.s - 1u] : 0u;
            of_head = quotient(sm.work[p.s] - before, a.c.kv_heads);
        }
    }
    __syncthreads();                      // `sm` is free
    if (whole ? blockIdx.x >= all_units : !p.left) return p;
    if (whole) {
        const Seq q = cut.open(p.s);
        const uint32_t units = cut.units(q);
        p.h = (blockIdx.x - before_units) / units;
        p.i = blockIdx.x - before_units - p.h * units;
        p.left = cut.cost(q, p.i);
    } else {
        p.h = (uint32_t)quotient(p.begin - before, of_head);
        enter_unit(cut, p, p.begin - before - of_head * p.h);
    }
    return p;
}

// Walks over the units of a piece, MOST tiles of keys at a time. The whole warp.
template <uint32_t KEYS, uint32_t EXTRA, uint32_t MOST = 0x7fffffffu>
struct Walk {
    const Cut<KEYS, EXTRA> &cut;
    Piece p;
    Seq q;
    uint32_t k_begin, k_end;              // the step's tiles of keys of the current unit
    bool head, tail;                      // the unit's first tile is in the piece, and its last in the step
    bool first;                           // it is the piece's first unit
    bool again;                           // there were steps of the unit before in this piece

    __device__ __forceinline__ Walk(const Cut<KEYS, EXTRA> &cut_, const Piece &p_) : cut(cut_), p(p_), first(true), again(false)
    {
        if (p.left) {
            q = cut.open(p.s, p.kept);
            set();
        }
    }
    __device__ __forceinline__ bool more() const { return p.left != 0u; }
    __device__ __forceinline__ uint32_t row0() const { return p.i * cut.tile; }
    __device__ __forceinline__ uint32_t rows() const { return min(q.rows - row0(), cut.tile); }
    __device__ __forceinline__ void set()
    {
        const uint32_t all = cut.cost(q, p.i);
        if (!again) head = p.skip == 0u;
        k_begin = q.k0 + p.skip;
        const uint32_t n = (uint32_t)min((uint64_t)min(all - p.skip, MOST), p.left);
        k_end = k_begin + n;
        tail = p.skip + n == all;
    }
    __device__ __forceinline__ void next()
    {
        p.left -= k_end - k_begin;
        if (!tail && p.left) {
            p.skip += k_end - k_begin;
            again = true;
            set();
            return;
        }
        p.skip = 0u;
        first = again = false;
        p.left -= min(p.left, (uint64_t)EXTRA);
        if (!p.left) return;
        if (++p.i >= cut.units(q)) {
            p.i = 0u;
            if (++p.h >= cut.a.c.kv_heads) {
                p.h = 0u;
                do q = cut.open(++p.s, p.kept);
                while (!q.rows);          // there is more, so a sequence with rows comes
            }
        }
        set();
    }
    // where this piece's part of a cut unit goes
    __device__ __forceinline__ uint32_t record() const { return 2u * blockIdx.x + (first ? 0u : 1u); }
    // nothing of the unit follows in this piece
    __device__ __forceinline__ bool leaves() const { return tail || p.left == k_end - k_begin; }
    // what the merge has to know: of the piece's first unit, if others began it and it ends here. Before the first next().
    __device__ __forceinline__ Part part() const
    {
        Part r{};
        r.first = ~0u;
        if (p.left && !head && cut.cost(q, p.i) - p.skip <= p.left) {
            uint32_t c = blockIdx.x - p.behind;
            r.first = 2u * c;
            if (p.each) {
                const uint64_t unit = p.begin - p.skip;   // the place of its first tile of keys
                c = (uint32_t)quotient(unit, p.each);
                r.first = 2u * c + (unit - p.each * c <= EXTRA ? 0u : 1u);
            }
            r.count = blockIdx.x - c + 1u;
            r.s = p.s;
            r.h = p.h;
            r.row0 = row0();
            r.rows = rows();
        }
        return r;
    }
};

__device__ __forceinline__ float *record_of(const AttnArgs &a, uint32_t i, uint32_t rows)
{
    return a.parts + kPartsBytes / 4u + (size_t)i * record_floats(rows);
}

// What a state (maximum, sum) counts against the maximum M; one that saw no position counts nothing, one of NaN stays
__device__ __forceinline__ float factor(float2 s, float M) { return s.x == -INFINITY ? (s.y == 0.f ? 0.f : 1.f) : ex2(s.x - M); }

// Four dimensions of an output row
template <bool BF>
__device__ __forceinline__ void store4(const AttnArgs &a, uint32_t s, uint32_t h, uint2 at, uint32_t d4, float4 x)
{
    reinterpret_cast<uint2 *>(a.out + ((size_t)s * a.r.tokens + at.x) * a.ldo + (size_t)(h * a.group + at.y) * kDim)[d4] =
        make_uint2(pack<BF>(x.x, x.y), pack<BF>(x.z, x.w));
}

// Whether a warp's lanes can keep the call's sequences: see kKeptSeqs. Units of `tile` rows, and tiles of `keys` positions.
inline bool lanes_keep(const AttnArgs &a, uint32_t tile, uint32_t keys, uint32_t extra)
{
    const uint64_t units = ((uint64_t)a.r.tokens * a.group + tile - 1u) / tile, line = units * a.c.nseq * a.c.kv_heads;
    return a.c.nseq <= kKeptSeqs && line < (1ull << 31) && line * ((a.c.limit + keys - 1u) / keys + extra) < (1ull << 31);
}

// Whatever the positions, each unit will be a piece of its own (find_kept, find_together), of a CTA or a cluster: a sequence has room for no
// more
inline bool always_whole(const AttnArgs &a, uint64_t units, uint32_t ctas, uint32_t keys, uint32_t worth, uint32_t cluster = 1)
{
    if (cluster > 1 && units * cluster <= ctas && ((a.c.limit + keys - 1u) / keys + cluster - 1u) / cluster <= worth) return true;
    return units <= ctas && (!a.keep || units <= 32ull * a.c.kv_heads) && (a.c.limit + keys - 1u) / keys <= worth;
}

}  // namespace

// paged_attn.cu: joins the partial sums of units of `rows` rows
cudaError_t launch_merge(const AttnArgs &a, bool bf, uint32_t rows, uint32_t ctas, int sms, cudaStream_t stream);

}  // namespace paged
}  // namespace atlas
