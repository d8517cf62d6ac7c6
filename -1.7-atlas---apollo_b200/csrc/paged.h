// Host/device description of the paged KV cache operators (paged.cu,
// paged_attn.cu; public interface in include/atlas_cuda.h).
//
// Pool of all layers, caller-owned device memory:
//   k, v    binary16 or bfloat16 [layer][page][kv_head][position in the page][128]
//   table   int32 [seq][max_pages]: the page of each run of `page` positions;
//           a number that is no page's: none
//   refs    int32 [page]: how many entries name it; 0: free
//   work    what the calls on the pages write: WorkHead, lists of pages, then
//           the attention's partial sums
#pragma once
#include <cstdint>
#include <cuda_runtime.h>

namespace atlas {
namespace paged {

constexpr uint32_t kDim = 128;            // head dimension
constexpr uint32_t kRowBytes = 2 * kDim;
constexpr uint32_t kMaxSeqs = 4096;
constexpr uint32_t kMaxCtas = 160;        // of an attention call: its partial sums have room for so many

struct Cache {
    uint16_t *k, *v;
    int32_t *table, *refs;
    uint32_t *work;
    uint32_t layers, pages, kv_heads, page_log2, nseq, max_pages;
    uint32_t limit;                       // positions that a sequence may have: max_pages << page_log2
};

// A call's token rows: sequence s has n_tok[s] (null: `tokens`) of the
// `tokens` rows, at positions pos0[s] ..
struct Rows {
    const uint32_t *pos0, *n_tok;
    uint32_t tokens;
};

// In the workspace: what the call that changes the table left for the one that
// moves the rows
struct WorkHead {
    uint32_t copies;                      // pages to copy
    uint32_t from;                        // pages numbered from here on have moved (compact)
    uint32_t pad[14];
};
// Then arrays of `pages` words: the copies, and what the plans need between their steps
enum WorkArray : uint32_t { kCopyFrom, kCopyTo, kCopyRows, kWriters, kLastWriter, kFresh, kWorkArrays };
constexpr uint32_t kMovedTo = kWriters;  // compact: the new number of a page that has moved

// Division by a number known at the launch: for x < 2^31, x * m >> (31 + L) is x / d, where 2^L >= d and m = ceil(2^(31 + L) / d)
// < 2^32 (m d exceeds 2^(31 + L) by less than d, so x m / 2^(31 + L) exceeds x / d by less than 2^-L <= 1 / d)
struct Divisor {
    uint32_t m, shift;                    // shift: L
};
inline Divisor divisor(uint32_t d)
{
    uint32_t l = 0;
    while ((1ull << l) < d) ++l;
    return Divisor{(uint32_t)(((1ull << (31u + l)) + d - 1u) / d), l};
}
__device__ __forceinline__ uint32_t divide(uint32_t x, const Divisor &d)
{
    return (uint32_t)((uint64_t)x * d.m >> 31) >> d.shift;
}

struct AttnArgs {
    Cache c;
    Rows r;
    const uint16_t *q;                    // [seq][tokens][q_heads][128], ldq elements between tokens
    uint16_t *out;
    uint64_t ldq, ldo;
    uint32_t q_heads, group, layer;
    Divisor by_group;
    float *parts;                         // partial sums: see Part
    uint32_t keep;                        // a warp's lanes keep the sequences' state
    uint32_t early;                       // the successor may start at once
};

__device__ __forceinline__ uint32_t row_count(const Rows &r, uint32_t s)
{
    return r.n_tok ? min(__ldcg(r.n_tok + s), r.tokens) : r.tokens;
}

}  // namespace paged
}  // namespace atlas
