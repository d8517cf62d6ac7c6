// Host/device description of the 8-bit KV cache operators (kv8.cu,
// kv8_prompt.cu; public interface in include/atlas_cuda.h).
//
// Cache of one layer, caller-owned device memory:
//   k, v              int8 codes [seq][kv_head][max_context][128]
//   k_scale, v_scale  fp32 [seq][kv_head][n_blocks]; value = code * scale of
//                     the block of 16, 32, 64 or 128 positions
//   k_sum             int16 [seq][kv_head][n_blocks][128]: sums of the K codes
//                     of each block (what the block scores are made from)
#pragma once
#include <cstdint>
#include <cuda_runtime.h>

namespace atlas {
namespace k8 {

constexpr uint32_t kDim = 128;        // head dimension
constexpr uint32_t kChunk = 16;       // positions a warp takes at a time: never across a block's end

struct Cache {
    int8_t *k, *v;
    float *k_scale, *v_scale;
    int16_t *k_sum;                   // may be null (no block selection)
    uint32_t nseq, kv_heads, max_context, block_log2, n_blocks;
};

// A call's token rows: sequence s has n_tok[s] (null: `tokens`) of the
// `tokens` rows, at positions pos0[s] ..
struct Rows {
    const uint32_t *pos0, *n_tok;
    uint32_t tokens;
};

struct AttnArgs {
    Cache c;
    Rows r;
    const float *q;                   // [seq][tokens][q_heads][128], ldq floats between tokens
    float *out;
    uint64_t ldq, ldo;
    uint32_t q_heads, group;
    float group_inv;                  // 1 / group, a little high
    uint32_t tiles;                   // row tiles per (sequence, KV head) - or per (sequence, KV head, token)
    uint32_t n_sel;                   // block selection: blocks per token and KV head
    int32_t *sel;                     // [seq][tokens][kv_heads][n_sel]
    uint32_t early;                   // the successor may start at once
};

// The prompt form's tiles of 128 rows per CTA, CTAs that share a unit's positions, and estimated time
struct PromptCut {
    uint32_t tiles, split;
    uint64_t cycles;
};

__device__ __forceinline__ uint32_t row_count(const Rows &r, uint32_t s)
{
    return r.n_tok ? min(__ldcg(r.n_tok + s), r.tokens) : r.tokens;
}

}  // namespace k8
}  // namespace atlas
