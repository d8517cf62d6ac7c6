// Attention of prompts over the 8-bit KV cache on tcgen05 tensor cores
// (sm_100a): kv8_attn's form for many query rows (gqa_single_token per token
// in the reference, src/brain_runtime.c:1407-1528).
//
// A CTA takes 256 query rows of one KV head (row r = token * group + head, so
// the group's heads share every key), as two tiles of 128 rows, and walks the
// cached positions 128 at a time:
//   S = Q K^T   tcgen05.mma kind::f16, M = 128, N = 128 keys, K = 128
//   O += P V    M = 128, N = 128 dimensions, K = 128 keys, P from tensor memory
// The codes of K and V are exact in binary16. Q (after a power of two per row)
// and P enter as two binary16 terms hi + lo, 22 bits, summed in the same fp32
// accumulator: twice the products of a binary16 attention for fp32-level
// accuracy. The block scales of K multiply the scores, those of V the weights:
// P = 2^6 p v_scale over the row's largest p v_scale so far (a second running
// maximum, of the score plus the scale's logarithm), so that one accumulator
// serves blocks of different scales, and the row loses bits neither to blocks
// that it gives no weight nor to blocks that it does not see.
//
// Warps of a CTA (16):
//   0-7    softmax, four per tile, one thread per row: maximum and exponentials
//          of the scores straight from tensor memory, P back into the columns
//          that the scores leave; the maximum is lazy (raised only when a score
//          passes it by 2^8). Each tile of keys' output is added to the earlier
//          ones in these threads' registers, which the other warps leave them;
//   8-11   codes -> binary16 in 128-byte swizzled K-major tiles: K [key][dimension],
//          V transposed on the way, [dimension][key]; the next codes are on their
//          way by cp.async while the MMAs still read the current ones;
//   12     issues the MMAs: P V of a tile, then the next keys' scores of the
//          same tile, so that one tile's softmax runs under the other's MMAs.
// Where few rows leave SMs idle, a CTA takes one tile of 128 rows: both softmax
// groups then have the same rows and take turns at the tiles of keys, each with
// an output and a state of its own, which are merged at the end. The place of the
// second tile's Q holds a second buffer of K and one of V then, group 1's.
//
// Tensor cores truncate their sums: an MMA that adds to an output loses 2^-24 of
// it on average where the values have one sign, a fifth of that where they have
// not, and nothing where its weights are zeros. So only a tile of keys (16 MMAs)
// is summed in tensor memory and then added to the earlier ones with rounding.
// Over 1024 positions of one sign, sums of 1 / 2 / 8 tiles lose 17 / 31 / 130 x
// 2^-24, at most 33 / 55 / 253 (one position with most of the weight). Taking the
// outputs out after every tile costs no time, as it runs beside the next scores.
// (Two threads per row, with the sums of eight tiles in local memory: 512 tokens
// of 28 heads on 4 17.3 us where this takes 19.4, 8192 of 40 heads on 8 1165 and
// 1264, 333 over 5001 of 16 on 2 73 to 84 and 68 to 73; eight tiles are too many,
// and with two 8192 take 1557.)
// Tensor memory: 2 x 128 columns of scores / weights, 2 x 128 of output.
// Shared memory: Q hi / lo 128 KB, K 32 KB, V 32 KB, their next codes 32 KB; Q's
// place stages the output.
//
// Few rows over many positions: the positions are split over a cluster of CTAs,
// and each merges a share of the rows through distributed shared memory.
//
// Bound by the chain of a tile's scores, softmax and output with one thread per
// row, next to the MMAs, which need 4130 cycles for 256 rows x 128 keys. 8192
// tokens of 40 heads on 8 run 1264 us, 66 % of the measured binary16-rate peak
// for two products.
// Every wait is bounded; after a timeout the CTA's rows are NaN.
#include <algorithm>
#include <atomic>
#include <cfloat>
#include <cmath>
#include "../../include/atlas_cuda.h"
#include "kv8.cuh"
#include "tcgen05.cuh"

namespace atlas {
namespace k8 {
namespace {

constexpr uint32_t kTileRows = 128, kTileKeys = 128;
constexpr uint32_t kMaxSplit = 8;                  // CTAs that share the positions of a tile's rows
// Warps by number: eight of softmax, four converters, the one that issues the MMAs (and three that fill up its warpgroup)
constexpr uint32_t kConvWarp = 8, kMmaWarp = 12, kPromptThreads = 16 * 32;
// Registers per thread of a warpgroup after the split, of 128 at launch
constexpr uint32_t kSoftmaxRegs = 192, kConvertRegs = 72, kMmaRegs = 56;
static_assert(2 * kSoftmaxRegs + kConvertRegs + kMmaRegs == 4 * 128, "what two warpgroups get is what the others leave");
constexpr uint32_t kHalf = 128 * 128;              // bytes of 128 rows x 64 binary16, swizzled
constexpr uint32_t kQTile = 4 * kHalf;             // one tile's Q: [hi, lo][2 x 64 dimensions]

struct PromptBars {
    uint64_t s_full[2], p_full[2], o_full[2];                                       // [tile]
    uint64_t k_full[2][2], k_empty[2][2], v_full[2][2], v_empty[2][2], q_full, fin;   // [buffer][half]
    uint32_t tmem, status;
    // what a score of the row is worth, in the exponent's base 2 (in [tile][0]); one tile: then what the groups'
    // states are
    float state[2][2][kTileRows];
};

// In the place of the next codes once they are used up
struct RowStates {
    float max[2][kTileRows], sum[2][kTileRows];
};

constexpr size_t kRawTile = 128 * 128;             // bytes of 128 rows of codes
constexpr size_t kPromptSmem = 2 * kQTile + 4 * kHalf + 2 * kRawTile + sizeof(PromptBars);
static_assert(kPromptSmem <= kMaxSmem, "the tiles exceed a CTA's shared memory");

// fp32 accumulator, binary16 operands, K-major, M = 128, N = 128
constexpr uint32_t kInstr = (1u << 4) | ((128u >> 3) << 17) | ((128u >> 4) << 24);

__device__ __forceinline__ float4 ld_cluster4(const void *p, uint32_t cta)
{
    uint32_t r;
    float4 v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_addr(p)), "r"(cta));
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(r));
    return v;
}
__device__ __forceinline__ float ld_cluster1(const void *p, uint32_t cta)
{
    uint32_t r;
    float v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_addr(p)), "r"(cta));
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(r));
    return v;
}

// What a warp knows of a tile's 16-key groups: lane i has the scale of the K codes (i < 8) or V codes (8 <= i < 16) of
// group i % 8, and of V's the base-2 logarithm
struct Scales {
    float scale, log2;
};

// From this lane's scale. A V scale of 0 counts as fp32's smallest number, 2^-149.
__device__ __forceinline__ Scales scales_from(float x, uint32_t lane)
{
    Scales s;
    s.scale = x == 0.f && lane >= 8u ? __uint_as_float(1u) : x;
    s.log2 = __log2f(s.scale);
    if (s.log2 < -149.0f) s.log2 = -149.0f;
    return s;
}

constexpr int kGroups = kTileKeys / 16;

// A row's softmax over one tile of keys: scores at tensor memory `at` (this
// warp's lanes), what a unit of one is worth in `factor`, of which the row sees
// the first `nvis` keys (MASK; else all). Returns the largest score; in `mw`, the
// largest sum of a score and the logarithm of its V scale. The next 16 columns
// are on their way while 16 are worked on.
template <bool MASK>
__device__ __forceinline__ float tile_max(uint32_t at, const Scales &sc, float factor, int nvis, float &mw)
{
    float m = -INFINITY, s[2][16];
    mw = -INFINITY;
    tmem_ld(at, s[0]);
#pragma unroll
    for (int c = 0; c < kGroups; ++c) {
        float(&v)[16] = s[c & 1];
        const float f = __shfl_sync(0xffffffffu, sc.scale, c) * factor, lg = __shfl_sync(0xffffffffu, sc.log2, 8 + c);
        tmem_wait_ld(v);
        if (c + 1 < kGroups) tmem_ld(at + 16u * (uint32_t)(c + 1), s[(c + 1) & 1]);
        if (MASK)
#pragma unroll
            for (int i = 0; i < 16; ++i) v[i] = 16 * c + i < nvis ? v[i] : -INFINITY;
        const float x = max3(max3(max3(v[0], v[1], v[2]), max3(v[3], v[4], v[5]), max3(v[6], v[7], v[8])),
                             max3(v[9], v[10], v[11]), max3(max3(v[12], v[13], v[14]), v[15], v[15]));
        if (!MASK || x != -INFINITY) {
            m = fmaxf(m, x * f);
            mw = fmaxf(mw, fmaf(x, f, lg));
        }
    }
    return m;
}

// The weights into the scores' columns, 16 keys at a time: 8 columns of hi, 8
// of lo. They are 2^(score + log2 v_scale - ref), so their rounding is that of
// the group's sum, which returns without the V scale, times 2^k. A group with so
// small a scale that binary16 would hold nothing even of the row's largest
// weight takes a larger one, still small enough for that, so that the sum keeps
// its part.
template <bool MASK>
__device__ __forceinline__ float tile_weights(uint32_t at, const Scales &sc, float factor, int nvis, float ref, int k)
{
    float sum = 0.f, s[2][16];
    const uint64_t minus = pair(-1.0f, -1.0f);
    tmem_ld(at, s[0]);
#pragma unroll
    for (int c = 0; c < kGroups; ++c) {
        const float(&v)[16] = s[c & 1];
        const float f = __shfl_sync(0xffffffffu, sc.scale, c) * factor, lg = __shfl_sync(0xffffffffu, sc.log2, 8 + c);
        const float sv = __shfl_sync(0xffffffffu, sc.scale, 8 + c), least = (float)(k - 80);
        const float off = (lg < least ? least : lg) - ref;   // a NaN stays
        tmem_wait_ld(s[c & 1]);
        if (c + 1 < kGroups) tmem_ld(at + 16u * (uint32_t)(c + 1), s[(c + 1) & 1]);
        const uint64_t f2 = pair(f, f), off2 = pair(off, off);
        uint32_t p[16];
        uint64_t part = 0;
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
            float w0, w1;
            unpair(fma2(pair(v[i], v[i + 1]), f2, off2), w0, w1);
            w0 = ex2(w0);
            w1 = ex2(w1);
            if (MASK) {   // a masked position counts nothing, whatever its block's scales are
                w0 = 16 * c + i < nvis ? w0 : 0.f;
                w1 = 16 * c + i + 1 < nvis ? w1 : 0.f;
            }
            const uint64_t w = pair(w0, w1);
            part = add2(part, w);
            // the upper 11 bits are exact in binary16, but for weights below 2^-14
            const float h0 = __uint_as_float(__float_as_uint(w0) & 0xffffe000u), h1 = __uint_as_float(__float_as_uint(w1) & 0xffffe000u);
            float l0, l1;
            unpair(fma2(pair(h0, h1), minus, w), l0, l1);
            p[i / 2] = h2_bits(h0, h1);
            p[8 + i / 2] = h2_bits(l0, l1);
        }
        float a0, a1;
        unpair(part, a0, a1);
        if (!MASK || 16 * c < nvis) {
            // 2^k / v_scale by halves: either may pass fp32's range
            const int k0 = k / 2, k1 = k - k0;
            const float r = rcp(sv * __int_as_float((127 - k0) << 23) * __int_as_float((127 - k1) << 23));
            sum = fmaf(a0 + a1, lg < least ? 0x1p80f : r, sum);
        }
        tmem_st(at + 16u * (uint32_t)c, p);
    }
    return sum;
}

// The integer below x; 0 for none
__device__ __forceinline__ int below(float x) { return x == x ? (int)fminf(fmaxf(floorf(x), -250.0f), 250.0f) : 0; }

__device__ __forceinline__ void copy16(uint32_t dst, const void *src, bool there)   // zeros where !there
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16u : 0u) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ void copy_wait1() { asm volatile("cp.async.wait_group 1;" ::: "memory"); }
__device__ __forceinline__ void copy_wait0() { asm volatile("cp.async.wait_group 0;" ::: "memory"); }

template <bool ONE>
__global__ void __launch_bounds__(kPromptThreads, 1) prompt_kernel(const __grid_constant__ AttnArgs a)
{
    extern __shared__ __align__(1024) uint8_t prompt_smem[];
    uint8_t *const qs = prompt_smem, *const ks = qs + 2 * kQTile, *const vs = ks + 2 * kHalf, *const raw = vs + 2 * kHalf;
    PromptBars &b = *reinterpret_cast<PromptBars *>(raw + 2 * kRawTile);
    RowStates &rs = *reinterpret_cast<RowStates *>(raw);
    volatile uint32_t *const err = &b.status;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
    const uint32_t C = cluster_size(), rank = cluster_rank(), s = blockIdx.z, h = blockIdx.y;
    // the last rows first: they see the most positions
    const uint32_t r0 = (a.tiles - 1u - blockIdx.x / C) * (ONE ? 1u : 2u) * kTileRows;
    TileRows tr{r0 / a.group, 0u, a.group, a.group_inv};
    tr.rem = r0 - tr.tok * a.group;
    if (threadIdx.x == 0) {
        for (int t = 0; t < 2; ++t) {
            mbar_init(&b.s_full[t], 1u);
            mbar_init(&b.p_full[t], 4u);
            mbar_init(&b.o_full[t], 1u);
            for (int hf = 0; hf < 2; ++hf) {
                mbar_init(&b.k_full[t][hf], 4u);
                mbar_init(&b.v_full[t][hf], 2u);
                mbar_init(&b.k_empty[t][hf], 1u);
                mbar_init(&b.v_empty[t][hf], 1u);
            }
        }
        mbar_init(&b.q_full, kConvWarp);
        mbar_init(&b.fin, 1u);
        b.status = kStatusOk;
        fence_mbar_init();
    }
    if (warp == kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&b.tmem)), "r"(512u)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = b.tmem;   // scores / weights of tile t: column 128 t; output: 256 + 128 t
    wait_predecessor(a.early);
    const uint64_t p0 = __ldcg(a.r.pos0 + s);
    const uint32_t all = row_count(a.r, s) * a.group;
    if (r0 >= all) {   // the whole cluster leaves
        if (warp == kMmaWarp) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
        return;
    }
    const uint32_t rows = min(all - r0, (ONE ? 1u : 2u) * kTileRows), tiles = rows > kTileRows ? 2u : 1u;
    const uint32_t limit = (uint32_t)min(p0 + tr.at(rows - 1u).x + 1u, (uint64_t)a.c.max_context);
    const uint32_t total = (limit + kTileKeys - 1u) / kTileKeys;
    uint32_t j0 = 0u, n = total;   // this CTA's tiles of keys
    if (C > 1u) {
        const uint32_t base = total / C, more = total - base * C;
        j0 = rank * base + min(rank, more);
        n = base + (rank < more ? 1u : 0u);
    }
    const size_t head = (size_t)s * a.c.kv_heads + h;
    // K's and V's buffer for tile of keys j, and how often it was used before
    auto buffer = [&](uint32_t j) { return ONE ? j & 1u : 0u; };
    auto uses = [&](uint32_t j) { return ONE ? j >> 1 : j; };
    uint8_t *const ks2 = qs + kQTile, *const vs2 = ks2 + 2 * kHalf;

    float row_m = -INFINITY, row_l = 0.f;   // softmax threads: their row's state, for the cluster

    // The end of a CTA, for every warp in the branch of its registers
    auto leave = [&]() {
        fence_before();
        __syncthreads();
        if (warp == kMmaWarp) {
            fence_after();
            asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
        }
    };
    auto merge = [&]() {
        // the converters' slots are free now
        rs.max[warp >> 2][(warp & 3u) * 32u + lane] = row_m;
        rs.sum[warp >> 2][(warp & 3u) * 32u + lane] = row_l;
        // Rows rank, rank + C, ... of the cluster's states, four at a time per warp:
        // lane = (row, CTA) for the maxima and sums, then 4 dimensions. A state that
        // saw no position counts nothing.
        static_assert(kMaxSplit == 8, "eight lanes per row");
        cluster_sync();
        for (uint32_t k0 = 4u * warp; rank + C * k0 < rows; k0 += 4u * kConvWarp) {
            // two CTAs' outputs are on their way meanwhile
            float4 y[2][4];
            auto load = [&](float4(&to)[4], uint32_t c) {
#pragma unroll
                for (uint32_t v = 0; v < 4; ++v) {
                    const uint32_t r = min(rank + C * (k0 + v), rows - 1u), row = r & (kTileRows - 1u);
                    to[v] = ld_cluster4(reinterpret_cast<const float4 *>(qs + (r / kTileRows) * kQTile) + row * 32u + (lane ^ (row & 31u)), c);
                }
            };
            auto add = [&](float4(&x)[4], const float4(&from)[4], float f, uint32_t c) {
#pragma unroll
                for (int v = 0; v < 4; ++v) {
                    const float fc = __shfl_sync(0xffffffffu, f, 8 * v + (int)c);
                    x[v].x = fmaf(fc, from[v].x, x[v].x);
                    x[v].y = fmaf(fc, from[v].y, x[v].y);
                    x[v].z = fmaf(fc, from[v].z, x[v].z);
                    x[v].w = fmaf(fc, from[v].w, x[v].w);
                }
            };
            load(y[0], 0u);
            load(y[1], 1u);
            const uint32_t u = lane >> 3, cta = lane & 7u, i = rank + C * (k0 + u);
            const bool there = cta < C && i < rows;
            const float mc = there ? ld_cluster1(&rs.max[i / kTileRows][i & (kTileRows - 1u)], cta) : -INFINITY;
            const float lc = there ? ld_cluster1(&rs.sum[i / kTileRows][i & (kTileRows - 1u)], cta) : 0.f;
            const bool bad = there && __float_as_uint(ld_cluster1(&b.status, cta)) != kStatusOk;
            float M = mc;
#pragma unroll
            for (int o = 4; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
            const float f = mc == -INFINITY && lc == 0.f ? 0.f : ex2(mc - M);
            float L = f * lc;
#pragma unroll
            for (int o = 4; o > 0; o >>= 1) L += __shfl_xor_sync(0xffffffffu, L, o);
            const bool any_bad = __any_sync(0xffffffffu, bad);
            float4 x[4];
#pragma unroll
            for (int v = 0; v < 4; ++v) x[v] = make_float4(0.f, 0.f, 0.f, 0.f);
            for (uint32_t c = 0; c < C; c += 2u) {
                add(x, y[0], f, c);
                if (c + 2u < C) load(y[0], c + 2u);
                if (c + 1u < C) add(x, y[1], f, c + 1u);
                if (c + 3u < C) load(y[1], c + 3u);
            }
#pragma unroll
            for (uint32_t v = 0; v < 4; ++v) {
                const uint32_t r = rank + C * (k0 + v);
                const float sum = __shfl_sync(0xffffffffu, L, 8 * v);
                if (r >= rows) continue;
                const uint2 at = tr.at(r);
                const float inv = any_bad || p0 + at.x >= a.c.max_context ? __int_as_float(0x7fffffff) : (1.0f / kOutUnit) / sum;
                reinterpret_cast<float4 *>(a.out + ((size_t)s * a.r.tokens + at.x) * a.ldo + (size_t)(h * a.group + at.y) * kDim)[lane] =
                    make_float4(x[v].x * inv, x[v].y * inv, x[v].z * inv, x[v].w * inv);
            }
        }
        cluster_sync();   // no CTA leaves while the cluster may read its states
    };

    auto leave_unmerged = [&]() {   // the warps that have left their registers to the others
        leave();
        if (C > 1u) {
            cluster_sync();
            cluster_sync();
        }
    };
    if (warp >= kMmaWarp) {
        // ------------------------------------------------------------- MMA --
        fewer_registers<kMmaRegs>();
        if (warp == kMmaWarp && elected()) {
            // a step of 16 along K is 32 bytes, 2 in a descriptor; 4 steps fill a swizzled tile
            const uint64_t qd = operand(smem_addr(qs)), kd[2] = {operand(smem_addr(ks)), operand(smem_addr(ks2))},
                           vd[2] = {operand(smem_addr(vs)), operand(smem_addr(vs2))};
            // K and V go by halves (64 dimensions, 64 keys): a half is converted
            // while the MMAs still read, or already read, the other.
            bool ok = n != 0u && mbar_wait(&b.q_full, 0u, err);
            // scores of keys j against Q tile `qt` into S of group t; P V of keys j into the group's output
            auto scores = [&](uint32_t t, uint32_t qt, uint32_t j, bool first_use, bool last_use) {
                const uint64_t q = qd + (uint64_t)(qt * (kQTile >> 4)), k = buffer(j) ? kd[1] : kd[0];
#pragma unroll
                for (uint32_t hf = 0; hf < 2u; ++hf) {
                    if (first_use) {
                        if (!(ok = ok && mbar_wait(&b.k_full[buffer(j)][hf], uses(j) & 1u, err))) return;
                        fence_after();
                    }
#pragma unroll
                    for (uint32_t st = 0; st < 4u; ++st) {
                        const uint32_t off = hf * (kHalf >> 4) + st * 2u;
                        mma_ss(tmem + 128u * t, q + off, k + off, kInstr, hf != 0u || st != 0u);
                        mma_ss(tmem + 128u * t, q + (2u * kHalf >> 4) + off, k + off, kInstr, 1u);
                    }
                    if (last_use) commit(&b.k_empty[buffer(j)][hf]);
                }
                commit(&b.s_full[t]);
            };
            auto output = [&](uint32_t t, uint32_t j, uint32_t turn, bool first_use, bool last_use) {
                if (!(ok = ok && mbar_wait(&b.p_full[t], turn & 1u, err))) return;
#pragma unroll
                for (uint32_t hf = 0; hf < 2u; ++hf) {
                    if (first_use && !(ok = ok && mbar_wait(&b.v_full[buffer(j)][hf], uses(j) & 1u, err))) return;
                    fence_after();
#pragma unroll
                    for (uint32_t st = 0; st < 4u; ++st) {
                        const uint64_t v = (buffer(j) ? vd[1] : vd[0]) + hf * (kHalf >> 4) + st * 2u;
                        const uint32_t p = tmem + 128u * t + 64u * hf + 16u * st;
                        mma_ts(tmem + 256u + 128u * t, p, v, kInstr, hf != 0u || st != 0u);
                        mma_ts(tmem + 256u + 128u * t, p + 8u, v, kInstr, 1u);
                    }
                    if (last_use) commit(&b.v_empty[buffer(j)][hf]);
                }
            };
            if (ONE) {   // the groups take turns at the keys
                for (uint32_t j = 0; ok && j < min(n, 2u); ++j) scores(j, 0u, j, true, true);
                for (uint32_t j = 0; ok && j < n; ++j) {
                    output(j & 1u, j, j >> 1, true, true);
                    if (!ok) break;
                    commit(&b.o_full[j & 1u]);
                    if (j + 2u < n) scores(j & 1u, 0u, j + 2u, true, true);
                }
            } else {
                for (uint32_t t = 0; ok && t < tiles; ++t) scores(t, t, 0u, t == 0u, t + 1u == tiles);
                for (uint32_t j = 0; ok && j < n; ++j) {
                    for (uint32_t t = 0; ok && t < tiles; ++t) {
                        output(t, j, j, t == 0u, t + 1u == tiles);
                        if (!ok) break;
                        commit(&b.o_full[t]);
                        if (j + 1u < n) scores(t, t, j + 1u, t == 0u, t + 1u == tiles);
                    }
                }
            }
            // nothing of this CTA is left in flight when tensor memory is freed
            commit(&b.fin);
            const uint64_t t0 = global_ns();
            while (!mbar_try_wait(&b.fin, 0u) && global_ns() - t0 < kWaitLimitNs) {
            }
        }
        __syncwarp();
        leave_unmerged();
        return;
    } else if (warp >= kConvWarp) {
        fewer_registers<kConvertRegs>();
        // ------------------------------------------------------- converters --
        // K: a thread takes 16 dimensions of 8 keys (8 lanes write the same
        // chunk of 8 rows); V: 8 keys x 16 dimensions (8 lanes write the 8
        // chunks of a row): neither has a bank conflict. A thread copies just
        // the codes that it converts, into slots [piece][thread].
        const uint32_t w = warp - kConvWarp, l8 = lane & 7u, q8 = lane >> 3;
        const int8_t *ksrc = a.c.k + (head * a.c.max_context + 8u * w + l8) * kDim + 16u * q8;
        const uint32_t kg = l8 + 8u * (w >> 1), dg = q8 + 4u * (w & 1u);
        const int8_t *vsrc = a.c.v + (head * a.c.max_context + 8u * kg) * kDim + 16u * dg;
        uint4 *const kslot = reinterpret_cast<uint4 *>(raw) + (w * 32u + lane), *const vslot = kslot + kRawTile / 16u;
        auto copy_k = [&](uint32_t j) {
            if (j < n) {
                const uint32_t key0 = (j0 + j) * kTileKeys;
#pragma unroll
                for (uint32_t i = 0; i < 8; ++i) {
                    const uint32_t row = 32u * (i >> 1);
                    copy16(smem_addr(kslot + 128u * i), ksrc + (size_t)(key0 + row) * kDim + 64u * (i & 1u),
                           key0 + row + 8u * w + l8 < limit);
                }
            }
            copy_commit();
        };
        auto copy_v = [&](uint32_t j) {
            if (j < n) {
                const uint32_t key0 = (j0 + j) * kTileKeys;
#pragma unroll
                for (uint32_t i = 0; i < 8; ++i)
                    copy16(smem_addr(vslot + 128u * i), vsrc + (size_t)(key0 + i) * kDim, key0 + 8u * kg + i < limit);
            }
            copy_commit();
        };
        copy_k(0u);
        copy_v(0u);
        for (uint32_t j = 0; j < n; ++j) {
            const uint32_t buf = buffer(j), used = uses(j);
            copy_wait1();   // K of this tile; V may still be on its way
            bool ok = true;
#pragma unroll
            for (uint32_t hf = 0; hf < 2u; ++hf) {
                if (used && !(ok = ok && wait_warp(&b.k_empty[buf][hf], (used - 1u) & 1u, err))) break;
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) {
                    const uint32_t row = 32u * i + 8u * w + l8;
                    const uint4 x = kslot[128u * (2u * i + hf)];
                    const uint32_t words[4] = {x.x, x.y, x.z, x.w};
                    uint32_t o[8];
#pragma unroll
                    for (int q = 0; q < 4; ++q) {   // two neighbouring dimensions, each in the low byte of a half
                        o[2 * q] = codes_h2<false>(__byte_perm(words[q], 0u, 0x4140u));
                        o[2 * q + 1] = codes_h2<false>(__byte_perm(words[q], 0u, 0x4342u));
                    }
                    uint8_t *dst = (buf ? ks2 : ks) + hf * kHalf;
                    *reinterpret_cast<uint4 *>(dst + swizzled(row, 2u * q8)) = make_uint4(o[0], o[1], o[2], o[3]);
                    *reinterpret_cast<uint4 *>(dst + swizzled(row, 2u * q8 + 1u)) = make_uint4(o[4], o[5], o[6], o[7]);
                }
                fence_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(&b.k_full[buf][hf]);
            }
            if (!ok) break;
            copy_k(j + 1u);
            copy_wait1();   // V of this tile; warps 0, 1 have its first 64 keys, 2, 3 the others
            if (used && !wait_warp(&b.v_empty[buf][w >> 1], (used - 1u) & 1u, err)) break;
            uint8_t *dst = (buf ? vs2 : vs) + (w >> 1) * kHalf;
            uint4 y[8];
#pragma unroll
            for (uint32_t i = 0; i < 8; ++i) y[i] = vslot[128u * i];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                uint32_t o[4][4];   // dimension 4 q + ., key pair
#pragma unroll
                for (int p = 0; p < 4; ++p) {
                    const uint4 &u = y[2 * p], &v = y[2 * p + 1];
                    const uint32_t lo = q == 0 ? u.x : q == 1 ? u.y : q == 2 ? u.z : u.w;
                    const uint32_t hi = q == 0 ? v.x : q == 1 ? v.y : q == 2 ? v.z : v.w;
                    const uint32_t e = __byte_perm(lo, hi, 0x5410u), f = __byte_perm(lo, hi, 0x7632u);
                    o[0][p] = codes_h2<false>(e);
                    o[1][p] = codes_h2<true>(e);
                    o[2][p] = codes_h2<false>(f);
                    o[3][p] = codes_h2<true>(f);
                }
#pragma unroll
                for (int d = 0; d < 4; ++d)
                    *reinterpret_cast<uint4 *>(dst + swizzled(16u * dg + 4u * (uint32_t)q + (uint32_t)d, l8)) =
                        make_uint4(o[d][0], o[d][1], o[d][2], o[d][3]);
            }
            fence_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(&b.v_full[buf][w >> 1]);
            copy_v(j + 1u);
        }
        copy_wait0();
        leave_unmerged();
        return;
    } else {
        more_registers<kSoftmaxRegs>();
        // --------------------------------------------------------- softmax --
        // First Q: a warp takes eight rows at a time, four per step (eight lanes a
        // row, rows 0 4 1 5 and 2 6 3 7: so two rows' swizzled chunks do not meet
        // in a bank). A power of two brings each row's largest value to [2^8, 2^9).
#pragma unroll 1
        for (uint32_t i0 = 8u * warp; i0 < tiles * kTileRows; i0 += 8u * kConvWarp) {
            const uint32_t l8 = lane & 7u, first = i0 + 4u * ((lane >> 3) & 1u) + (lane >> 4);
            float4 x[2][4];
#pragma unroll
            for (uint32_t u = 0; u < 2; ++u) {
                const uint2 r = tr.at(first + 2u * u);
                const float4 *src = reinterpret_cast<const float4 *>(a.q + ((size_t)s * a.r.tokens + r.x) * a.ldq + (size_t)(h * a.group + r.y) * kDim) + l8;
#pragma unroll
                for (uint32_t k = 0; k < 4; ++k) x[u][k] = first + 2u * u < rows ? __ldcg(src + 8u * k) : make_float4(0.f, 0.f, 0.f, 0.f);
            }
#pragma unroll
            for (uint32_t u = 0; u < 2; ++u) {
                const uint32_t i = first + 2u * u, row = i & (kTileRows - 1u);
                uint32_t mx = 0u;   // absolute values order as their bits do, NaN above infinity
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    mx = max(max(max(mx, __float_as_uint(x[u][k].x) & 0x7fffffffu), __float_as_uint(x[u][k].y) & 0x7fffffffu),
                             max(__float_as_uint(x[u][k].z) & 0x7fffffffu, __float_as_uint(x[u][k].w) & 0x7fffffffu));
#pragma unroll
                for (int o = 4; o > 0; o >>= 1) mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, o));
                const bool bad = mx >= 0x7f800000u;   // a non-finite value: every score of the row NaN
                const int e = max((int)(mx >> 23) - 127, -118);
                const float f = bad ? 0.f : __int_as_float((135 - e) << 23);
                if (l8 == 0u) b.state[i / kTileRows][0][row] = bad ? __int_as_float(0x7fffffff) : kScoreScale * __int_as_float((119 + e) << 23);
                uint8_t *q = qs + (i / kTileRows) * kQTile + (l8 & 1u) * 8u;
#pragma unroll
                for (uint32_t k = 0; k < 4; ++k) {
                    const float v[4] = {x[u][k].x * f, x[u][k].y * f, x[u][k].z * f, x[u][k].w * f};
                    float hi[4];
#pragma unroll
                    for (int c = 0; c < 4; ++c) hi[c] = bad ? 0.f : __uint_as_float(__float_as_uint(v[c]) & 0xffffe000u);
                    uint8_t *dst = q + (k >> 1) * kHalf + swizzled(row, (l8 >> 1) + 4u * (k & 1u));
                    *reinterpret_cast<uint2 *>(dst) = make_uint2(h2_bits(hi[0], hi[1]), h2_bits(hi[2], hi[3]));
                    *reinterpret_cast<uint2 *>(dst + 2 * kHalf) =
                        bad ? make_uint2(0u, 0u) : make_uint2(h2_bits(v[0] - hi[0], v[1] - hi[1]), h2_bits(v[2] - hi[2], v[3] - hi[3]));
                }
            }
        }
        fence_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(&b.q_full);
        meet(3u, 32u * kConvWarp);   // the rows' factors are there

        // One thread per row, with the output of the tiles of keys before the current one in registers. A warp whose wait
        // ran out goes on to the barriers, without touching tensor memory.
        const uint32_t t = warp >> 2, quarter = warp & 3u, row = quarter * 32u + lane, base = ONE ? 0u : t * kTileRows;
        if (ONE || t < tiles) {
            const uint32_t at = tmem + ((quarter * 32u) << 16) + 128u * t, i = base + row;
            const float factor = b.state[ONE ? 0u : t][0][row];
            const uint32_t open = (uint32_t)min(p0 + tr.at(base).x, (uint64_t)0x7fffffffu);
            const uint32_t last = i < rows ? (uint32_t)min(p0 + tr.at(i).x, (uint64_t)0x7fffffffu) : open;
            const float *scales = (lane & 8u ? a.c.v_scale : a.c.k_scale) + head * a.c.n_blocks;
            auto scale_of = [&](uint32_t j) {
                return __ldcg(scales + min(((j0 + j) * kTileKeys + 16u * (lane & 7u)) >> a.c.block_log2, a.c.n_blocks - 1u));
            };
            constexpr uint32_t j_step = ONE ? 2u : 1u;
            const uint32_t j_first = ONE ? t : 0u;
            // m: the row's largest score; mw: the largest score + logarithm of the V scale, against which weights are
            // taken; l: the sum of weights without their V scales, times 2^k, k the integer below mw - m that keeps it in
            // range
            float m = -INFINITY, l = 0.f, mw = -INFINITY, next = j_first < n ? scale_of(j_first) : 0.f;
            int k = 0;
            uint64_t acc[kDim / 2];   // two dimensions each
#pragma unroll
            for (int c = 0; c < (int)kDim / 2; ++c) acc[c] = 0ull;
            bool ok = true;
            auto take_output = [&](uint32_t turn) {
                ok = ok && wait_warp(&b.o_full[t], turn & 1u, err);
                fence_after();
                if (!ok) return;
                float o[2][16];
                tmem_ld(at + 256u, o[0]);
#pragma unroll
                for (int c = 0; c < 8; ++c) {
                    tmem_wait_ld(o[c & 1]);
                    if (c < 7) tmem_ld(at + 256u + 16u * (uint32_t)(c + 1), o[(c + 1) & 1]);
#pragma unroll
                    for (int d = 0; d < 8; ++d) acc[8 * c + d] = add2(acc[8 * c + d], pair(o[c & 1][2 * d], o[c & 1][2 * d + 1]));
                }
            };
            for (uint32_t j = j_first; j < n; j += j_step) {
                const uint32_t turn = j / j_step;
                if (turn) take_output(turn - 1u);   // while the next scores are made
                const Scales sc = scales_from(next, lane);
                if (j + j_step < n) next = scale_of(j + j_step);
                const uint32_t key0 = (j0 + j) * kTileKeys;
                const bool masked = key0 + kTileKeys - 1u > open;   // some row does not see all of the tile
                const int nvis = last < key0 ? 0 : (int)min(last - key0 + 1u, kTileKeys);
                ok = ok && wait_warp(&b.s_full[t], turn & 1u, err);
                fence_after();
                if (!ok) break;
                float xw;
                const float x = masked ? tile_max<true>(at, sc, factor, nvis, xw) : tile_max<false>(at, sc, factor, kTileKeys, xw);
                const float was = m, before = mw;
                if (x > m + kLazy) m = x;
                if (xw > mw + kLazy) mw = xw;
                if (m != was || mw != before) {
                    const int now = below(mw - m);
                    l *= was == -INFINITY ? 0.f : ex2(before - mw + (float)(now - k));
                    k = now;
                }
                if (__any_sync(0xffffffffu, mw != before)) {
                    const float fv = mw == before ? 1.0f : before == -INFINITY ? 0.f : ex2(before - mw);
                    const uint64_t fv2 = pair(fv, fv);
#pragma unroll
                    for (int c = 0; c < (int)kDim / 2; ++c) acc[c] = mul2(acc[c], fv2);
                }
                l += masked ? tile_weights<true>(at, sc, factor, nvis, mw - 6.0f, k)
                            : tile_weights<false>(at, sc, factor, kTileKeys, mw - 6.0f, k);
                tmem_wait_st();
                fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&b.p_full[t]);
            }
            if (j_first < n) take_output((n - 1u - j_first) / j_step);
            // output = acc 2^k / l; what is merged is taken against the largest score: both times 2^(mw - m), less the 2^6 of
            // the weights, and kOutUnit
            const float rest = m == -INFINITY ? 0.f : ex2(mw - m - (float)k) * 0x1p-6f;
            const float back = (ONE || C > 1u ? rest * kOutUnit : 1.0f / l) * ex2((float)k);
            row_m = m;
            row_l = l * rest;
            float4 *stage = reinterpret_cast<float4 *>(qs + t * kQTile);
#pragma unroll
            for (uint32_t c = 0; c < kDim / 4u; ++c) {
                float4 v;
                unpair(acc[2 * c], v.x, v.y);
                unpair(acc[2 * c + 1], v.z, v.w);
                stage[row * 32u + (c ^ (row & 31u))] = make_float4(v.x * back, v.y * back, v.z * back, v.w * back);
            }
            if constexpr (ONE) {
                // both groups' states of a row -> one, in the place of group 0's; a state that saw no position counts nothing
                meet(3u, 32u * kConvWarp);   // both groups have the rows' factors
                b.state[t][0][row] = row_m;
                b.state[t][1][row] = row_l;
                meet(3u, 32u * kConvWarp);
                const float m1 = b.state[t ^ 1u][0][row], l1 = b.state[t ^ 1u][1][row], M = fmaxf(row_m, m1);
                const float own = row_m == -INFINITY && row_l == 0.f ? 0.f : ex2(row_m - M), other = m1 == -INFINITY && l1 == 0.f ? 0.f : ex2(m1 - M);
                row_l = row_l * own + l1 * other;
                row_m = M;
                meet(3u, 32u * kConvWarp);
                b.state[t][0][row] = C > 1u ? own : own * (1.0f / kOutUnit) / row_l;
                meet(3u, 32u * kConvWarp);
            } else {
                meet(1u + t, 128u);
            }
            if (ONE || C == 1u) {
                const bool failed = *err != kStatusOk;
                const uint32_t each = ONE ? 16u : 32u, w0 = (ONE ? warp : quarter) * each;   // rows of the tile for this warp
                stage = reinterpret_cast<float4 *>(qs + (ONE ? 0u : t * kQTile));
#pragma unroll 8
                for (uint32_t i0 = w0; i0 < w0 + each; ++i0) {
                    const uint32_t at4 = i0 * 32u + (lane ^ (i0 & 31u));
                    float4 x = stage[at4];
                    if constexpr (ONE) {
                        const float4 y = reinterpret_cast<float4 *>(qs + kQTile)[at4];
                        const float f0 = b.state[0][0][i0], f1 = b.state[1][0][i0];
                        x = make_float4(x.x * f0 + y.x * f1, x.y * f0 + y.y * f1, x.z * f0 + y.z * f1, x.w * f0 + y.w * f1);
                        if (C > 1u) {
                            stage[at4] = x;
                            continue;
                        }
                    }
                    const uint2 r = tr.at(base + i0);
                    if (failed || p0 + r.x >= a.c.max_context) x.x = x.y = x.z = x.w = __int_as_float(0x7fffffff);
                    if (base + i0 < rows)
                        reinterpret_cast<float4 *>(a.out + ((size_t)s * a.r.tokens + r.x) * a.ldo + (size_t)(h * a.group + r.y) * kDim)[lane] = x;
                }
            }
        }
    }
    leave();
    if (C > 1u) merge();
}

// Lets the kernel take its shared memory; refuses a build of it whose launch has fewer registers than the warpgroups then
// ask for, as that would wait for good.
template <auto KERNEL>
cudaError_t prepare(int dev)
{
    static std::atomic<int> registers{0};
    int n = registers.load(std::memory_order_relaxed);
    if (!n) {
        cudaFuncAttributes at{};
        const cudaError_t e = cudaFuncGetAttributes(&at, KERNEL);
        if (e != cudaSuccess) return e;
        registers.store(n = at.numRegs, std::memory_order_relaxed);
    }
    if ((uint32_t)n * 4u < 2u * kSoftmaxRegs + kConvertRegs + kMmaRegs) return cudaErrorLaunchOutOfResources;
    return allow<KERNEL>(dev, (int)kPromptSmem);
}

}  // namespace

// How a call is cut up, and an estimate of its longest CTA's time in cycles
// (1.8 per ns, as few_cycles'). Two tiles per CTA, or one; and up to 8 CTAs per
// unit, two tiles of keys each at least. What does not fit the device at once
// takes two tiles and whole units; what does goes by the time: a tile of keys
// takes 5400 cycles with one tile of rows and 6900 with two, what is before and
// after 14500 and 18000, a merge of two tiles 10000 (of one, nothing that shows).
// Measured, us, tiles of rows x CTAs per unit: 333 tokens over 5001 positions of
// 16 heads on 2, one 132, two x 1 / 2 / 3 151 / 99 / 69; 512 tokens of 28 on 4,
// one 20.0, two 27.4 and 23.8; 256 over 2048, one x 1 / 2 43.8 / 35.0, two x 2 /
// 3 / 4 / 5 43.8 / 37.2 / 33.4 / 53.9 (28 clusters of 5 do not fit at once); 8 sequences of 40 on 8, 35 rows over 2000 and 16000
// positions, one x 2 32.7 and 196, two x 2 37.6 and 215. The positions are those
// that the cache has room for, not those of the call, which only the device knows:
// 512 tokens with room for 32768 take two x 2, 23.3 us.
PromptCut prompt_cut(const AttnArgs &a, int dev, int sms)
{
    auto at_once = [&](uint32_t t, uint32_t c) -> uint32_t {   // units of c CTAs; clusters do not fill all SMs
        if (c == 1) return (uint32_t)sms;
        const cudaError_t e = t == 1 ? prepare<prompt_kernel<true>>(dev) : prepare<prompt_kernel<false>>(dev);
        if (e != cudaSuccess) return 0u;   // the launch will say so
        return t == 1 ? clusters_at_once<prompt_kernel<true>>(dev, c, kPromptThreads, kPromptSmem)
                      : clusters_at_once<prompt_kernel<false>>(dev, c, kPromptThreads, kPromptSmem);
    };
    const uint32_t rows = a.r.tokens * a.group, keys = (a.c.max_context + kTileKeys - 1) / kTileKeys;
    const uint64_t heads = (uint64_t)a.c.kv_heads * a.c.nseq;
    PromptCut best{2u, 1u, ~0ull};
    for (uint32_t t = 1; t <= 2; ++t) {
        const uint64_t units = (rows + t * kTileRows - 1) / (t * kTileRows) * heads;
        for (uint32_t c = 1; c <= kMaxSplit && units * c <= (uint64_t)sms && (c == 1 || 2 * c <= keys); ++c) {
            if (units > at_once(t, c)) continue;   // a second wave costs more than the split saves
            const uint64_t cycles = (uint64_t)(t == 1 ? 5400 : 6900) * ((keys + c - 1) / c) + (t == 1 ? 14500 : c == 1 ? 18000 : 28000);
            if (cycles < best.cycles) best = PromptCut{t, c, cycles};
        }
    }
    if (best.cycles == ~0ull) {
        const uint64_t units = (rows + 2u * kTileRows - 1) / (2u * kTileRows) * heads;
        best.cycles = (units + (uint64_t)sms - 1) / (uint64_t)sms * (6900ull * keys + 18000ull);
    }
    return best;
}

// Attention of many query rows; see AttnArgs
cudaError_t launch_prompt(AttnArgs a, const PromptCut &cut, int dev, int sms, cudaStream_t stream)
{
    const uint32_t rows = a.r.tokens * a.group, C = cut.split;
    a.tiles = (rows + cut.tiles * kTileRows - 1) / (cut.tiles * kTileRows);
    const dim3 grid(C * a.tiles, a.c.kv_heads, a.c.nseq);
    const cudaError_t e = cut.tiles == 1 ? prepare<prompt_kernel<true>>(dev) : prepare<prompt_kernel<false>>(dev);
    if (e != cudaSuccess) return e;
    return cut.tiles == 1 ? launch(prompt_kernel<true>, grid, kPromptThreads, kPromptSmem, C, a, sms, stream)
                          : launch(prompt_kernel<false>, grid, kPromptThreads, kPromptSmem, C, a, sms, stream);
}

}  // namespace k8
}  // namespace atlas
