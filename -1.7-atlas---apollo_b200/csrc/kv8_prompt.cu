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
// accuracy. The block scales of K multiply the scores, those of V the weights
// (over a running power of two vref, so that one accumulator serves blocks of
// different scales; p <= 2^8 and v_scale < 2 vref keep P below 2^15).
//
// Warps of a CTA (13, so that a thread may have 128 registers):
//   0-7    softmax, one warpgroup per tile, one thread per row: maximum and
//          exponentials of the scores straight from tensor memory, P back into
//          the columns that the scores leave; the maximum is lazy (raised only
//          when a score passes it by 2^8), so the output is rescaled rarely;
//   8-11   codes -> binary16 in 128-byte swizzled K-major tiles: K [key][dimension],
//          V transposed on the way, [dimension][key]; the next tiles' codes are in
//          registers while the MMAs still read the current ones;
//   12     issues the MMAs: P V of a tile, then the next keys' scores of the
//          same tile, so that one tile's softmax runs under the other's MMAs.
// Tensor memory: 2 x 128 columns of scores / weights, 2 x 128 of output.
// Shared memory: Q hi / lo 128 KB, K 32 KB, V 32 KB; Q's place stages the output.
//
// Few rows over many positions: the positions are split over a cluster of CTAs,
// and each merges a share of the rows through distributed shared memory.
//
// Bound by the tensor pipe (4096 cycles per 256 rows x 128 keys) next to the
// softmax's issue slots. Every wait is bounded; after a timeout the CTA's rows
// are NaN.
#include <cfloat>
#include <cmath>
#include "../../include/atlas_cuda.h"
#include "kv8.cuh"

namespace atlas {
namespace k8 {
namespace {

constexpr uint32_t kTileRows = 128, kTileKeys = 128;
constexpr uint32_t kPromptThreads = 13 * 32, kMmaWarp = 12;
constexpr uint32_t kHalf = 128 * 128;              // bytes of 128 rows x 64 binary16, swizzled
constexpr uint32_t kQTile = 4 * kHalf;             // one tile's Q: [hi, lo][2 x 64 dimensions]

struct PromptBars {
    uint64_t s_full[2], p_full[2], o_full[2], k_full, k_empty, v_full, v_empty, fin;
    uint32_t tmem, status;
    float row_factor[2][kTileRows];                // what a score of the row is worth, in the exponent's base 2
    float row_max[2][kTileRows], row_sum[2][kTileRows];
};

constexpr size_t kPromptSmem = 2 * kQTile + 4 * kHalf + sizeof(PromptBars) + 1024;
static_assert(kPromptSmem <= kMaxSmem, "the tiles exceed a CTA's shared memory");

__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

__device__ __forceinline__ bool wait_warp(uint64_t *bar, uint32_t parity, volatile uint32_t *err)
{
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, err));
}

// Shared-memory operand: K-major, 128-byte swizzle, 8-row groups 1024 bytes apart
__device__ __forceinline__ uint64_t operand(uint32_t saddr)
{
    return (uint64_t)((saddr >> 4) & 0x3FFFu) | ((uint64_t)1u << 16) | ((uint64_t)(1024u >> 4) << 32) |
           ((uint64_t)1u << 46) | ((uint64_t)2u << 61);
}

// fp32 accumulator, binary16 operands, K-major, M = 128, N = 128
constexpr uint32_t kInstr = (1u << 4) | ((128u >> 3) << 17) | ((128u >> 4) << 24);

__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t accumulate)
{
    asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n"
                 ::"r"(d), "l"(a), "l"(b), "r"(kInstr), "r"(accumulate)
                 : "memory");
}

// A from tensor memory
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t accumulate)
{
    asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n"
                 ::"r"(d), "r"(a), "l"(b), "r"(kInstr), "r"(accumulate)
                 : "memory");
}

// Arrives on `bar` once every MMA that this thread issued is done
__device__ __forceinline__ void commit(uint64_t *bar)
{
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_addr(bar)) : "memory");
}

__device__ __forceinline__ void tmem_ld(uint32_t addr, float (&r)[32])
{
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n"
        "tcgen05.wait::ld.sync.aligned;"
        : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]), "=f"(r[8]),
          "=f"(r[9]), "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15]), "=f"(r[16]),
          "=f"(r[17]), "=f"(r[18]), "=f"(r[19]), "=f"(r[20]), "=f"(r[21]), "=f"(r[22]), "=f"(r[23]), "=f"(r[24]),
          "=f"(r[25]), "=f"(r[26]), "=f"(r[27]), "=f"(r[28]), "=f"(r[29]), "=f"(r[30]), "=f"(r[31])
        : "r"(addr)
        : "memory");
}

__device__ __forceinline__ void tmem_st(uint32_t addr, const uint32_t (&r)[32])
{
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
        ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
          "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]),
          "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]),
          "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}

__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Byte offset of 16-byte chunk `chunk` of a row of a swizzled tile of 128-byte rows
__device__ __forceinline__ uint32_t swizzled(uint32_t row, uint32_t chunk)
{
    return row * 128u + ((chunk ^ (row & 7u)) << 4);
}

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

// A row's softmax over one tile of keys: scores at tensor memory `at` (this
// warp's lanes), scale of 16-key group i in lane i (K) and 8 + i (V) of `sc`,
// of which the row sees the first `nvis` keys (MASK; else all).
template <bool MASK>
__device__ __forceinline__ float tile_max(uint32_t at, float sc, float factor, int nvis)
{
    float m = -INFINITY;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        float s[32];
        tmem_ld(at + 32u * (uint32_t)c, s);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float x = -INFINITY;
#pragma unroll
            for (int i = 0; i < 16; ++i)
                x = fmaxf(x, MASK && 32 * c + 16 * h + i >= nvis ? -INFINITY : s[16 * h + i]);
            const float f = __shfl_sync(0xffffffffu, sc, 2 * c + h) * factor;
            if (!MASK || x != -INFINITY) m = fmaxf(m, x * f);
        }
    }
    return m;
}

// The weights into the scores' columns, 32 keys at a time: 16 columns of hi, 16 of lo. Returns their sum.
template <bool MASK>
__device__ __forceinline__ float tile_weights(uint32_t at, float sc, float factor, int nvis, float m, float vinv)
{
    float sum = 0.f;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        float s[32];
        tmem_ld(at + 32u * (uint32_t)c, s);
        uint32_t p[32];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const float f = __shfl_sync(0xffffffffu, sc, 2 * c + h) * factor;
            const float pf = __shfl_sync(0xffffffffu, sc, 8 + 2 * c + h) * vinv;
            float part = 0.f;
#pragma unroll
            for (int i = 0; i < 16; i += 2) {
                float hi[2], lo[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const bool seen = !MASK || 32 * c + 16 * h + i + e < nvis;
                    float w = ex2(fmaf(s[16 * h + i + e], f, -m));
                    if (MASK && !seen) w = 0.f;
                    part += w;
                    w *= pf;
                    if (MASK && !seen) w = 0.f;   // whatever the block's scale is
                    hi[e] = __uint_as_float(__float_as_uint(w) & 0xffffe000u);   // exact in binary16
                    lo[e] = w - hi[e];
                }
                p[8 * h + i / 2] = h2_bits(hi[0], hi[1]);
                p[16 + 8 * h + i / 2] = h2_bits(lo[0], lo[1]);
            }
            sum += part;
        }
        tmem_st(at + 32u * (uint32_t)c, p);
    }
    return sum;
}

__global__ void __launch_bounds__(kPromptThreads, 1) prompt_kernel(const __grid_constant__ AttnArgs a)
{
    extern __shared__ uint8_t smem_raw[];
    uint8_t *const smem = smem_raw + ((1024u - (smem_addr(smem_raw) & 1023u)) & 1023u);
    uint8_t *const qs = smem, *const ks = smem + 2 * kQTile, *const vs = ks + 2 * kHalf;
    PromptBars &b = *reinterpret_cast<PromptBars *>(vs + 2 * kHalf);
    volatile uint32_t *const err = &b.status;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
    const uint32_t C = cluster_size(), rank = cluster_rank(), s = blockIdx.z, h = blockIdx.y;
    // the last rows first: they see the most positions
    const uint32_t r0 = (a.tiles - 1u - blockIdx.x / C) * 2u * kTileRows;
    TileRows tr{r0 / a.group, 0u, a.group, a.group_inv};
    tr.rem = r0 - tr.tok * a.group;
    if (threadIdx.x == 0) {
        for (int t = 0; t < 2; ++t) {
            mbar_init(&b.s_full[t], 1u);
            mbar_init(&b.p_full[t], 4u);
            mbar_init(&b.o_full[t], 1u);
        }
        mbar_init(&b.k_full, 4u);
        mbar_init(&b.v_full, 4u);
        mbar_init(&b.k_empty, 1u);
        mbar_init(&b.v_empty, 1u);
        mbar_init(&b.fin, 1u);
        b.status = kStatusOk;
        fence_mbar_init();
    }
    wait_predecessor(a.early);
    const uint64_t p0 = __ldcg(a.r.pos0 + s);
    const uint32_t all = row_count(a.r, s) * a.group;
    if (r0 >= all) return;   // the whole cluster leaves
    const uint32_t rows = min(all - r0, 2u * kTileRows), tiles = rows > kTileRows ? 2u : 1u;
    const uint32_t limit = (uint32_t)min(p0 + tr.at(rows - 1u).x + 1u, (uint64_t)a.c.max_context);
    const uint32_t total = (limit + kTileKeys - 1u) / kTileKeys;
    const uint32_t j0 = (uint32_t)((uint64_t)total * rank / C), n = (uint32_t)((uint64_t)total * (rank + 1u) / C) - j0;
    const size_t head = (size_t)s * a.c.kv_heads + h;

    if (warp == kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&b.tmem)), "r"(512u)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    } else {
        // Q: four rows at a time per warp, lane = 4 dimensions; a power of two
        // brings each row's largest value to [2^8, 2^9)
#pragma unroll 1
        for (uint32_t i0 = 4u * warp; i0 < tiles * kTileRows; i0 += 4u * kMmaWarp) {
            float4 x[4];
#pragma unroll
            for (uint32_t u = 0; u < 4; ++u) {
                const uint2 r = tr.at(i0 + u);
                x[u] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (i0 + u < rows)
                    x[u] = __ldcg(reinterpret_cast<const float4 *>(a.q + ((size_t)s * a.r.tokens + r.x) * a.ldq +
                                                                  (size_t)(h * a.group + r.y) * kDim) + lane);
            }
#pragma unroll
            for (uint32_t u = 0; u < 4; ++u) {
                const uint32_t i = i0 + u, row = i & (kTileRows - 1u);
                float v[4] = {x[u].x, x[u].y, x[u].z, x[u].w};
                uint32_t mx = 0u;
#pragma unroll
                for (int e = 0; e < 4; ++e) mx = max(mx, __float_as_uint(v[e]) & 0x7fffffffu);
                mx = __reduce_max_sync(0xffffffffu, mx);
                const bool bad = mx >= 0x7f800000u;   // a non-finite value: every score of the row NaN
                // v * 2^(8 - e) as two factors, so that neither leaves the range
                const int e = bad ? 0 : max((int)(mx >> 23) - 127, -126), half = (8 - e) / 2;
                const float f0 = __int_as_float((127 + half) << 23), f1 = __int_as_float((127 + 8 - e - half) << 23);
                const float g0 = __int_as_float((127 - half) << 23), g1 = __int_as_float((127 - 8 + e + half) << 23);
                float hi[4], lo[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    v[k] = bad ? 0.f : v[k] * f0 * f1;
                    hi[k] = __uint_as_float(__float_as_uint(v[k]) & 0xffffe000u);
                    lo[k] = v[k] - hi[k];
                }
                if (lane == 0)
                    b.row_factor[i / kTileRows][row] = bad ? __int_as_float(0x7fffffff) : kScoreScale * g0 * g1;
                uint8_t *q = qs + (i / kTileRows) * kQTile + (lane >> 4) * kHalf + swizzled(row, (lane & 15u) >> 1) + (lane & 1u) * 8u;
                *reinterpret_cast<uint2 *>(q) = make_uint2(h2_bits(hi[0], hi[1]), h2_bits(hi[2], hi[3]));
                *reinterpret_cast<uint2 *>(q + 2 * kHalf) = make_uint2(h2_bits(lo[0], lo[1]), h2_bits(lo[2], lo[3]));
            }
        }
        fence_async();
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = b.tmem;   // scores / weights of tile t: column 128 t; output: 256 + 128 t

    if (warp == kMmaWarp) {
        // ------------------------------------------------------------- MMA --
        if (lane == 0) {
            const uint32_t qa = smem_addr(qs), ka = smem_addr(ks), va = smem_addr(vs);
            auto scores = [&](uint32_t t) {
                for (uint32_t st = 0; st < 8u; ++st) {
                    const uint32_t off = (st >> 2) * kHalf + (st & 3u) * 32u;
                    const uint64_t k = operand(ka + off);
                    mma_ss(tmem + 128u * t, operand(qa + t * kQTile + off), k, st != 0u);
                    mma_ss(tmem + 128u * t, operand(qa + t * kQTile + 2u * kHalf + off), k, 1u);
                }
                commit(&b.s_full[t]);
            };
            bool ok = n != 0u;
            if (ok && (ok = mbar_wait(&b.k_full, 0u, err))) {
                fence_after();
                for (uint32_t t = 0; t < tiles; ++t) scores(t);
                commit(&b.k_empty);
            }
            for (uint32_t j = 0; ok && j < n; ++j) {
                if (!(ok = mbar_wait(&b.v_full, j & 1u, err))) break;
                for (uint32_t t = 0; t < tiles; ++t) {
                    if (!(ok = mbar_wait(&b.p_full[t], j & 1u, err))) break;
                    fence_after();
                    for (uint32_t st = 0; st < 8u; ++st) {
                        const uint64_t v = operand(va + (st >> 2) * kHalf + (st & 3u) * 32u);
                        const uint32_t p = tmem + 128u * t + (st >> 1) * 32u + (st & 1u) * 8u;
                        mma_ts(tmem + 256u + 128u * t, p, v, j != 0u || st != 0u);
                        mma_ts(tmem + 256u + 128u * t, p + 16u, v, 1u);
                    }
                    if (t + 1u == tiles) commit(&b.v_empty);
                    if (j + 1u == n) {
                        commit(&b.o_full[t]);
                        continue;
                    }
                    if (t == 0u) {
                        if (!(ok = mbar_wait(&b.k_full, (j + 1u) & 1u, err))) break;
                        fence_after();
                    }
                    scores(t);
                    if (t + 1u == tiles) commit(&b.k_empty);
                }
            }
            // nothing of this CTA is left in flight when tensor memory is freed
            commit(&b.fin);
            const uint64_t t0 = global_ns();
            while (!mbar_try_wait(&b.fin, 0u) && global_ns() - t0 < kWaitLimitNs) {
            }
        }
        __syncwarp();
    } else if (warp >= 8) {
        // ------------------------------------------------------- converters --
        // K: a thread takes 16 dimensions of 8 keys (8 lanes write the same
        // chunk of 8 rows); V: 8 keys x 16 dimensions (8 lanes write the 8
        // chunks of a row): neither has a bank conflict.
        const uint32_t w = warp - 8u, l8 = lane & 7u, q8 = lane >> 3;
        const int8_t *ksrc = a.c.k + (head * a.c.max_context + 8u * w + l8) * kDim + 16u * q8;
        const uint32_t kg = l8 + 8u * (w >> 1), dg = q8 + 4u * (w & 1u);
        const int8_t *vsrc = a.c.v + (head * a.c.max_context + 8u * kg) * kDim + 16u * dg;
        uint4 x[8], y[8];
        auto load_k = [&](uint32_t j) {
            const uint32_t key0 = (j0 + j) * kTileKeys;
#pragma unroll
            for (uint32_t i = 0; i < 8; ++i) {
                const uint32_t row = 32u * (i >> 1);
                x[i] = make_uint4(0u, 0u, 0u, 0u);
                if (key0 + row + 8u * w + l8 < limit)
                    x[i] = __ldcg(reinterpret_cast<const uint4 *>(ksrc + (size_t)(key0 + row) * kDim + 64u * (i & 1u)));
            }
        };
        auto load_v = [&](uint32_t j) {
            const uint32_t key0 = (j0 + j) * kTileKeys;
#pragma unroll
            for (uint32_t i = 0; i < 8; ++i) {
                y[i] = make_uint4(0u, 0u, 0u, 0u);
                if (key0 + 8u * kg + i < limit) y[i] = __ldcg(reinterpret_cast<const uint4 *>(vsrc + (size_t)(key0 + i) * kDim));
            }
        };
        if (n) {
            load_k(0u);
            load_v(0u);
        }
        for (uint32_t j = 0; j < n; ++j) {
            if (j && !wait_warp(&b.k_empty, (j - 1u) & 1u, err)) break;
#pragma unroll
            for (uint32_t i = 0; i < 8; ++i) {
                const uint32_t row = 32u * (i >> 1) + 8u * w + l8;
                uint8_t *dst = ks + (i & 1u) * kHalf;
                const uint32_t words[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
                uint32_t o[8];
#pragma unroll
                for (int q = 0; q < 4; ++q) {   // two neighbouring dimensions, each in the low byte of a half
                    o[2 * q] = codes_h2<false>(__byte_perm(words[q], 0u, 0x4140u));
                    o[2 * q + 1] = codes_h2<false>(__byte_perm(words[q], 0u, 0x4342u));
                }
                *reinterpret_cast<uint4 *>(dst + swizzled(row, 2u * q8)) = make_uint4(o[0], o[1], o[2], o[3]);
                *reinterpret_cast<uint4 *>(dst + swizzled(row, 2u * q8 + 1u)) = make_uint4(o[4], o[5], o[6], o[7]);
            }
            fence_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(&b.k_full);
            if (j + 1u < n) load_k(j + 1u);
            if (j && !wait_warp(&b.v_empty, (j - 1u) & 1u, err)) break;
            uint8_t *dst = vs + (kg >> 3) * kHalf;
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
                    *reinterpret_cast<uint4 *>(dst + swizzled(16u * dg + 4u * (uint32_t)q + (uint32_t)d, kg & 7u)) =
                        make_uint4(o[d][0], o[d][1], o[d][2], o[d][3]);
            }
            fence_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(&b.v_full);
            if (j + 1u < n) load_v(j + 1u);
        }
    } else {
        // --------------------------------------------------------- softmax --
        const uint32_t t = warp >> 2, quarter = warp & 3u, row = quarter * 32u + lane, i = t * kTileRows + row;
        if (t < tiles) {
            const uint32_t at = tmem + ((quarter * 32u) << 16) + 128u * t;
            const float factor = b.row_factor[t][row];
            const uint32_t open = (uint32_t)min(p0 + tr.at(t * kTileRows).x, (uint64_t)0x7fffffffu);
            const uint32_t last = i < rows ? (uint32_t)min(p0 + tr.at(i).x, (uint64_t)0x7fffffffu) : open;
            const float *scales = (lane & 8u ? a.c.v_scale : a.c.k_scale) + head * a.c.n_blocks;
            auto scale_of = [&](uint32_t j) {
                return __ldcg(scales + min(((j0 + j) * kTileKeys + 16u * (lane & 7u)) >> a.c.block_log2, a.c.n_blocks - 1u));
            };
            float m = -INFINITY, l = 0.f, next = n ? scale_of(0u) : 0.f;
            uint32_t vref = kTinyScale;
            for (uint32_t j = 0; j < n; ++j) {
                const float sc = next;
                if (j + 1u < n) next = scale_of(j + 1u);
                const uint32_t key0 = (j0 + j) * kTileKeys;
                const bool masked = key0 + kTileKeys - 1u > open;   // some row does not see all of the tile
                const int nvis = last < key0 ? 0 : (int)min(last - key0 + 1u, kTileKeys);
                // the largest V scale of the tile's stored positions (a NaN counts nothing)
                float top = lane >= 8u && lane < 16u && key0 + 16u * (lane & 7u) < limit ? sc : 0.f;
                top = __uint_as_float(__reduce_max_sync(0xffffffffu, top > 0.f && top < INFINITY ? __float_as_uint(top) : 0u));
                if (!wait_warp(&b.s_full[t], j & 1u, err)) break;
                fence_after();
                const float x = masked ? tile_max<true>(at, sc, factor, nvis) : tile_max<false>(at, sc, factor, 128);
                float f = 1.0f;
                if (x > m + kLazy) {
                    f = m == -INFINITY ? 0.f : ex2(m - x);
                    m = x;
                    l *= f;
                }
                if (top >= 2.0f * __uint_as_float(vref)) {
                    const uint32_t now = __float_as_uint(top) & 0x7f800000u;
                    f *= now - vref > 120u << 23 ? 0.f : __uint_as_float((127u << 23) - (now - vref));
                    vref = now;
                }
                if (j && __any_sync(0xffffffffu, f != 1.0f)) {
#pragma unroll 1
                    for (uint32_t c = 0; c < 128u; c += 32u) {
                        float o[32];
                        uint32_t u[32];
                        tmem_ld(at + 256u + c, o);
#pragma unroll
                        for (int k = 0; k < 32; ++k) u[k] = __float_as_uint(o[k] * f);
                        tmem_st(at + 256u + c, u);
                    }
                }
                const float vinv = __uint_as_float((260u << 23) - vref);   // 2^6 / vref
                l += masked ? tile_weights<true>(at, sc, factor, nvis, m, vinv) : tile_weights<false>(at, sc, factor, 128, m, vinv);
                tmem_wait_st();
                fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&b.p_full[t]);
            }
            // the output into Q's place: row-major, 16-byte chunks XORed with the row
            const bool have = n && wait_warp(&b.o_full[t], 0u, err);
            fence_after();
            const float back = C > 1u ? __uint_as_float(vref) * (1.0f / 64.0f) : __uint_as_float(vref) * (1.0f / 64.0f) / l;
            float4 *stage = reinterpret_cast<float4 *>(qs + t * kQTile);
#pragma unroll 1
            for (uint32_t c = 0; c < 4u; ++c) {
                float o[32];
                if (have) tmem_ld(at + 256u + 32u * c, o);
#pragma unroll
                for (uint32_t k = 0; k < 8; ++k)
                    stage[row * 32u + ((8u * c + k) ^ (row & 31u))] =
                        have ? make_float4(o[4 * k] * back, o[4 * k + 1] * back, o[4 * k + 2] * back, o[4 * k + 3] * back)
                             : make_float4(0.f, 0.f, 0.f, 0.f);
            }
            b.row_max[t][row] = m;
            b.row_sum[t][row] = l;
            __syncwarp();
            if (C == 1u) {
                for (uint32_t k = 0; k < 32u && t * kTileRows + quarter * 32u + k < rows; ++k) {
                    const uint32_t rr = quarter * 32u + k;
                    const uint2 r = tr.at(t * kTileRows + rr);
                    float4 x = stage[rr * 32u + (lane ^ (rr & 31u))];
                    if (*err != kStatusOk || p0 + r.x >= a.c.max_context)
                        x.x = x.y = x.z = x.w = __int_as_float(0x7fffffff);
                    reinterpret_cast<float4 *>(a.out + ((size_t)s * a.r.tokens + r.x) * a.ldo +
                                               (size_t)(h * a.group + r.y) * kDim)[lane] = x;
                }
            }
        }
    }
    fence_before();
    __syncthreads();
    if (warp == kMmaWarp) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
    if (C == 1u) return;
    // Rows rank, rank + C, ... of the cluster's states: a warp per row, lane = 4
    // dimensions. A state that saw no position counts nothing.
    cluster_sync();
    if (warp < kMmaWarp) {
        for (uint32_t i = rank + C * warp; i < rows; i += C * kMmaWarp) {
            const uint32_t t = i / kTileRows, row = i & (kTileRows - 1u);
            const float mc = lane < C ? ld_cluster1(&b.row_max[t][row], lane) : -INFINITY;
            const float lc = lane < C ? ld_cluster1(&b.row_sum[t][row], lane) : 0.f;
            const bool bad = lane < C && __float_as_uint(ld_cluster1(&b.status, lane)) != kStatusOk;
            float M = mc;
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o, 16));
            const float f = mc == -INFINITY && lc == 0.f ? 0.f : ex2(mc - M);
            float L = f * lc;
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) L += __shfl_xor_sync(0xffffffffu, L, o, 16);
            L = __shfl_sync(0xffffffffu, L, 0);
            const bool any_bad = __any_sync(0xffffffffu, bad);
            const float4 *stage = reinterpret_cast<const float4 *>(qs + t * kQTile);
            float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
            for (uint32_t c = 0; c < C; ++c) {
                const float4 y = ld_cluster4(&stage[row * 32u + (lane ^ (row & 31u))], c);
                const float fc = __shfl_sync(0xffffffffu, f, (int)c);
                x.x = fmaf(fc, y.x, x.x);
                x.y = fmaf(fc, y.y, x.y);
                x.z = fmaf(fc, y.z, x.z);
                x.w = fmaf(fc, y.w, x.w);
            }
            const uint2 r = tr.at(i);
            const float inv = any_bad || p0 + r.x >= a.c.max_context ? __int_as_float(0x7fffffff) : 1.0f / L;
            reinterpret_cast<float4 *>(a.out + ((size_t)s * a.r.tokens + r.x) * a.ldo + (size_t)(h * a.group + r.y) * kDim)[lane] =
                make_float4(x.x * inv, x.y * inv, x.z * inv, x.w * inv);
        }
    }
    cluster_sync();   // no CTA leaves while the cluster may read its states
}

}  // namespace

// Attention of many query rows; see AttnArgs. a.tiles is set here.
cudaError_t launch_prompt(AttnArgs a, int dev, int sms, cudaStream_t stream)
{
    cudaError_t e = allow<prompt_kernel>(dev, (int)kPromptSmem);
    if (e != cudaSuccess) return e;
    a.tiles = (a.r.tokens * a.group + 2 * kTileRows - 1) / (2 * kTileRows);
    // CTAs per unit: while they all fit at once, at most 8, and 2 tiles of keys each
    const uint64_t units = (uint64_t)a.tiles * a.c.kv_heads * a.c.nseq;
    uint32_t C = 1;
    while (C < 8 && units * C * 2 <= (uint64_t)sms && (uint64_t)C * 2 * 2 * kTileKeys <= a.c.max_context) C *= 2;
    return launch(prompt_kernel, dim3(C * a.tiles, a.c.kv_heads, a.c.nseq), kPromptThreads, kPromptSmem, C, a, sms, stream);
}

}  // namespace k8
}  // namespace atlas
