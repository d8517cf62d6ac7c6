// Attention over a paged KV cache for few query rows per KV head (sm_100a), and
// the kernel that joins partial sums. The form for many rows is in
// paged_prompt.cu. (gqa_single_token in the reference, src/brain_runtime.c:1407-1528,
// over one region of fp32 rows.)
//
// A unit is 8 NT query rows (token, head of the group; token-major) of a KV
// head. A CTA takes a piece of the line of all units' keys (paged.cuh), 16
// positions at a time dealt out over its warps, each with a softmax state
// of its own (running maximum, sum, output), joined in shared memory at a unit's
// end. 16 positions lie in one page: two TMA copies (16 rows of K, 16 of V,
// swizzled) bring them into a ring of the warp's own, and positions without a
// page are passed over.
//
//   S^T = K Q^T     m16n8k16 (rows are positions, columns query rows)
//   O^T += V^T P^T  m16n8k16 (rows are dimensions); P in two 16-bit terms
//                   hi + lo, so that it costs the output nothing; the MMAs truncate
//                   their sums, so each 16 positions' is added to the output in fp32
//
// The maximum is lazy: a row's is raised only when a score passes it by 2^6, so
// 16 positions need no reduction over lanes.
// Where there are enough clusters to give each unit one, its CTAs have the unit
// together, and join their states through distributed shared memory.
// Bound by HBM for long caches (8 sequences of 32768 positions, 40 heads on 8, 1.07
// GB: 165 to 167 us in a row of calls, 98 % of the copy rate; 171 to 173 for calls one by
// one; 256 sequences of 100 to 8000 positions, 28 heads on 4, 362 us, 96 %; 64 of them
// 94, 85 %), by latency for short ones: launch, piece, pages' numbers, first copies, a
// round of chunks a microsecond, sums (640 positions 6.9 us, 8447 11.5, 8 sequences
// around 2303 13.7 in tables that have no room for more; where there is room for 32768,
// 8.3, 12.6 and 14.2: the launch that joins partial sums follows), and by the search for a
// CTA's piece for very many sequences (4096 of 100 to 300 positions 725 us, 37 %).
#include <algorithm>
#include <cfloat>
#include <cmath>
#include "../../include/atlas_cuda.h"
#include "paged.cuh"

namespace atlas {
namespace paged {

using k8::kScoreScale;
using k8::pair;
using k8::unpair;
using k8::add2;
using k8::mul2;
using k8::wait_predecessor;

namespace {

constexpr uint32_t kChunk = 16, kWarps = 12, kThreads = kWarps * 32, kStages = 2;
constexpr uint32_t kHalfChunk = kChunk * 128, kSlot = 4 * kHalfChunk;   // 16 rows x 64 dimensions; K and V of 16 positions
constexpr uint32_t kRecStride = kDim + 4;
// Chunks: what joining partial sums takes, where a sequence has no room for more than leaves none, so that the launch
// that joins them is left out (640 positions 6.9 us instead of 8.3; 8447 11.5 instead of 12.6), and where it follows in any case;
// and what beginning and ending a unit takes. In tables with room for 32768 positions, with 95, 48 or 32 instead of 64: 16 heads
// on 2 over 32767 18.8, 15.4 or 15.4 us instead of 15.4; 28 on 4 over 20000 15.1, 15.1 or 14.1 instead of 15.1; 40 on 8 over 30000
// 27.5, 28.3 or 28.3 instead of 27.6. With 8 instead of 32 for a unit's ends nothing changes by 1 %.
constexpr uint32_t kWorth = 96, kWorthMore = 64, kExtra = 32;
static_assert(kWorthMore < kWorth, "it tells a call that may leave partial sums");
constexpr float kLazy = 6.0f;
// Weights are 2^(score - maximum + kUnit). binary16: their largest, 2^15, keeps the low term's bits; bfloat16 has fp32's
// range, and small weights leave the sums of large values room
template <bool BF>
constexpr float kUnit = BF ? -24.0f : 9.0f;

struct FewArgs : AttnArgs {
    CUtensorMap kmap, vmap;      // [2][rows of the pool][64] each
    uint32_t worth;              // so many chunks longer may a CTA's work get before units are cut
};

template <int NT>
struct alignas(1024) Smem {
    union {
        uint8_t ring[kWarps][kStages][kSlot];
        float wrec[kWarps][8 * NT][kRecStride];    // the warps' outputs, once the ring is done with
        PieceSmem piece;
    } u;
    uint64_t full[kWarps][kStages];
    uint32_t err;
    alignas(16) uint16_t q[8 * NT][kDim + 8];      // rows 68 words apart: the warps' reads have no bank conflict
    float2 wml[kWarps][8 * NT];
    // what the cluster's CTAs send: of each, this CTA's share of the rows' dimensions, and all rows' maxima and sums
    float4 sent[8 * NT * (kDim / 4) + k8::kMaxCluster];
    float2 sent_ml[k8::kMaxCluster][8 * NT];
};

template <bool BF>
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    if (BF)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// The same onto zeros
template <bool BF>
__device__ __forceinline__ void mma_first(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    if (BF)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
            : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
            : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}

__device__ __forceinline__ uint32_t transpose8(uint32_t x)
{
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

__device__ __forceinline__ void load_matrices(uint32_t (&d)[4], uint32_t addr)
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void load_matrices_t(uint32_t (&d)[4], uint32_t addr)
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
                 : "r"(addr)
                 : "memory");
}

// 16 rows of the pool from row `row` on, as two halves of 64 dimensions, each [16][128 bytes], 16-byte chunk c of row r
// at chunk c ^ (r % 8)
__device__ __forceinline__ void load_rows(uint32_t dst, const CUtensorMap *map, uint32_t row, uint64_t *bar)
{
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                 ::"r"(dst), "l"(map), "r"(0), "r"((int)row), "r"(0), "r"(smem_addr(bar))
                 : "memory");
}

// To another CTA of the cluster
__device__ __forceinline__ void send(const float4 *p, uint32_t cta, float4 v)
{
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_addr(p)), "r"(cta));
    asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(r), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w) : "memory");
}
__device__ __forceinline__ void send(const float2 *p, uint32_t cta, float2 v)
{
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_addr(p)), "r"(cta));
    asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(r), "f"(v.x), "f"(v.y) : "memory");
}
// Split: arrive once the CTA runs, wait before the first access to another CTA's shared memory
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.aligned;" ::: "memory"); }

// What this thread did to the ring's place comes before the copies that follow
__device__ __forceinline__ void fence_ring() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

constexpr uint32_t kNone = ~0u;

template <bool BF, int NT>
__global__ void __launch_bounds__(kThreads, 1) few_kernel(const __grid_constant__ FewArgs a)
{
    constexpr uint32_t R = 8 * NT;
    extern __shared__ __align__(1024) uint8_t few_smem[];
    Smem<NT> &sm = *reinterpret_cast<Smem<NT> *>(few_smem);
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u, g = lane >> 2, t = lane & 3u, cluster = k8::cluster_size();
    if (cluster > 1u) cluster_arrive();
    if (lane == 0u) {
        for (uint32_t i = 0; i < kStages; ++i) mbar_init(&sm.full[warp][i], 1u);
        fence_mbar_init();
    }
    if (threadIdx.x == 0u) {
        sm.err = kStatusOk;
        asm volatile("prefetch.tensormap [%0];" ::"l"(&a.kmap) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&a.vmap) : "memory");
    }
    __syncthreads();
    wait_predecessor(a.early);
    const Cut<kChunk, kExtra> cut{a, R, Divisor{1u << 31, NT == 1 ? 3u : 4u}};
    const Piece piece = a.keep ? find_kept(cut, kWarps, a.worth, cluster) : find_together<kWarps>(cut, sm.u.piece, kWarps, a.worth);
    if (cluster > 1u && (piece.shared == 1u || !piece.left)) cluster_wait();
    const uint32_t deal = kWarps * piece.shared;   // warps that share a unit's chunks
    Walk<kChunk, kExtra> w(cut, piece);
    if (!a.keep) {                        // the ring's place is free
        fence_ring();
        __syncthreads();
    }
    auto tell_part = [&]() {
        const Part part = w.part();
        if (lane == 0u) reinterpret_cast<Part *>(a.parts)[blockIdx.x] = part;
    };
    if (!w.more() && warp == kWarps - 1u) tell_part();
    const uint32_t ring = smem_addr(sm.u.ring[warp][0]);
    uint64_t *const full = sm.full[warp];
    // where ldmatrix reads: K of 16 dimensions (16 positions x 2 chunks), V of 16 dimensions (the same, to be transposed)
    uint32_t koff[4], voff[4];
#pragma unroll
    for (uint32_t i = 0; i < 4u; ++i) {
        koff[i] = (lane & 15u) * 128u + (((2u * i + (lane >> 4)) ^ (lane & 7u)) << 4);
        voff[i] = 2u * kHalfChunk + ((lane & 7u) + 8u * (lane >> 4)) * 128u + (((2u * i + ((lane >> 3) & 1u)) ^ (lane & 7u)) << 4);
    }
    const float inv_group = 1.000001f / (float)a.group;
    uint32_t slot = 0u, phase = 0u, slot_in = 0u;
    bool ok = true;

    for (; w.more(); w.next()) {
        const uint32_t rows = w.rows(), row0 = w.row0(), s = w.p.s, h = w.p.h;
        TileRows tr{divide(row0, a.by_group), 0u, a.group, inv_group};
        tr.rem = row0 - tr.tok * a.group;
        const uint64_t p0 = w.q.p0;
        const uint32_t seen = cut.keys(w.q, row0 + rows);          // chunks that some row sees
        const uint32_t k_end = min(w.k_end, seen), first = w.k_begin + (piece.shared > 1u ? k8::cluster_rank() * kWarps : 0u) + warp;
        const int32_t *const entries = a.c.table + (size_t)s * a.c.max_pages;
        const uint32_t page_chunks = a.c.page_log2 - 4u;           // log2 of chunks per page
        const uint32_t head0 = a.layer * a.c.pages * a.c.kv_heads + h;
        // the pages of this warp's chunks first + deal (base + lane), and of the next 32; their loads are on their way first
        auto entry_of = [&](uint32_t base) {
            const uint32_t c = first + deal * (base + lane);
            return c < k_end ? (uint32_t)__ldcg(entries + (c >> page_chunks)) : ~0u;
        };
        uint32_t base = 0u, ent = entry_of(0u), ent_next = entry_of(32u);
        // The queries come once for all warps (with a read of each warp's own, the many CTAs that have a KV head's units
        // crowd on its lines of L2: 8447 positions 12.9 us instead of 11.3)
        uint4 qv[(R * 16u + kThreads - 1u) / kThreads];
#pragma unroll
        for (uint32_t k = 0; k < sizeof(qv) / 16u; ++k) {
            const uint32_t x = k * kThreads + threadIdx.x;
            if (x < R * 16u) {
                const uint2 at = tr.at(min(x / 16u, rows - 1u));
                qv[k] = __ldcg(reinterpret_cast<const uint4 *>(a.q + ((size_t)s * a.r.tokens + at.x) * a.ldq + (size_t)(h * a.group + at.y) * kDim) + x % 16u);
            }
        }
        uint32_t have = __ballot_sync(0xffffffffu, ent < a.c.pages);
        // the next chunk of this warp's that has a page; its copies are issued into the next slot
        auto issue = [&]() -> uint32_t {
            while (!have) {
                base += 32u;
                if (first + deal * base >= k_end) return kNone;
                ent = ent_next;
                ent_next = entry_of(base + 32u);
                have = __ballot_sync(0xffffffffu, ent < a.c.pages);
            }
            const uint32_t b = (uint32_t)__ffs((int)have) - 1u;
            have &= have - 1u;
            const uint32_t e = __shfl_sync(0xffffffffu, ent, (int)b), c = first + deal * (base + b);
            if (lane == 0u) {
                const uint32_t row = ((head0 + e * a.c.kv_heads) << a.c.page_log2) + ((c & ((1u << page_chunks) - 1u)) << 4);
                const uint32_t dst = ring + slot_in * kSlot;
                mbar_arrive_expect_tx(full + slot_in, kSlot);
                load_rows(dst, &a.kmap, row, full + slot_in);
                load_rows(dst + kSlot / 2u, &a.vmap, row, full + slot_in);
            }
            if (++slot_in == kStages) slot_in = 0u;
            return c;
        };
        uint32_t chunk[kStages];          // on their way; kNone: nothing more
#pragma unroll
        for (uint32_t i = 0; i < kStages; ++i) chunk[i] = issue();
        if (w.first && warp == kWarps - 1u) tell_part();

#pragma unroll
        for (uint32_t k = 0; k < sizeof(qv) / 16u; ++k) {
            const uint32_t x = k * kThreads + threadIdx.x;
            if (x < R * 16u) *reinterpret_cast<uint4 *>(&sm.q[x / 16u][8u * (x % 16u)]) = qv[k];
        }
        __syncthreads();
        // B operands: column g, dimensions 16 st + 2 t, + 1, + 8, + 9. Those of two tiles of rows stay in shared memory: with them
        // in registers, too, the loop spills
        auto operand = [&](int nt, int st, int half) { return *reinterpret_cast<const uint32_t *>(&sm.q[8u * (uint32_t)nt + g][16 * st + 8 * half + 2u * t]); };
        uint32_t qf[NT == 1 ? 8 : 1][2];
        if (NT == 1)
#pragma unroll
            for (int st = 0; st < 8; ++st) {
                qf[NT == 1 ? st : 0][0] = operand(0, st, 0);
                qf[NT == 1 ? st : 0][1] = operand(0, st, 1);
            }
        auto query = [&](int nt, int st, int half) { return NT == 1 ? qf[NT == 1 ? st : 0][half] : operand(nt, st, half); };
        uint32_t last[NT][2];             // the last position that columns 2 t and 2 t + 1 see
        const uint32_t open = (uint32_t)min(p0 + tr.tok, (uint64_t)0x7fffffffu);   // every row sees the positions up to it
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const uint32_t r = 8u * (uint32_t)nt + 2u * t + (uint32_t)e;
                last[nt][e] = r < rows ? (uint32_t)min(p0 + tr.at(r).x, (uint64_t)0x7fffffffu) : open;
            }

        uint64_t o[NT][8][2];             // dimensions 16 j + g and 16 j + g + 8: columns 2 t and 2 t + 1
        float m[NT][2], l[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            m[nt][0] = m[nt][1] = -INFINITY;
            l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
            for (int j = 0; j < 8; ++j) o[nt][j][0] = o[nt][j][1] = 0ull;
        }
        while (ok && chunk[0] != kNone) {
            const uint32_t key = chunk[0] * kChunk;
            ok = __all_sync(0xffffffffu, mbar_wait(full + slot, phase, &sm.err));
            if (!ok) break;
            const uint32_t in = ring + slot * kSlot;
            if (++slot == kStages) slot = 0u, phase ^= 1u;
            // two sums, so that the products wait for one another half as long
            float y[NT][4], y2[NT][4];
#pragma unroll
            for (uint32_t st = 0; st < 4u; ++st) {
                uint32_t ka[4], kb[4];
                load_matrices(ka, in + koff[st]);
                load_matrices(kb, in + kHalfChunk + koff[st]);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    if (st == 0u) {
                        mma_first<BF>(y[nt], ka, query(nt, 0, 0), query(nt, 0, 1));
                        mma_first<BF>(y2[nt], kb, query(nt, 4, 0), query(nt, 4, 1));
                    } else {
                        mma<BF>(y[nt], ka, query(nt, (int)st, 0), query(nt, (int)st, 1));
                        mma<BF>(y2[nt], kb, query(nt, (int)st + 4, 0), query(nt, (int)st + 4, 1));
                    }
                }
            }
            // scores: positions key + g (elements 0, 1) and key + g + 8 (2, 3), columns 2 t and 2 t + 1
            const bool masked = key + kChunk - 1u > open;   // some row does not see all of the chunk
            const uint32_t pa = key + g, pb = key + g + 8u;
            bool raise = false;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e) y[nt][e] = (y[nt][e] + y2[nt][e]) * kScoreScale;
            if (masked)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if ((e < 2 ? pa : pb) > last[nt][e & 1]) y[nt][e] = -INFINITY;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e) raise |= y[nt][e] > m[nt][e & 1] + kLazy;
            if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    float f[2] = {1.0f, 1.0f};
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float x = fmaxf(y[nt][e], y[nt][2 + e]);
                        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
                        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
                        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
                        if (x > m[nt][e] + kLazy) {
                            f[e] = m[nt][e] == -INFINITY ? 0.f : ex2(m[nt][e] - x);
                            m[nt][e] = x;
                            l[nt][e] *= f[e];
                        }
                    }
                    const uint64_t f2 = pair(f[0], f[1]);
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        o[nt][j][0] = mul2(o[nt][j][0], f2);
                        o[nt][j][1] = mul2(o[nt][j][1], f2);
                    }
                }
            }
            uint32_t bh[NT][2], bl[NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                float z[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    // a row that has seen no position yet has no maximum: its weights are 0 (NaN scores stay)
                    z[e] = y[nt][e] == -INFINITY ? 0.f : ex2(y[nt][e] - m[nt][e & 1] + kUnit<BF>);
                    l[nt][e & 1] += z[e];
                }
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const uint32_t hi = pack<BF>(z[2 * half], z[2 * half + 1]);
                    bh[nt][half] = transpose8(hi);
                    bl[nt][half] = transpose8(pack<BF>(z[2 * half] - unpack1<BF>(hi & 0xffffu), z[2 * half + 1] - unpack1<BF>(hi >> 16)));
                }
            }
            uint32_t bad = 0u;            // a value that is not finite where some row does not see it
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                uint32_t va[4];           // dimensions 16 j + g (0, 2) and + 8 (1, 3); positions 2 t, 2 t + 1 (0, 1) and + 8 (2, 3)
                load_matrices_t(va, in + (uint32_t)(j >> 2) * kHalfChunk + voff[j & 3]);
                if (masked) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint32_t p = key + 2u * t + (i < 2 ? 0u : 8u);
                        uint32_t n = nonfinite2<BF>(va[i]);
                        n &= (p > open ? 0xffffu : 0u) | (p + 1u > open ? 0xffff0000u : 0u);
                        va[i] &= ~n;
                        bad |= n;
                    }
                }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    float x[4];
                    mma_first<BF>(x, va, bl[nt][0], bl[nt][1]);
                    mma<BF>(x, va, bh[nt][0], bh[nt][1]);
                    o[nt][j][0] = add2(o[nt][j][0], pair(x[0], x[1]));
                    o[nt][j][1] = add2(o[nt][j][1], pair(x[2], x[3]));
                }
            }
            if (masked && __any_sync(0xffffffffu, bad != 0u)) {   // into the rows that do see them
                for (uint32_t k = 0; k < kChunk; ++k) {
                    if (key + k <= open) continue;
#pragma unroll
                    for (int j = 0; j < 8; ++j)
#pragma unroll
                        for (int hf = 0; hf < 2; ++hf) {
                            const uint32_t c = (2u * (uint32_t)(j & 3) + (uint32_t)hf) ^ (k & 7u);
                            uint16_t b;
                            asm volatile("ld.shared.u16 %0, [%1];" : "=h"(b) : "r"(in + 2u * kHalfChunk + (uint32_t)(j >> 2) * kHalfChunk + k * 128u + c * 16u + 2u * g) : "memory");
                            const float v = unpack1<BF>(b);
                            if (v - v == 0.f) continue;
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt)
                                o[nt][j][hf] = add2(o[nt][j][hf], pair(key + k <= last[nt][0] ? v : 0.f, key + k <= last[nt][1] ? v : 0.f));
                        }
                }
            }
            __syncwarp();                 // every lane is done with the slot
#pragma unroll
            for (uint32_t i = 0; i + 1u < kStages; ++i) chunk[i] = chunk[i + 1u];
            chunk[kStages - 1u] = issue();
        }
        if (!ok) {                        // nothing of this warp is left in flight; the rest of its rows become NaN
#pragma unroll
            for (uint32_t i = 0; i < kStages; ++i) {
                if (chunk[i] == kNone) break;
                const uint64_t t0 = global_ns();
                while (!mbar_try_wait(full + slot, phase) && global_ns() - t0 < kWaitLimitNs) {
                }
                if (++slot == kStages) slot = 0u, phase ^= 1u;
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) l[nt][0] = l[nt][1] = __int_as_float(0x7fffffff);
        }
        __syncthreads();                  // every warp is done with the ring: it takes the warps' outputs
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float x = l[nt][e];
                x += __shfl_xor_sync(0xffffffffu, x, 4);
                x += __shfl_xor_sync(0xffffffffu, x, 8);
                x += __shfl_xor_sync(0xffffffffu, x, 16);
                const uint32_t i = 8u * (uint32_t)nt + 2u * t + (uint32_t)e;
                if (g == 0u) sm.wml[warp][i] = make_float2(m[nt][e], x);
#pragma unroll
                for (int j = 0; j < 8; ++j)
#pragma unroll
                    for (int hf = 0; hf < 2; ++hf) {
                        float v[2];
                        unpair(o[nt][j][hf], v[0], v[1]);
                        sm.u.wrec[warp][i][16 * j + 8 * hf + (int)g] = v[e];
                    }
            }
        __syncthreads();
        const bool whole = w.head && w.tail;
        const uint32_t share = (R * (kDim / 4u) + piece.shared - 1u) / piece.shared;   // of a unit's sums, for each CTA that has it
        if (piece.shared > 1u) cluster_wait();
        float *const rec = record_of(a, w.record(), R);
        for (uint32_t x = threadIdx.x; x < rows * (kDim / 4u); x += kThreads) {
            const uint32_t i = x / (kDim / 4u), d = x % (kDim / 4u);
            float M = -INFINITY, L = 0.f, f[kWarps];
#pragma unroll
            for (uint32_t v = 0; v < kWarps; ++v) M = fmaxf(M, sm.wml[v][i].x);
#pragma unroll
            for (uint32_t v = 0; v < kWarps; ++v) {
                const float2 ml = sm.wml[v][i];
                f[v] = factor(ml, M);
                L = fmaf(f[v], ml.y, L);
            }
            float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (uint32_t v = 0; v < kWarps; ++v) {
                const float4 z = *reinterpret_cast<const float4 *>(&sm.u.wrec[v][i][4u * d]);
                y.x = fmaf(f[v], z.x, y.x);
                y.y = fmaf(f[v], z.y, y.y);
                y.z = fmaf(f[v], z.z, y.z);
                y.w = fmaf(f[v], z.w, y.w);
            }
            if (piece.shared > 1u) {
                const uint32_t to = x / share, rank = k8::cluster_rank();
                send(&sm.sent[rank * share + (x - to * share)], to, y);
                if (d < cluster) send(&sm.sent_ml[rank][i], d, make_float2(M, L));
            } else if (whole) {
                const float inv = L == 0.f ? 0.f : 1.0f / L;
                store4<BF>(a, s, h, tr.at(i), d, make_float4(y.x * inv, y.y * inv, y.z * inv, y.w * inv));
            } else {
                __stcg(reinterpret_cast<float4 *>(rec) + i * (kDim / 4u) + d, y);
                if (d == 0u) __stcg(reinterpret_cast<float2 *>(rec + R * kDim) + i, make_float2(M, L));
            }
        }
        if (piece.shared > 1u) {          // each CTA of the cluster joins its share
            k8::cluster_sync();           // nothing remote is touched from here on
            const uint32_t x = k8::cluster_rank() * share + threadIdx.x, i = x / (kDim / 4u), d = x % (kDim / 4u);
            static_assert(R * (kDim / 4u) <= 2u * kThreads, "a thread has one of the share's");
            if (threadIdx.x < share && i < rows) {
                float M = -INFINITY, L = 0.f;
                for (uint32_t c = 0; c < cluster; ++c) M = fmaxf(M, sm.sent_ml[c][i].x);
                float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
                for (uint32_t c = 0; c < cluster; ++c) {
                    const float2 ml = sm.sent_ml[c][i];
                    const float4 z = sm.sent[c * share + threadIdx.x];
                    const float f = factor(ml, M);
                    L = fmaf(f, ml.y, L);
                    y.x = fmaf(f, z.x, y.x);
                    y.y = fmaf(f, z.y, y.y);
                    y.z = fmaf(f, z.z, y.z);
                    y.w = fmaf(f, z.w, y.w);
                }
                const float inv = L == 0.f ? 0.f : 1.0f / L;
                store4<BF>(a, s, h, tr.at(i), d, make_float4(y.x * inv, y.y * inv, y.z * inv, y.w * inv));
            }
        }
        fence_ring();
        __syncthreads();                  // the ring may fill again
    }
}

// --------------------------------------------------------- partial sums ----
//
// The units that pieces cut: the CTAs whose number is that of the piece that a
// unit ends in join its records, a warp one or two rows (lane: a record's maximum
// and sum, then 4 dimensions), with the first records' loads on their way before
// their weights are known. Bound by latency (6.6 us behind a chunk's call, cold and
// alone); a call whose pieces are whole units leaves nothing to join, and one that
// cannot leave anything does not launch this.
struct MergeArgs : AttnArgs {
    uint32_t tile;                        // rows of a record
};

constexpr uint32_t kMergeWarps = 8;

// ROWS a warp, AHEAD records on their way: few rows have many records, many rows few
template <bool BF, uint32_t ROWS, uint32_t AHEAD>
__global__ void __launch_bounds__(kMergeWarps * 32) part_merge_kernel(const __grid_constant__ MergeArgs a)
{
    static_assert(32u % AHEAD == 0u, "the records of a round are loaded whole");
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
    wait_predecessor(a.early);
    const uint4 lo = __ldcg(reinterpret_cast<const uint4 *>(a.parts) + 2u * blockIdx.x), hi = __ldcg(reinterpret_cast<const uint4 *>(a.parts) + 2u * blockIdx.x + 1u);
    const uint32_t first = lo.x, count = lo.y, s = lo.z, h = lo.w, row0 = hi.x, rows = hi.y;
    const uint32_t r0 = (blockIdx.y * kMergeWarps + warp) * ROWS;
    if (first == ~0u || r0 >= rows) return;
    // record i of the unit
    auto record = [&](uint32_t i) { return record_of(a, i ? 2u * (first / 2u + i) : first, a.tile); };
    float M[ROWS], L[ROWS], f[ROWS];   // f: record b + lane's factor
    float4 x[ROWS], y[ROWS][AHEAD];
    auto load = [&](uint32_t i0) {
#pragma unroll
        for (uint32_t u = 0; u < ROWS; ++u)
#pragma unroll
            for (uint32_t i = 0; i < AHEAD; ++i)
                if (i0 + i < count) y[u][i] = __ldcg(reinterpret_cast<const float4 *>(record(i0 + i)) + min(r0 + u, rows - 1u) * (kDim / 4u) + lane);
    };
    load(0u);
#pragma unroll
    for (uint32_t u = 0; u < ROWS; ++u) {
        M[u] = -INFINITY;
        L[u] = 0.f;
        x[u] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    for (uint32_t b = 0; b < count; b += 32u) {
        float2 ml[ROWS];
#pragma unroll
        for (uint32_t u = 0; u < ROWS; ++u)
            ml[u] = b + lane < count ? __ldcg(reinterpret_cast<const float2 *>(record(b + lane) + a.tile * kDim) + min(r0 + u, rows - 1u)) : make_float2(-INFINITY, 0.f);
#pragma unroll
        for (uint32_t u = 0; u < ROWS; ++u) {
            float most = ml[u].x;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
            most = fmaxf(most, M[u]);
            const float before = factor(make_float2(M[u], L[u]), most);
            f[u] = factor(ml[u], most);
            float sum = f[u] * ml[u].y;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            M[u] = most;
            L[u] = fmaf(before, L[u], sum);
            x[u] = make_float4(x[u].x * before, x[u].y * before, x[u].z * before, x[u].w * before);
        }
        const uint32_t n = min(count - b, 32u);
        for (uint32_t i0 = 0; i0 < n; i0 += AHEAD) {
#pragma unroll
            for (uint32_t u = 0; u < ROWS; ++u)
#pragma unroll
                for (uint32_t i = 0; i < AHEAD; ++i) {
                    const float fi = __shfl_sync(0xffffffffu, f[u], (int)(i0 + i));
                    if (i0 + i >= n) continue;
                    x[u].x = fmaf(fi, y[u][i].x, x[u].x);
                    x[u].y = fmaf(fi, y[u][i].y, x[u].y);
                    x[u].z = fmaf(fi, y[u][i].z, x[u].z);
                    x[u].w = fmaf(fi, y[u][i].w, x[u].w);
                }
            load(b + i0 + AHEAD);
        }
    }
#pragma unroll
    for (uint32_t u = 0; u < ROWS; ++u) {
        if (r0 + u >= rows) break;
        const float inv = L[u] == 0.f ? 0.f : 1.0f / L[u];
        const uint32_t row = row0 + r0 + u, tok = row / a.group;
        store4<BF>(a, s, h, make_uint2(tok, row - tok * a.group), lane, make_float4(x[u].x * inv, x[u].y * inv, x[u].z * inv, x[u].w * inv));
    }
}

// CTAs that share a unit, and CTAs in all: the largest clusters that give each unit one, all on the device at once, with a
// round of chunks for each CTA; else none, and all SMs
template <bool BF, int NT>
cudaError_t launch_few_of(FewArgs &a, uint64_t units, int dev, int sms, uint32_t &ctas, cudaStream_t stream)
{
    const cudaError_t e = k8::allow<few_kernel<BF, NT>>(dev, (int)sizeof(Smem<NT>));
    if (e != cudaSuccess) return e;
    uint32_t cluster = 1;
    ctas = std::min((uint32_t)sms, kMaxCtas);
    const uint32_t rounds = (a.c.limit + kChunk * kWarps - 1) / (kChunk * kWarps);
    for (uint32_t c = std::min({k8::kMaxCluster, rounds, (uint32_t)(units <= (uint64_t)sms ? sms / units : 0)}); a.keep && c > 1; --c) {
        const uint32_t n = std::min(k8::clusters_at_once<few_kernel<BF, NT>>(dev, c, kThreads, sizeof(Smem<NT>)), kMaxCtas / c);
        if (n < units) continue;
        cluster = c;
        ctas = n * c;
        break;
    }
    a.worth = always_whole(a, units, ctas, kChunk, kWorth, cluster) ? kWorth : kWorthMore;
    return k8::launch(few_kernel<BF, NT>, dim3(ctas), kThreads, sizeof(Smem<NT>), cluster, a, sms, stream);
}

}  // namespace

cudaError_t launch_merge(const AttnArgs &a, bool bf, uint32_t rows, uint32_t ctas, int sms, cudaStream_t stream)
{
    MergeArgs m{};
    static_cast<AttnArgs &>(m) = a;
    m.tile = rows;
    const uint32_t threads = kMergeWarps * 32;
    if (rows <= 16) {
        const dim3 grid(ctas, (rows + kMergeWarps - 1) / kMergeWarps);
        return bf ? k8::launch(part_merge_kernel<true, 1, 8>, grid, threads, 0, 1, m, sms, stream)
                  : k8::launch(part_merge_kernel<false, 1, 8>, grid, threads, 0, 1, m, sms, stream);
    }
    const dim3 grid(ctas, (rows + 2 * kMergeWarps - 1) / (2 * kMergeWarps));
    return bf ? k8::launch(part_merge_kernel<true, 2, 4>, grid, threads, 0, 1, m, sms, stream)
              : k8::launch(part_merge_kernel<false, 2, 4>, grid, threads, 0, 1, m, sms, stream);
}

// The few-rows form, for units of 8 nt rows; maps: see FewArgs
cudaError_t launch_few(const AttnArgs &a, const CUtensorMap &kmap, const CUtensorMap &vmap, bool bf, int nt, int dev, int sms,
                       cudaStream_t stream)
{
    FewArgs f{};
    static_cast<AttnArgs &>(f) = a;
    f.kmap = kmap;
    f.vmap = vmap;
    f.keep = lanes_keep(a, 8u * (uint32_t)nt, kChunk, kExtra);
    const uint32_t rows = 8u * (uint32_t)nt;
    const uint64_t units = (uint64_t)a.c.nseq * a.c.kv_heads * (((uint64_t)a.r.tokens * a.group + rows - 1) / rows);
    uint32_t ctas;
    const cudaError_t e = nt == 1 ? (bf ? launch_few_of<true, 1>(f, units, dev, sms, ctas, stream) : launch_few_of<false, 1>(f, units, dev, sms, ctas, stream))
                                  : (bf ? launch_few_of<true, 2>(f, units, dev, sms, ctas, stream) : launch_few_of<false, 2>(f, units, dev, sms, ctas, stream));
    if (e != cudaSuccess || f.worth == kWorth) return e;
    return launch_merge(a, bf, rows, ctas, sms, stream);
}

}  // namespace paged
}  // namespace atlas
