// Attention over a paged KV cache for many query rows per KV head, on tcgen05
// tensor cores (sm_100a): paged_attn's form for prompts and larger chunks.
// (gqa_single_token per token in the reference, src/brain_runtime.c:1407-1528.)
//
// A unit is one or two tiles of whole tokens' query rows of a KV head (row =
// token * group + head: the group's heads share every key), up to 128 rows each.
// A CTA takes a piece of the line of all units' keys (paged.cuh), 128 at a time:
//   S = Q K^T   M = 128, N = 128 keys, K = 128 dimensions, into tensor memory
//   P = 2^(S - maximum), as 16-bit values into the columns that S leaves
//   O += P V    M = 128, N = 128 dimensions, K = 128 keys, A from tensor memory;
//               V as it lies in the pages: [key][dimension], N along the rows
// Q, K and V come by TMA into 128-byte swizzled tiles; a page is one copy per 64
// dimensions, and one that is not there is read from behind the pool's end, which
// gives zeros.
//
// Warps of a CTA (12):
//   0-7   softmax, one thread per row, its 128 scores in registers: maximum
//         (lazy: raised only when a score passes it by 2^8, and only then the output
//         in tensor memory is taken down), weights in two halves of 64 keys, each
//         multiplied by V while the next is made; at a unit's end, the output;
//   8     plans and copies; 9 issues the MMAs: P V of a tile of keys, then the next keys'
//         scores of the same rows, so that one tile's softmax runs under the other's
//         MMAs;
//   10-11 of a tile of keys that not all rows see, take values out of V that are
//         not finite: a weight of 0 would not hide them. The softmax threads
//         add them to the rows that do see them. A slot of the ring waits for them as
//         for the MMAs.
// With one tile of rows, both softmax groups have it and take turns at the keys,
// each with an output and a state of its own, joined at the end.
//
// P is rounded to the cache's type, as the product's operand, while its sum is not: a
// choice. Its rest as a second term would make three products of two, on the pipe that
// bounds long prompts. Each weight is off by half a step at most and independently of the
// others: against 64 bits, outputs are off by 2.8e-4 (binary16) and 2.0e-3 (bfloat16),
// relative 2-norm, where a plain form in fp32, rounded once at the end, is off by 2.1e-4
// and 1.6e-3. (paged_attn.cu, where the products cost nothing, takes both terms.)
//
// Tensor cores truncate their sums: 2^-24 of the output per MMA of 16 keys at
// most, so 256 tiles of keys (2048 MMAs, 2^-13) are summed in tensor memory, and
// longer pieces in steps of that, joined in fp32.
// Tensor memory: 2 x 128 columns of scores / weights, 2 x 128 of output.
// Every wait is bounded; after a timeout the CTA's rows are NaN.
//
// Bound by the chain of a row tile's scores, softmax and second product, about 3200
// cycles per 128 keys, of which two run: the tensor pipe and the exponentials are both
// busy 56 % of the time. 8192 tokens of 40 heads on 8: 661 to 686 us with the partial sums
// in short rows of calls, 1.0 to 1.04 PFLOP/s, 60 to 62 % of the measured bfloat16 rate;
// 757, 0.91 PFLOP/s and 54 %, when repeated under the power cap. (An earlier build with a
// quarter of the exponentials on the FMA units: 633 instead of 623.) Short calls are bound
// by what comes before the first scores and behind the last: 512 tokens of 28 heads on 4
// 16 us, 7 tokens of 4 sequences over 8001 27.8; in tables with room for 32768 positions 19
// and 28, as the launch that joins follows.
#include <algorithm>
#include <atomic>
#include <cfloat>
#include <cmath>
#include <type_traits>
#include "../../include/atlas_cuda.h"
#include "paged.cuh"
#include "tcgen05.cuh"

namespace atlas {
namespace paged {

using k8::add2;
using k8::fma2;
using k8::kScoreScale;
using k8::pair;
using k8::unpair;
using k8::wait_predecessor;

namespace {

constexpr uint32_t kTileRows = 128, kTileKeys = 128, kMostTiles = 256;
constexpr uint32_t kLoadWarp = 8, kMmaWarp = 9, kCheckWarp = 10, kCheckers = 2, kThreads = 12 * 32;
// Registers per thread of a warpgroup after the split, of 168 at launch
constexpr uint32_t kSoftmaxRegs = 208, kOtherRegs = 88, kLaunchRegs = 168;
static_assert(2 * kSoftmaxRegs + kOtherRegs <= 3 * kLaunchRegs, "what the softmax warps get is what the others leave");
constexpr uint32_t kHalf = 128 * 128;              // bytes of 128 rows x 64 values, swizzled
constexpr uint32_t kTile = 2 * kHalf;
constexpr uint32_t kMaxStages = 6;
// tiles of keys: what joining partial sums takes, and beginning and ending a unit. With 1 or 5 instead of 3: 7 tokens of 4
// sequences over 8001 30.3 or 28.8 us instead of 27.8, 8192 tokens 743 or 684 instead of 677, 8 x 2048 517 or 526 instead of 517
constexpr uint32_t kWorth = 6, kExtra = 3;
constexpr float kLazy = 8.0f;
// Weights are 2^(score - maximum + kUnit): binary16 keeps 24 bits below the largest; bfloat16 has fp32's range, and small
// weights leave the sums of large values room
template <bool BF>
constexpr float kUnit = BF ? -24.0f : 6.0f;

// Weights go to the second product in so many parts: with four, the softmax warps' extra waits cost more than the product's
// earlier start gains but in the longest calls (7 tokens of 4 sequences over 8001 29.7 us instead of 27.8, 333 over 5001 48
// instead of 42, 8 x 2048 531 instead of 517, 8192 635 to 667 instead of 669 to 686)
constexpr uint32_t kParts = 2;

struct PromptArgs : AttnArgs {
    CUtensorMap kmap, vmap;      // [2][rows of the pool][64] each
    CUtensorMap qmap;            // [2][token][head][64]
    uint32_t tokens_per_tile;
    Divisor by_tile;             // by a unit's rows
    uint32_t wide;               // output rows lie on 32-byte boundaries
};

// Some tiles of keys of a unit, as the planner hands them to the other warps
struct Step {
    uint32_t n, k_begin;                           // tiles of keys (0: the end), the first one
    uint32_t s, h, rows, tok0, p0;
    uint32_t record, whole, again;                 // where partial sums go; it is all of its unit; it goes on with a unit
    uint32_t bad;                                  // a value was taken out of V
};
constexpr uint32_t kSteps = 4;

struct OneState {
    float2 state[2][kTileRows];                    // [group]: the rows' maxima and sums
};
struct NoState {
};

template <bool ONE>
struct Bars : std::conditional_t<ONE, OneState, NoState> {
    Step step[kSteps];
    uint64_t s_full[2], p_full[2][kParts], o_full[2], o_free[2], x_full[2], x_free[2], full[kMaxStages], free[kMaxStages], checked[kMaxStages], step_full[kSteps],
        step_free[kSteps], q_full, q_free, fin;
    uint32_t tmem, status;
    uint32_t here[8];                              // of the tile of keys at its number % 8: bit i, its i-th 16 positions have a page
};

template <bool ONE>
constexpr uint32_t kStages = ONE ? 6u : 5u;
template <bool ONE>
constexpr size_t kSmem = (ONE ? 1 : 2) * kTile + kStages<ONE> * kTile + sizeof(Bars<ONE>);
template <bool ONE>
constexpr uint32_t kRecordRows = ONE ? kTileRows : 2 * kTileRows;
static_assert(kSmem<true> <= k8::kMaxSmem && kSmem<false> <= k8::kMaxSmem, "the tiles exceed a CTA's shared memory");
static_assert(sizeof(PieceSmem) <= 2 * kTile, "find_together works in the stages' place");

// fp32 accumulator, M = 128, N = 128; A and B of one 16-bit type; B as rows along N where ACROSS
template <bool BF, bool ACROSS>
constexpr uint32_t kInstr = (1u << 4) | (BF ? (1u << 7) | (1u << 10) : 0u) | (ACROSS ? 1u << 16 : 0u) | ((128u >> 3) << 17) | ((128u >> 4) << 24);

// A box of 64 values x rows of the pool
__device__ __forceinline__ void load_box(uint32_t dst, const CUtensorMap *map, uint32_t row, uint32_t half, uint64_t *bar)
{
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                 ::"r"(dst), "l"(map), "r"(0), "r"((int)row), "r"((int)half), "r"(smem_addr(bar))
                 : "memory");
}
// 64 values x the group's heads x a tile's tokens of Q
__device__ __forceinline__ void load_queries(uint32_t dst, const CUtensorMap *map, uint32_t head, uint32_t token, uint32_t half, uint64_t *bar)
{
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
                 ::"r"(dst), "l"(map), "r"(0), "r"((int)head), "r"((int)token), "r"((int)half), "r"(smem_addr(bar))
                 : "memory");
}

// 32 bytes at once, to a 32-byte boundary
__device__ __forceinline__ void store32(void *p, const uint32_t (&x)[8])
{
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3]), "r"(x[4]),
                 "r"(x[5]), "r"(x[6]), "r"(x[7])
                 : "memory");
}

// Where the tiles of keys of a step go: one buffer after the other
template <uint32_t STAGES>
struct Ring {
    uint32_t slot = 0u, phase = 0u;
    __device__ __forceinline__ void next()
    {
        if (++slot == STAGES) {
            slot = 0u;
            phase ^= 1u;
        }
    }
};

template <bool BF, bool ONE>
__global__ void __launch_bounds__(kThreads, 1) prompt_kernel(const __grid_constant__ PromptArgs a)
{
    constexpr uint32_t STAGES = kStages<ONE>;
    extern __shared__ __align__(1024) uint8_t prompt_smem[];
    uint8_t *const qs = prompt_smem, *const kv = qs + (ONE ? 1u : 2u) * kTile;
    Bars<ONE> &b = *reinterpret_cast<Bars<ONE> *>(kv + STAGES * kTile);
    volatile uint32_t *const err = &b.status;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
    if (threadIdx.x == 0) {
        for (int t = 0; t < 2; ++t) {
            mbar_init(&b.s_full[t], 1u);
            for (uint32_t c = 0; c < kParts; ++c) mbar_init(&b.p_full[t][c], 4u);
            mbar_init(&b.o_full[t], 1u);
            mbar_init(&b.o_free[t], ONE ? 8u : 4u);
            mbar_init(&b.x_full[t], 4u);
            mbar_init(&b.x_free[t], 4u);
        }
        for (uint32_t i = 0; i < STAGES; ++i) {
            mbar_init(&b.full[i], 1u);
            mbar_init(&b.free[i], 1u + kCheckers);     // the MMAs and the warps that look through V
            mbar_init(&b.checked[i], kCheckers);
        }
        for (uint32_t i = 0; i < kSteps; ++i) {
            mbar_init(&b.step_full[i], 1u);
            mbar_init(&b.step_free[i], 11u);       // every warp but the one that plans
        }
        mbar_init(&b.q_full, 1u);
        mbar_init(&b.q_free, 1u);
        mbar_init(&b.fin, 1u);
        b.status = kStatusOk;
        fence_mbar_init();
    }
    if (warp == kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&b.tmem)), "r"(512u)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (warp == kLoadWarp && lane < 3u)
        asm volatile("prefetch.tensormap [%0];" ::"l"(lane == 0u ? &a.qmap : lane == 1u ? &a.kmap : &a.vmap) : "memory");
    wait_predecessor(a.early);
    const uint32_t tile_rows = a.tokens_per_tile * a.group;      // of 128 in tensor memory
    const Cut<kTileKeys, kExtra> cut{a, (ONE ? 1u : 2u) * tile_rows, a.by_tile};
    Piece piece;
    piece.left = 0u;
    if (!a.keep) piece = find_together<kThreads / 32u>(cut, *reinterpret_cast<PieceSmem *>(kv), 2u, kWorth);
    fence_before();
    fence_async();
    __syncthreads();
    fence_after();
    const uint32_t tmem = b.tmem;   // scores / weights of group t: column 128 t; output: 256 + 128 t

    // The end of a CTA, for every warp in the branch of its registers
    auto leave = [&]() {
        fence_before();
        __syncthreads();
        if (warp == kMmaWarp) {
            fence_after();
            asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
        }
    };
    // step number i: whether there is one; a warp that is done with it lets its place be used again
    auto there_is = [&](uint32_t i) { return wait_warp(&b.step_full[i % kSteps], i / kSteps & 1u, err) && b.step[i % kSteps].n != 0u; };
    auto done_with = [&](uint32_t i) {
        __syncwarp();
        if (lane == 0u) mbar_arrive(&b.step_free[i % kSteps]);
    };
    // tiles of rows that the unit has
    auto tiles_of = [&](uint32_t rows) { return !ONE && rows > tile_rows ? 2u : 1u; };
    if (warp >= kLoadWarp) {
        fewer_registers<kOtherRegs>();   // the whole warpgroup
        if (warp == kLoadWarp) {
            // ------------------------------------------- plan and copies --
            // The only warp that follows the piece through its units; the others get steps. It is ahead of them all.
            if (a.keep) piece = find_kept(cut, 2u, kWorth);
            Walk<kTileKeys, kExtra, kMostTiles> w(cut, piece);
            Ring<STAGES> ring;
            uint32_t used = 0u, i = 0u, number = 0u;   // copies so far; steps; tiles of keys
            bool ok = true;
            const uint32_t page_log2 = a.c.page_log2, per = 7u - page_log2;   // log2 of pages per tile of keys
            const uint32_t of = lane >> 1, half = lane & 1u;                   // this lane's page of a tile and half of its dimensions
            const bool mine = of < (1u << per);
            const uint32_t nowhere = (a.c.layers * a.c.pages * a.c.kv_heads) << page_log2;   // behind the pool's end: zeros
            for (;; ++i) {
                const bool more = w.more();
                if (i >= kSteps) ok = wait_warp(&b.step_free[i % kSteps], (i / kSteps - 1u) & 1u, err);
                if (!ok) break;
                const uint32_t n = more ? w.k_end - w.k_begin : 0u, k_begin = w.k_begin;
                // this lane's page of the step's tile j, and where it begins; the first ones' loads are on their way first of all
                const uint32_t seen = more ? (uint32_t)min((uint64_t)w.q.p0 + divide(w.row0() + w.rows() - 1u, a.by_group) + 1u, (uint64_t)a.c.limit) : 0u;
                const int32_t *const entries = a.c.table + (size_t)w.p.s * a.c.max_pages;
                const uint32_t head0 = a.layer * a.c.pages * a.c.kv_heads + w.p.h;
                auto page_of = [&](uint32_t j) {
                    const uint32_t e = ((k_begin + j) << per) + of;
                    return mine && j < n && (uint64_t)e << page_log2 < seen ? (uint32_t)__ldcg(entries + e) : ~0u;
                };
                auto row_of = [&](uint32_t e) { return e < a.c.pages ? (head0 + e * a.c.kv_heads) << page_log2 : nowhere; };
                uint32_t page = page_of(0u), page_next = page_of(1u);
                const uint32_t tiles = more ? tiles_of(w.rows()) : 0u, tok0 = more ? divide(w.row0(), a.by_group) : 0u;
                if (more) {
                    if (i) ok = wait_warp(&b.q_free, (i - 1u) & 1u, err);
                    if (!ok) break;
                    if (lane == 0u) {
                        mbar_arrive_expect_tx(&b.q_full, tiles * tile_rows * 256u);
                        for (uint32_t t = 0; t < tiles; ++t)
                            for (uint32_t hf = 0; hf < 2u; ++hf)
                                load_queries(smem_addr(qs + t * kTile + hf * kHalf), &a.qmap, w.p.h * a.group, w.p.s * a.r.tokens + tok0 + t * a.tokens_per_tile, hf,
                                             &b.q_full);
                    }
                }
                if (lane == 0u) {
                    Step &st = b.step[i % kSteps];
                    st.n = n;
                    st.bad = 0u;
                    if (more) {
                        st.s = w.p.s;
                        st.h = w.p.h;
                        st.rows = w.rows();
                        st.tok0 = tok0;
                        st.p0 = w.q.p0;
                        st.k_begin = k_begin;
                        st.record = w.record();
                        st.again = w.again ? 1u : 0u;
                        st.whole = w.leaves() && w.head && w.tail ? 1u : 0u;
                    }
                    mbar_arrive(&b.step_full[i % kSteps]);
                }
                __syncwarp();
                if (!more) break;
                uint32_t at = row_of(page), next = row_of(page_next);
                // which of a tile's 16 positions have a page, for the softmax warps; before K's copies, whose end they wait for
                auto tell = [&](uint32_t row) {
                    const uint32_t have = __ballot_sync(0xffffffffu, mine && row != nowhere);   // lane 2 i: page i
                    if (lane == 0u) {
                        uint32_t bits = 0u;
                        for (uint32_t k = 0; k < 8u; ++k) bits |= (have >> (2u * (k >> (page_log2 - 4u))) & 1u) << k;
                        b.here[number & 7u] = bits;
                    }
                    ++number;
                };
                auto copy = [&](const CUtensorMap *map, uint32_t row) {
                    if (used >= STAGES) ok = ok && wait_warp(&b.free[ring.slot], ring.phase ^ 1u, err);
                    if (!ok) return;
                    if (lane == 0u) mbar_arrive_expect_tx(&b.full[ring.slot], kTile);
                    __syncwarp();
                    if (mine) load_box(smem_addr(kv + ring.slot * kTile + half * kHalf) + ((of << page_log2) << 7), map, row, half, &b.full[ring.slot]);
                    ring.next();
                    ++used;
                };
                // in the order in which the MMAs take them: with one tile of rows, a tile of K more before V
                if (ONE) {
                    tell(at);
                    copy(&a.kmap, at);
                }
                for (uint32_t j = 0; ok && j < n; ++j) {
                    page = page_of(j + 2u);
                    if (!ONE || j + 1u < n) {
                        tell(ONE ? next : at);
                        copy(&a.kmap, ONE ? next : at);
                    }
                    copy(&a.vmap, at);
                    at = next;
                    next = row_of(page);
                }
                if (!ok) break;
                w.next();
            }
            const Part part = Walk<kTileKeys, kExtra, kMostTiles>(cut, piece).part();
            if (lane == 0u) reinterpret_cast<Part *>(a.parts)[blockIdx.x] = part;
            if (!ok) {   // nothing of this CTA is left in flight: the last copies are waited for
                const uint64_t t0 = global_ns();
                for (uint32_t k = 0; k < 2u && k < i + 1u; ++k)
                    while (!mbar_try_wait(&b.q_full, (i - k) & 1u) && global_ns() - t0 < kWaitLimitNs) {
                    }
                for (uint32_t k = 0; k < min(used, STAGES); ++k) {
                    const uint32_t n = used - 1u - k, slot = n % STAGES;
                    while (!mbar_try_wait(&b.full[slot], n / STAGES & 1u) && global_ns() - t0 < kWaitLimitNs) {
                    }
                }
            }
            leave();
            if (b.status != kStatusOk) {   // a wait ran out: all rows of the piece become NaN, those of partial sums by their sums of weights
                const float nan = __int_as_float(0x7fffffff);
                for (Walk<kTileKeys, kExtra> u(cut, piece); u.more(); u.next())
                    for (uint32_t r = lane; r < u.rows(); r += 32u) {
                        if (u.head && u.tail) {
                            const uint32_t row = u.row0() + r, tok = divide(row, a.by_group);
                            for (uint32_t d = 0; d < kDim / 4u; ++d) store4<BF>(a, u.p.s, u.p.h, make_uint2(tok, row - tok * a.group), d, make_float4(nan, nan, nan, nan));
                        } else {
                            *(reinterpret_cast<float2 *>(record_of(a, u.record(), kRecordRows<ONE>) + kRecordRows<ONE> * kDim) + r) = make_float2(0.f, nan);
                        }
                    }
            }
        } else if (warp == kMmaWarp) {
            // --------------------------------------------------------- MMA --
            const bool leader = elected();
            Ring<STAGES> ring;
            uint32_t i = 0u, turns[2] = {0u, 0u}, ends[2] = {0u, 0u};   // of a group: tiles of keys, and steps, so far
            uint32_t check_phase = 0u;                 // bit k: of slot k
            bool ok = true;
            const uint64_t qd = operand(smem_addr(qs)), kd = operand(smem_addr(kv)), vd = operand_across(smem_addr(kv), kHalf);
            for (; ok && there_is(i); ++i) {
                const Step &st = b.step[i % kSteps];
                const uint32_t tiles = tiles_of(st.rows), n = st.n, k_begin = st.k_begin;
                const uint64_t open = (uint64_t)st.p0 + st.tok0;   // every row sees the positions up to it
                done_with(i);
                if (leader) {
                    ok = mbar_wait(&b.q_full, i & 1u, err);
                    // scores of the keys in ring slot `slot` by tile of rows qt, into group t's columns
                    auto scores = [&](uint32_t t, uint32_t qt, uint32_t slot) {
                        const uint64_t q = qd + (uint64_t)(qt * (kTile >> 4)), k = kd + (uint64_t)(slot * (kTile >> 4));
#pragma unroll
                        for (uint32_t s = 0; s < 8u; ++s) {
                            const uint32_t off = (s >> 2) * (kHalf >> 4) + (s & 3u) * 2u;
                            mma_ss(tmem + 128u * t, q + off, k + off, kInstr<BF, false>, s != 0u);
                        }
                        commit(&b.s_full[t]);
                    };
                    // group t's weights times the values in slot `slot`
                    auto output = [&](uint32_t t, uint32_t slot, bool begin) {
                        const uint64_t v = vd + (uint64_t)(slot * (kTile >> 4));
#pragma unroll
                        for (uint32_t c = 0; c < kParts; ++c) {
                            if (!(ok = ok && mbar_wait(&b.p_full[t][c], turns[t] & 1u, err))) return;
                            fence_after();
#pragma unroll
                            for (uint32_t s = 8u / kParts * c; s < 8u / kParts * (c + 1u); ++s)   // 16 keys: 8 columns of P, 2048 bytes of V
                                mma_ts(tmem + 256u + 128u * t, tmem + 128u * t + 8u * s, v + s * 128u, kInstr<BF, true>, !begin || s != 0u);
                        }
                        ++turns[t];
                    };
                    // the tile of V of the step's keys j is there, and looked through if need be
                    auto values = [&](uint32_t j, const Ring<STAGES> &r) {
                        ok = ok && mbar_wait(&b.full[r.slot], r.phase, err);
                        if ((uint64_t)(k_begin + j + 1u) * kTileKeys > open + 1u) {
                            ok = ok && mbar_wait(&b.checked[r.slot], check_phase >> r.slot & 1u, err);
                            check_phase ^= 1u << r.slot;
                        }
                    };
                    auto keys = [&](const Ring<STAGES> &r) { ok = ok && mbar_wait(&b.full[r.slot], r.phase, err); };
                    // a group's output may be overwritten
                    auto fresh = [&](uint32_t t) {
                        if (ends[t]) ok = ok && mbar_wait(&b.o_free[t], (ends[t] - 1u) & 1u, err);
                    };
                    Ring<STAGES> rk = ring;
                    keys(rk);
                    if (ONE) {   // the groups take turns at the keys
                        if (ok) {
                            fence_after();
                            scores(0u, 0u, rk.slot);
                            commit(&b.free[rk.slot]);
                            rk.next();
                        }
                        for (uint32_t j = 0; ok && j < n; ++j) {
                            const uint32_t t = j & 1u;
                            if (j + 1u < n) {   // K of the next tile lies before V of this one
                                if (j == 0u) {
                                    keys(rk);
                                    if (!ok) break;
                                    fence_after();
                                    scores(1u, 0u, rk.slot);
                                    commit(&b.free[rk.slot]);
                                }
                                rk.next();
                            }
                            // rk: V of tile j
                            values(j, rk);
                            if (j < 2u) fresh(t);
                            if (!ok) break;
                            fence_after();
                            output(t, rk.slot, j < 2u);
                            if (!ok) break;
                            commit(&b.free[rk.slot]);
                            if (j + 2u >= n) commit(&b.o_full[t]);
                            rk.next();
                            if (j + 2u < n) {   // K of tile j + 2
                                keys(rk);
                                if (!ok) break;
                                fence_after();
                                scores(t, 0u, rk.slot);
                                commit(&b.free[rk.slot]);
                                if (j + 3u == n) commit(&b.q_free);
                            }
                        }
                        if (ok && n <= 2u) commit(&b.q_free);
                        for (uint32_t t = 0; t < min(n, 2u); ++t) ++ends[t];
                    } else {
                        if (ok) {
                            fence_after();
                            for (uint32_t t = 0; t < tiles; ++t) scores(t, t, rk.slot);
                            commit(&b.free[rk.slot]);
                            if (n == 1u) commit(&b.q_free);
                        }
                        for (uint32_t j = 0; ok && j < n; ++j) {
                            Ring<STAGES> rv = rk;
                            rv.next();
                            rk = rv;
                            rk.next();   // K of the next tile
                            for (uint32_t t = 0; ok && t < tiles; ++t) {
                                if (t == 0u) values(j, rv);
                                if (j == 0u) fresh(t);
                                if (!ok) break;
                                fence_after();
                                output(t, rv.slot, j == 0u);
                                if (!ok) break;
                                if (t + 1u == tiles) commit(&b.free[rv.slot]);
                                if (j + 1u == n) commit(&b.o_full[t]);
                                if (j + 1u < n) {
                                    if (t == 0u) keys(rk);
                                    if (!ok) break;
                                    fence_after();
                                    scores(t, t, rk.slot);
                                    if (t + 1u == tiles) {
                                        commit(&b.free[rk.slot]);
                                        if (j + 2u == n) commit(&b.q_free);
                                    }
                                }
                            }
                        }
                        for (uint32_t t = 0; t < tiles; ++t) ++ends[t];
                    }
                    ring = rk;
                }
                __syncwarp();
                ok = __any_sync(0xffffffffu, leader && ok);
            }
            if (leader) {
                // nothing of this CTA is left in flight when tensor memory is freed
                commit(&b.fin);
                const uint64_t t0 = global_ns();
                while (!mbar_try_wait(&b.fin, 0u) && global_ns() - t0 < kWaitLimitNs) {
                }
            }
            __syncwarp();
            leave();
        } else {
            // ------------------------------------------------------ checks --
            // Every copy is waited for, in order: a barrier tells a phase only from the one before. So that the next copy into a slot
            // is not done before a warp has seen this one, each arrives on the slot's `free`, too.
            Ring<STAGES> ring;
            uint32_t i = 0u;
            bool ok = true;
            auto leave_slot = [&]() {
                if (lane == 0u) mbar_arrive(&b.free[ring.slot]);
                ring.next();
            };
            auto pass = [&]() {
                ok = ok && wait_warp(&b.full[ring.slot], ring.phase, err);
                if (ok) leave_slot();
            };
            for (; ok && there_is(i); ++i) {
                Step &st = b.step[i % kSteps];
                const uint32_t n = st.n, k_begin = st.k_begin;
                const uint64_t open = (uint64_t)st.p0 + st.tok0;
                if (ONE) pass();
                for (uint32_t j = 0; ok && j < n; ++j) {
                    if (ONE ? j + 1u < n : true) pass();
                    const uint64_t key0 = (uint64_t)(k_begin + j) * kTileKeys;
                    ok = ok && wait_warp(&b.full[ring.slot], ring.phase, err);
                    if (!ok) break;
                    if (key0 + kTileKeys > open + 1u) {
                        // keys from `from` on are not seen by all rows; eight keys' 64 values a turn, 16 bytes a lane. A value's exponent
                        // is all ones where adding one to it carries into the sign's place.
                        constexpr uint32_t kExp = BF ? 0x7f807f80u : 0x7c007c00u, kOne = BF ? 0x00800080u : 0x04000400u;
                        const uint32_t from = open >= key0 ? (uint32_t)(open - key0) + 1u : 0u;
                        uint4 *const v = reinterpret_cast<uint4 *>(kv + ring.slot * kTile);
                        bool found = false;
#pragma unroll 4
                        for (uint32_t x = from * 8u + (threadIdx.x - kCheckWarp * 32u); x < kTileKeys * 8u; x += 32u * kCheckers)
#pragma unroll
                            for (uint32_t hf = 0; hf < 2u; ++hf) {
                                const uint4 y = v[hf * (kHalf / 16u) + x];
                                const uint32_t any = ((y.x & kExp) + kOne) | ((y.y & kExp) + kOne) | ((y.z & kExp) + kOne) | ((y.w & kExp) + kOne);
                                if (any & 0x80008000u) {
                                    v[hf * (kHalf / 16u) + x] = make_uint4(y.x & ~nonfinite2<BF>(y.x), y.y & ~nonfinite2<BF>(y.y), y.z & ~nonfinite2<BF>(y.z), y.w & ~nonfinite2<BF>(y.w));
                                    found = true;
                                }
                            }
                        if (found) st.bad = 1u;
                        fence_async();
                        __syncwarp();
                        if (lane == 0u) mbar_arrive(&b.checked[ring.slot]);
                    }
                    leave_slot();
                }
                done_with(i);
            }
            leave();
        }
    } else {
        more_registers<kSoftmaxRegs>();
        // --------------------------------------------------------- softmax --
        const uint32_t t = warp >> 2, quarter = warp & 3u, row = quarter * 32u + lane;
        const uint32_t at = tmem + ((quarter * 32u) << 16) + 128u * t, out_at = tmem + ((quarter * 32u) << 16) + 256u;
        uint32_t turns = 0u, ends[2] = {0u, 0u}, number = 0u;   // number: tiles of keys of the steps before
        float mc = -INFINITY, lc = 0.f;                          // the state of the unit's steps before
        bool ok = true;
        for (uint32_t i = 0; ok && there_is(i); ++i) {
            const Step &st = b.step[i % kSteps];
            const uint32_t n = st.n;
            if (!ONE && t >= tiles_of(st.rows)) {
                number += n;
                done_with(i);
                continue;
            }
            constexpr uint32_t j_step = ONE ? 2u : 1u;
            const uint32_t j_first = ONE ? t : 0u;
            const float group_inv = 1.000001f / (float)a.group;
            // the last position that this row sees, and that all rows see
            uint32_t last, open;
            {
                const uint32_t base = ONE ? 0u : t * tile_rows, tok0 = st.tok0 + (ONE ? 0u : t * a.tokens_per_tile);
                open = (uint32_t)min((uint64_t)st.p0 + tok0, (uint64_t)0x7fffffffu);
                last = row < tile_rows && base + row < st.rows ? (uint32_t)min((uint64_t)st.p0 + TileRows{tok0, 0u, a.group, group_inv}.at(row).x, (uint64_t)0x7fffffffu) : open;
            }
            float m = -INFINITY, l = 0.f;
            uint32_t key0 = (st.k_begin + j_first) * kTileKeys;
            for (uint32_t j = j_first; j < n; j += j_step, key0 += j_step * kTileKeys) {
                ok = wait_warp(&b.s_full[t], turns & 1u, err);
                if (!ok) break;
                ++turns;
                fence_after();
                const uint32_t here = b.here[(number + j) & 7u];
                const bool masked = key0 + kTileKeys - 1u > open || here != 0xffu;   // some row does not see all of the tile
                float x[4][32], most[4];
                tmem_ld(at, x[0]);
                tmem_ld(at + 32u, x[1]);
                tmem_wait_ld(x[0]);
                tmem_wait_ld(x[1]);
                tmem_ld(at + 64u, x[2]);
                tmem_ld(at + 96u, x[3]);
                if (masked) {
                    const int nvis = last < key0 ? 0 : (int)min(last - key0 + 1u, kTileKeys);
                    tmem_wait_ld(x[2]);
                    tmem_wait_ld(x[3]);
#pragma unroll
                    for (int c = 0; c < 4; ++c)
#pragma unroll
                        for (int i = 0; i < 32; ++i)
                            x[c][i] = 32 * c + i < nvis && (here >> (2 * c + i / 16) & 1u) ? x[c][i] : -INFINITY;
                }
                auto largest = [&](int c) {
                    most[c] = max3(x[c][0], x[c][1], x[c][2]);
#pragma unroll
                    for (int i = 3; i < 31; i += 2) most[c] = max3(most[c], x[c][i], x[c][i + 1]);
                    most[c] = max3(most[c], x[c][31], x[c][31]);
                };
                largest(0);
                largest(1);
                tmem_wait_ld(x[2]);
                tmem_wait_ld(x[3]);
                largest(2);
                largest(3);
                const float top = max3(max3(most[0], most[1], most[2]), most[3], most[3]) * kScoreScale;
                const bool up = top > m + kLazy;
                if (__any_sync(0xffffffffu, up)) {
                    const float f = up ? (m == -INFINITY ? 0.f : ex2(m - top)) : 1.0f;
                    if (up) m = top;
                    l *= f;
                    if (j != j_first) {   // the products before these scores are done
#pragma unroll
                        for (uint32_t c = 0; c < 8u; ++c) {
                            float o[16];
                            uint32_t y[16];
                            tmem_ld(out_at + 128u * t + 16u * c, o);
                            tmem_wait_ld(o);
#pragma unroll
                            for (int i = 0; i < 16; ++i) y[i] = __float_as_uint(o[i] * f);
                            tmem_st(out_at + 128u * t + 16u * c, y);
                        }
                    }
                }
                // a row that has seen nothing yet has no maximum: its weights are 0
                const float off = m == -INFINITY ? 0.f : kUnit<BF> - m;
                const uint64_t f2 = pair(kScoreScale, kScoreScale), off2 = pair(off, off);
                uint64_t sum = 0ull;
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    uint32_t p[16];
#pragma unroll
                    for (int k = 0; k < 32; k += 2) {
                        float w0, w1;
                        unpair(fma2(pair(x[c][k], x[c][k + 1]), f2, off2), w0, w1);
                        w0 = ex2(w0);
                        w1 = ex2(w1);
                        sum = add2(sum, pair(w0, w1));
                        p[k / 2] = pack<BF>(w0, w1);
                    }
                    tmem_st(at + 16u * (uint32_t)c, p);
                    if ((c + 1) % (4 / kParts) == 0) {
                        tmem_wait_st();
                        fence_before();
                        __syncwarp();
                        if (lane == 0u) mbar_arrive(&b.p_full[t][c / (4 / kParts)]);
                    }
                }
                float s0, s1;
                unpair(sum, s0, s1);
                l += s0 + s1;
            }
            number += n;
            if (!ok) break;
            // ---- the end of the step: this thread's row, 128 columns; with one tile of rows, 64 of both groups' outputs
            const bool have[2] = {ONE || t == 0u, ONE ? n > 1u : t == 1u};
            float f[2] = {1.0f, 1.0f};
            if constexpr (ONE) {
                if (i) ok = wait_warp(&b.x_free[t], (i - 1u) & 1u, err);   // the other group has read the last one
                if (!ok) break;
                b.state[t][row] = make_float2(m, l);
                __syncwarp();
                if (lane == 0u) mbar_arrive(&b.x_full[t]);
                ok = wait_warp(&b.x_full[t ^ 1u], i & 1u, err);
                if (!ok) break;
                // in the same order in both groups
                const float2 s0 = b.state[0][row], s1 = b.state[1][row];
                __syncwarp();
                if (lane == 0u) mbar_arrive(&b.x_free[t ^ 1u]);
                m = fmaxf(s0.x, s1.x);
                f[0] = factor(s0, m);
                f[1] = factor(s1, m);
                l = f[0] * s0.y + f[1] * s1.y;
            }
#pragma unroll
            for (uint32_t g = 0; g < 2u; ++g)
                if (have[g]) {
                    ok = ok && wait_warp(&b.o_full[g], ends[g] & 1u, err);
                    ++ends[g];
                }
            if (!ok) break;
            fence_after();
            const uint32_t base = ONE ? 0u : t * tile_rows;
            const bool there = row < tile_rows && base + row < st.rows, again = st.again != 0u, whole = st.whole != 0u, bad = st.bad != 0u;
            const uint2 mine = TileRows{st.tok0 + (ONE ? 0u : t * a.tokens_per_tile), 0u, a.group, group_inv}.at(row);
            float fc = 0.f;
            if (again) {   // the steps before
                const float M = fmaxf(m, mc), g = factor(make_float2(m, l), M);
                fc = factor(make_float2(mc, lc), M);
                f[0] *= g;
                f[1] *= g;
                l = fmaf(g, l, fc * lc);
                m = M;
            }
            mc = m;
            lc = l;
            float *const record = record_of(a, st.record, kRecordRows<ONE>), *const rec = record + (base + row) * kDim;
            const float inv = whole ? (l == 0.f ? 0.f : 1.0f / l) : 1.0f;
            uint16_t *const out = a.out + ((size_t)st.s * a.r.tokens + mine.x) * a.ldo + (size_t)(st.h * a.group + mine.y) * kDim;
            constexpr uint32_t kColumns = ONE ? kDim / 2u : kDim;
            const uint32_t c0 = ONE ? t * kColumns : 0u;
            // some columns' outputs, times their factors, into o; RARE: with what was taken out of V, and the steps before. A factor of 0
            // is multiplied by, too: infinities that the row sees stay to be seen.
            auto outputs = [&](auto &o, uint32_t c, auto rare) {
                constexpr bool RARE = decltype(rare)::value;
                constexpr int N = sizeof(o) / sizeof(o[0]);
                tmem_ld(out_at + (ONE ? 0u : 128u * t) + c, o);
                tmem_wait_ld(o);
                if (ONE || RARE)
#pragma unroll
                    for (int k = 0; k < N; ++k) o[k] *= f[ONE ? 0 : t];
                if (ONE && have[1]) {
                    float y[N];
                    tmem_ld(out_at + 128u + c, y);
                    tmem_wait_ld(y);
#pragma unroll
                    for (int k = 0; k < N; ++k) o[k] = fmaf(f[1], y[k], o[k]);
                }
                if (!RARE || !there) return;
                if (bad) {   // what was taken out of V, to the rows that see it
                    const uint32_t page_log2 = a.c.page_log2;
                    const int32_t *const entries = a.c.table + (size_t)st.s * a.c.max_pages;
                    const uint64_t k1 = min(min((uint64_t)last + 1u, (uint64_t)(st.k_begin + n) * kTileKeys), (uint64_t)a.c.limit);
                    for (uint64_t p = max((uint64_t)st.k_begin * kTileKeys, (uint64_t)st.p0 + st.tok0 + 1u); p < k1; ++p) {
                        const uint32_t e = (uint32_t)__ldcg(entries + (p >> page_log2));
                        if (e >= a.c.pages) continue;
                        const uint16_t *v = a.c.v + (((((size_t)a.layer * a.c.pages + e) * a.c.kv_heads + st.h) << page_log2) + (p & ((1u << page_log2) - 1u))) * kDim + c;
#pragma unroll
                        for (int k = 0; k < N; ++k) {
                            const float y = unpack1<BF>(__ldcg(v + k));
                            if (!(y - y == 0.f)) o[k] += y;
                        }
                    }
                }
                if (again)
#pragma unroll
                    for (int k = 0; k < N; ++k) o[k] = fmaf(fc, __ldcg(rec + c + k), o[k]);
            };
            auto store = [&](const auto &o, uint32_t c) {
                constexpr int N = sizeof(o) / sizeof(o[0]);
                if (!there) return;
                if (whole) {
#pragma unroll
                    for (int k = 0; k < N; k += 16) {
                        uint32_t y[8];
#pragma unroll
                        for (int q = 0; q < 8; ++q) y[q] = pack<BF>(o[k + 2 * q] * inv, o[k + 2 * q + 1] * inv);
                        uint16_t *to = out + c + k;
                        if (a.wide) {
                            store32(to, y);
                        } else {
                            reinterpret_cast<uint4 *>(to)[0] = make_uint4(y[0], y[1], y[2], y[3]);
                            reinterpret_cast<uint4 *>(to)[1] = make_uint4(y[4], y[5], y[6], y[7]);
                        }
                    }
                } else {
#pragma unroll
                    for (int k = 0; k < N; k += 8) {
                        uint32_t y[8];
#pragma unroll
                        for (int q = 0; q < 8; ++q) y[q] = __float_as_uint(o[k + q]);
                        store32(rec + c + k, y);
                    }
                }
            };
            if (bad || again) {
#pragma unroll 1
                for (uint32_t c = c0; c < c0 + kColumns; c += 16u) {
                    float o[16];
                    outputs(o, c, std::true_type{});
                    store(o, c);
                }
            } else {
#pragma unroll 1
                for (uint32_t c = c0; c < c0 + kColumns; c += 32u) {
                    float o[32];
                    outputs(o, c, std::false_type{});
                    store(o, c);
                }
            }
            fence_before();
            __syncwarp();
            if (lane == 0u)
                for (uint32_t g = 0; g < 2u; ++g)
                    if (have[g]) mbar_arrive(&b.o_free[g]);
            if (!whole && there && (!ONE || t == 0u)) reinterpret_cast<float2 *>(record + kRecordRows<ONE> * kDim)[base + row] = make_float2(m, l);
            done_with(i);
        }
        leave();
    }
}

// Lets the kernel take its shared memory; refuses a build of it whose launch has fewer registers than the warpgroups then
// ask for, as that would wait for good.
template <auto KERNEL>
cudaError_t prepare(int dev, size_t smem)
{
    static std::atomic<int> registers{0};
    int n = registers.load(std::memory_order_relaxed);
    if (!n) {
        cudaFuncAttributes at{};
        const cudaError_t e = cudaFuncGetAttributes(&at, KERNEL);
        if (e != cudaSuccess) return e;
        registers.store(n = at.numRegs, std::memory_order_relaxed);
    }
    if ((uint32_t)n * 3u < 2u * kSoftmaxRegs + kOtherRegs) return cudaErrorLaunchOutOfResources;
    return k8::allow<KERNEL>(dev, (int)smem);
}

template <bool BF, bool ONE>
cudaError_t launch_prompt_of(const PromptArgs &p, int dev, int sms, cudaStream_t stream)
{
    const cudaError_t e = prepare<prompt_kernel<BF, ONE>>(dev, kSmem<ONE>);
    if (e != cudaSuccess) return e;
    return k8::launch(prompt_kernel<BF, ONE>, dim3(std::min((uint32_t)sms, kMaxCtas)), kThreads, kSmem<ONE>, 1, p, sms, stream);
}

}  // namespace

// The form for many rows, `tiles` (1 or 2) tiles of 128 / group whole tokens per unit; maps: see PromptArgs
cudaError_t launch_prompt(const AttnArgs &a, const CUtensorMap &kmap, const CUtensorMap &vmap, const CUtensorMap &qmap, bool bf, uint32_t tiles, int dev,
                          int sms, cudaStream_t stream)
{
    PromptArgs p{};
    static_cast<AttnArgs &>(p) = a;
    p.kmap = kmap;
    p.vmap = vmap;
    p.qmap = qmap;
    p.tokens_per_tile = kTileRows / a.group;
    p.by_tile = divisor(tiles * p.tokens_per_tile * a.group);
    p.keep = lanes_keep(a, tiles * p.tokens_per_tile * a.group, kTileKeys, kExtra);
    p.wide = ((reinterpret_cast<uintptr_t>(a.out) | a.ldo * 2) & 31u) == 0;
    const cudaError_t e = tiles == 1 ? (bf ? launch_prompt_of<true, true>(p, dev, sms, stream) : launch_prompt_of<false, true>(p, dev, sms, stream))
                                     : (bf ? launch_prompt_of<true, false>(p, dev, sms, stream) : launch_prompt_of<false, false>(p, dev, sms, stream));
    if (e != cudaSuccess) return e;
    const uint32_t ctas = std::min((uint32_t)sms, kMaxCtas), per = tiles * p.tokens_per_tile;
    const uint64_t units = (uint64_t)a.c.nseq * a.c.kv_heads * ((a.r.tokens + per - 1) / per);
    if (always_whole(p, units, ctas, kTileKeys, kWorth)) return cudaSuccess;
    return launch_merge(a, bf, tiles * kTileRows, ctas, sms, stream);
}

}  // namespace paged
}  // namespace atlas
