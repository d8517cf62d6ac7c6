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
//   8     copies; 9 issues the MMAs: P V of a tile of keys, then the next keys'
//         scores of the same rows, so that one tile's softmax runs under the other's
//         MMAs;
//   10-11 of a tile of keys that not all rows see, take values out of V that are
//         not finite: a weight of 0 would not hide them. The softmax threads
//         add them to the rows that do see them.
// With one tile of rows, both softmax groups have it and take turns at the keys,
// each with an output and a state of its own, joined at the end.
//
// Tensor cores truncate their sums: 2^-24 of the output per MMA of 16 keys at
// most, so 256 tiles of keys (2048 MMAs, 2^-13) are summed in tensor memory, and
// longer pieces in steps of that, joined in fp32.
// Tensor memory: 2 x 128 columns of scores / weights, 2 x 128 of output.
// Every wait is bounded; after a timeout the CTA's rows are NaN.
#include <algorithm>
#include <atomic>
#include <cfloat>
#include <cmath>
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
constexpr uint32_t kSlots = 4, kWorth = 4, kCross = 2;        // tiles of keys: what joining partial sums takes, and passing to another unit
constexpr float kLazy = 8.0f;
// Weights are 2^(score - maximum + kUnit): binary16 keeps 24 bits below the largest; bfloat16 has fp32's range, and small
// weights leave the sums of large values room
template <bool BF>
constexpr float kUnit = BF ? -24.0f : 6.0f;

struct PromptArgs : AttnArgs {
    CUtensorMap kmap, vmap;      // [2][rows of the pool][64] each
    CUtensorMap qmap;            // [2][token][head][64]
    uint32_t tokens_per_tile;
    Divisor by_tile;             // by a unit's rows
    uint32_t wide;               // output rows lie on 32-byte boundaries
};

struct Bars {
    uint64_t s_full[2], p_full[2][2], o_full[2], o_free[2], full[kMaxStages], free[kMaxStages], checked[kMaxStages], q_full, q_free, fin;
    uint32_t tmem, status;
    uint32_t bad[4];                               // the step in which a value was taken out, at its number % 4
    float2 state[2][kTileRows];                    // one tile of rows: the groups' maxima and sums
};

template <bool ONE>
constexpr uint32_t kStages = ONE ? 6u : 5u;
template <bool ONE>
constexpr size_t kSmem = (ONE ? 1 : 2) * kTile + kStages<ONE> * kTile + sizeof(Bars);
static_assert(kSmem<true> <= k8::kMaxSmem && kSmem<false> <= k8::kMaxSmem, "the tiles exceed a CTA's shared memory");
static_assert(sizeof(PieceSmem) <= 2 * kTile, "find_piece works in the stages' place");

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
    Bars &b = *reinterpret_cast<Bars *>(kv + STAGES * kTile);
    volatile uint32_t *const err = &b.status;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
    if (threadIdx.x == 0) {
        for (int t = 0; t < 2; ++t) {
            mbar_init(&b.s_full[t], 1u);
            mbar_init(&b.p_full[t][0], 4u);
            mbar_init(&b.p_full[t][1], 4u);
            mbar_init(&b.o_full[t], 1u);
            mbar_init(&b.o_free[t], ONE ? 8u : 4u);
        }
        for (uint32_t i = 0; i < STAGES; ++i) {
            mbar_init(&b.full[i], 1u);
            mbar_init(&b.free[i], 1u);
            mbar_init(&b.checked[i], kCheckers);
        }
        mbar_init(&b.q_full, 1u);
        mbar_init(&b.q_free, 1u);
        mbar_init(&b.fin, 1u);
        b.status = kStatusOk;
        for (int i = 0; i < 4; ++i) b.bad[i] = ~0u;
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
    const Cut<kTileKeys> cut{a, (ONE ? 1u : 2u) * tile_rows, a.by_tile};
    const Piece piece = find_piece<kTileKeys, kThreads / 32u, kSlots>(cut, *reinterpret_cast<PieceSmem *>(kv), 2u, kWorth, kCross);
    fence_before();
    fence_async();
    __syncthreads();
    fence_after();
    const uint32_t tmem = b.tmem;   // scores / weights of group t: column 128 t; output: 256 + 128 t
    Walk<kTileKeys, kMostTiles> w(cut, piece);

    // The end of a CTA, for every warp in the branch of its registers
    auto leave = [&]() {
        fence_before();
        __syncthreads();
        if (warp == kMmaWarp) {
            fence_after();
            asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
        }
    };
    // tiles of rows that the unit has
    auto tiles_of = [&](uint32_t rows) { return !ONE && rows > tile_rows ? 2u : 1u; };
    if (warp >= kLoadWarp) {
    fewer_registers<kOtherRegs>();   // the whole warpgroup
    if (warp == kLoadWarp) {
        // ---------------------------------------------------------- copies --
        Ring<STAGES> ring;
        uint32_t used = 0u, steps = 0u;            // tiles copied so far
        bool ok = true;
        const uint32_t page_log2 = a.c.page_log2, per = 7u - page_log2;   // log2 of pages per tile of keys
        const uint32_t of = lane >> 1, half = lane & 1u;                   // this lane's page of a tile and half of its dimensions
        const bool mine = of < (1u << per);
        const uint32_t nowhere = (a.c.layers * a.c.pages * a.c.kv_heads) << page_log2;   // behind the pool's end: zeros
        for (; ok && w.more(); w.next(), ++steps) {
            const uint32_t s = w.p.s, h = w.p.h, row0 = w.row0(), rows = w.rows(), tiles = tiles_of(rows);
            const uint32_t seen = (uint32_t)min((uint64_t)w.q.p0 + divide(row0 + rows - 1u, a.by_group) + 1u, (uint64_t)a.c.limit);
            const int32_t *const entries = a.c.table + (size_t)s * a.c.max_pages;
            // where this lane's page of tile j begins
            auto page_row = [&](uint32_t j) {
                const uint32_t e0 = (j << per) + of;
                const uint32_t e = mine && j < w.k_end && (uint64_t)e0 << page_log2 < seen ? (uint32_t)__ldcg(entries + e0) : ~0u;
                return e < a.c.pages ? ((a.layer * a.c.pages + e) * a.c.kv_heads + h) << page_log2 : nowhere;
            };
            if (steps) ok = wait_warp(&b.q_free, (steps - 1u) & 1u, err);
            if (!ok) break;
            if (lane == 0u) {
                mbar_arrive_expect_tx(&b.q_full, tiles * tile_rows * 256u);
                const uint32_t token = s * a.r.tokens + divide(row0, a.by_group);
                for (uint32_t t = 0; t < tiles; ++t)
                    for (uint32_t hf = 0; hf < 2u; ++hf)
                        load_queries(smem_addr(qs + t * kTile + hf * kHalf), &a.qmap, h * a.group, token + t * a.tokens_per_tile, hf, &b.q_full);
            }
            auto copy = [&](const CUtensorMap *map, uint32_t row) {
                if (used >= STAGES) ok = wait_warp(&b.free[ring.slot], ring.phase ^ 1u, err);
                if (!ok) return;
                if (lane == 0u) mbar_arrive_expect_tx(&b.full[ring.slot], kTile);
                __syncwarp();
                if (mine) load_box(smem_addr(kv + ring.slot * kTile + half * kHalf) + ((of << page_log2) << 7), map, row, half, &b.full[ring.slot]);
                ring.next();
                ++used;
            };
            // in the order in which the MMAs take them: with one tile of rows, a tile of K more before V
            uint32_t at = page_row(w.k_begin), next = page_row(w.k_begin + 1u);
            if (ONE) {
                copy(&a.kmap, at);
                for (uint32_t j = w.k_begin; ok && j < w.k_end; ++j) {
                    const uint32_t after = page_row(j + 2u);
                    if (j + 1u < w.k_end) copy(&a.kmap, next);
                    if (ok) copy(&a.vmap, at);
                    at = next;
                    next = after;
                }
            } else {
                for (uint32_t j = w.k_begin; ok && j < w.k_end; ++j) {
                    const uint32_t after = page_row(j + 2u);
                    copy(&a.kmap, at);
                    if (ok) copy(&a.vmap, at);
                    at = next;
                    next = after;
                }
            }
        }
        if (!ok) {   // nothing of this CTA is left in flight: the last copies are waited for
            const uint64_t t0 = global_ns();
            if (steps)
                while (!mbar_try_wait(&b.q_full, (steps - 1u) & 1u) && global_ns() - t0 < kWaitLimitNs) {
                }
            for (uint32_t i = 0; i < min(used, STAGES); ++i) {
                const uint32_t n = used - 1u - i, slot = n % STAGES;
                while (!mbar_try_wait(&b.full[slot], n / STAGES & 1u) && global_ns() - t0 < kWaitLimitNs) {
                }
            }
        }
        leave();
    } else if (warp == kMmaWarp) {
        // ------------------------------------------------------------- MMA --
        const bool leader = elected();
        Ring<STAGES> ring;
        uint32_t steps = 0u, turns[2] = {0u, 0u}, ends[2] = {0u, 0u};   // of a group: tiles of keys, and steps, so far
        uint32_t check_phase = 0u;                 // bit i: of slot i
        bool ok = true;
        const uint64_t qd = operand(smem_addr(qs)), kd = operand(smem_addr(kv)), vd = operand_across(smem_addr(kv), kHalf);
        for (; ok && w.more(); w.next(), ++steps) {
            const uint32_t tiles = tiles_of(w.rows()), n = w.k_end - w.k_begin;
            const uint64_t open = (uint64_t)w.q.p0 + divide(w.row0(), a.by_group);   // every row sees the positions up to it
            if (leader) {
                ok = mbar_wait(&b.q_full, steps & 1u, err);
                // scores of the keys in ring slot `slot` by tile of rows qt, into group t's columns
                auto scores = [&](uint32_t t, uint32_t qt, uint32_t slot) {
                    const uint64_t q = qd + (uint64_t)(qt * (kTile >> 4)), k = kd + (uint64_t)(slot * (kTile >> 4));
#pragma unroll
                    for (uint32_t st = 0; st < 8u; ++st) {
                        const uint32_t off = (st >> 2) * (kHalf >> 4) + (st & 3u) * 2u;
                        mma_ss(tmem + 128u * t, q + off, k + off, kInstr<BF, false>, st != 0u);
                    }
                    commit(&b.s_full[t]);
                };
                // group t's weights times the values in slot `slot`
                auto output = [&](uint32_t t, uint32_t slot, bool begin) {
                    const uint64_t v = vd + (uint64_t)(slot * (kTile >> 4));
#pragma unroll
                    for (uint32_t hf = 0; hf < 2u; ++hf) {
                        if (!(ok = ok && mbar_wait(&b.p_full[t][hf], turns[t] & 1u, err))) return;
                        fence_after();
#pragma unroll
                        for (uint32_t st = 4u * hf; st < 4u * hf + 4u; ++st)   // 16 keys: 8 columns of P, 2048 bytes of V
                            mma_ts(tmem + 256u + 128u * t, tmem + 128u * t + 8u * st, v + st * 128u, kInstr<BF, true>, !begin || st != 0u);
                    }
                    ++turns[t];
                };
                // the tile of V of keys j is there, and looked through if need be
                auto values = [&](uint32_t j, const Ring<STAGES> &r) {
                    ok = ok && mbar_wait(&b.full[r.slot], r.phase, err);
                    if ((uint64_t)(j + 1u) * kTileKeys > open + 1u) {
                        ok = ok && mbar_wait(&b.checked[r.slot], check_phase >> r.slot & 1u, err);
                        check_phase ^= 1u << r.slot;
                    }
                };
                auto keys = [&](const Ring<STAGES> &r) { ok = ok && mbar_wait(&b.full[r.slot], r.phase, err); };
                // a group's output may be overwritten
                auto fresh = [&](uint32_t t) {
                    if (ends[t]) ok = ok && mbar_wait(&b.o_free[t], (ends[t] - 1u) & 1u, err);
                };
                if (ONE) {   // the groups take turns at the keys
                    const uint32_t groups = min(n, 2u);
                    Ring<STAGES> rk = ring;
                    keys(rk);
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
                        values(w.k_begin + j, rk);
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
                    for (uint32_t t = 0; t < groups; ++t) ++ends[t];
                    ring = rk;
                } else {
                    Ring<STAGES> rk = ring;
                    keys(rk);
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
                            if (t == 0u) values(w.k_begin + j, rv);
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
                    ring = rk;
                }
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
        // ---------------------------------------------------------- checks --
        // Every copy is waited for, in order: a barrier tells a phase only from the one before.
        if (threadIdx.x == kCheckWarp * 32u) reinterpret_cast<Part *>(a.parts)[blockIdx.x] = w.part();
        Ring<STAGES> ring;
        uint32_t steps = 0u;
        bool ok = true;
        for (; ok && w.more(); w.next(), ++steps) {
            const uint32_t n = w.k_end - w.k_begin;
            const uint64_t open = (uint64_t)w.q.p0 + divide(w.row0(), a.by_group);
            auto pass = [&]() {
                ok = ok && wait_warp(&b.full[ring.slot], ring.phase, err);
                ring.next();
            };
            if (ONE) pass();
            for (uint32_t j = 0; ok && j < n; ++j) {
                if (ONE ? j + 1u < n : true) pass();
                const uint64_t key0 = (uint64_t)(w.k_begin + j) * kTileKeys;
                ok = ok && wait_warp(&b.full[ring.slot], ring.phase, err);
                if (!ok) break;
                if (key0 + kTileKeys > open + 1u) {
                    // keys from `from` on are not seen by all rows; a thread has 16 bytes of a key's row
                    const uint32_t from = open >= key0 ? (uint32_t)(open - key0) + 1u : 0u;
                    uint8_t *const v = kv + ring.slot * kTile;
                    bool found = false;
                    for (uint32_t x = from * 8u + (threadIdx.x - kCheckWarp * 32u); x < kTileKeys * 8u; x += 32u * kCheckers)
#pragma unroll
                        for (uint32_t hf = 0; hf < 2u; ++hf) {
                            uint4 *const p = reinterpret_cast<uint4 *>(v + hf * kHalf) + x;
                            uint4 y = *p;
                            const uint4 bad = make_uint4(nonfinite2<BF>(y.x), nonfinite2<BF>(y.y), nonfinite2<BF>(y.z), nonfinite2<BF>(y.w));
                            if (bad.x | bad.y | bad.z | bad.w) {
                                *p = make_uint4(y.x & ~bad.x, y.y & ~bad.y, y.z & ~bad.z, y.w & ~bad.w);
                                found = true;
                            }
                        }
                    if (found) b.bad[steps & 3u] = steps;
                    fence_async();
                    __syncwarp();
                    if (lane == 0u) mbar_arrive(&b.checked[ring.slot]);
                }
                ring.next();
            }
        }
        leave();
    }
    } else {
        more_registers<kSoftmaxRegs>();
        // --------------------------------------------------------- softmax --
        // A warp whose wait ran out goes on to the units' ends without touching tensor memory.
        const uint32_t t = warp >> 2, quarter = warp & 3u, row = quarter * 32u + lane;
        const uint32_t at = tmem + ((quarter * 32u) << 16) + 128u * t, out_at = tmem + ((quarter * 32u) << 16) + 256u;
        const float group_inv = 1.000001f / (float)a.group;
        const uint32_t page_log2 = a.c.page_log2;
        uint32_t steps = 0u, turns = 0u, ends[2] = {0u, 0u};
        bool ok = true;
        for (; w.more(); w.next(), ++steps) {
            const uint32_t s = w.p.s, h = w.p.h, row0 = w.row0(), rows = w.rows(), tiles = tiles_of(rows), n = w.k_end - w.k_begin;
            if (!ONE && t >= tiles) continue;
            const uint32_t base = ONE ? 0u : t * tile_rows, tok0 = divide(row0, a.by_group) + (ONE ? 0u : t * a.tokens_per_tile);
            const uint2 mine = TileRows{tok0, 0u, a.group, group_inv}.at(row);
            const bool there = row < tile_rows && base + row < rows;
            const uint64_t p0 = w.q.p0;
            const uint32_t open = (uint32_t)min(p0 + tok0, (uint64_t)0x7fffffffu);
            const uint32_t last = there ? (uint32_t)min(p0 + mine.x, (uint64_t)0x7fffffffu) : open;
            const int32_t *const entries = a.c.table + (size_t)s * a.c.max_pages;
            // bit i: the 16 positions from 16 i on of tile j have a page
            auto pages_of = [&](uint32_t j) {
                const uint32_t p = j * kTileKeys + 16u * (lane & 7u);
                return p < a.c.limit && (uint32_t)__ldcg(entries + (p >> page_log2)) < a.c.pages;
            };
            constexpr uint32_t j_step = ONE ? 2u : 1u;
            const uint32_t j_first = ONE ? t : 0u;
            float m = -INFINITY, l = 0.f;
            bool next = j_first < n && pages_of(w.k_begin + j_first);
            for (uint32_t j = j_first; j < n; j += j_step) {
                const uint32_t here = __ballot_sync(0xffffffffu, next) & 0xffu;
                if (j + j_step < n) next = pages_of(w.k_begin + j + j_step);
                const uint32_t key0 = (w.k_begin + j) * kTileKeys;
                const bool masked = key0 + kTileKeys - 1u > open || here != 0xffu;   // some row does not see all of the tile
                ok = ok && wait_warp(&b.s_full[t], turns & 1u, err);
                if (!ok) break;
                ++turns;
                fence_after();
                float x[4][32];
#pragma unroll
                for (int c = 0; c < 4; ++c) tmem_ld(at + 32u * (uint32_t)c, x[c]);
#pragma unroll
                for (int c = 0; c < 4; ++c) tmem_wait_ld(x[c]);
                if (masked) {
                    const int nvis = last < key0 ? 0 : (int)min(last - key0 + 1u, kTileKeys);
#pragma unroll
                    for (int c = 0; c < 4; ++c)
#pragma unroll
                        for (int i = 0; i < 32; ++i)
                            x[c][i] = 32 * c + i < nvis && (here >> (2 * c + i / 16) & 1u) ? x[c][i] : -INFINITY;
                }
                float most[4];
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    most[c] = fmaxf(x[c][0], x[c][1]);
#pragma unroll
                    for (int i = 2; i < 32; i += 2) most[c] = max3(most[c], x[c][i], x[c][i + 1]);
                }
                const float top = fmaxf(max3(most[0], most[1], most[2]), most[3]) * kScoreScale;
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
                for (int hf = 0; hf < 2; ++hf) {
                    uint32_t p[32];
#pragma unroll
                    for (int i = 0; i < 64; i += 2) {
                        const float *v = &x[2 * hf + i / 32][i % 32];
                        float w0, w1;
                        unpair(fma2(pair(v[0], v[1]), f2, off2), w0, w1);
                        w0 = ex2(w0);
                        w1 = ex2(w1);
                        sum = add2(sum, pair(w0, w1));
                        p[i / 2] = pack<BF>(w0, w1);
                    }
                    tmem_st(at + 32u * (uint32_t)hf, p);
                    tmem_wait_st();
                    fence_before();
                    __syncwarp();
                    if (lane == 0u) mbar_arrive(&b.p_full[t][hf]);
                }
                float s0, s1;
                unpair(sum, s0, s1);
                l += s0 + s1;
            }
            // ---- the end of the step: this thread's row, 128 columns; with one tile of rows, 64 of both groups' outputs
            const bool have[2] = {ONE || t == 0u, ONE ? n > 1u : t == 1u};
            float f[2] = {1.0f, 1.0f};
            if (ONE) {
                b.state[t][row] = make_float2(m, l);
                meet(1u, 256u);
                const float2 other = b.state[t ^ 1u][row];
                meet(1u, 256u);
                const float M = fmaxf(m, other.x);
                const float mine_f = m == -INFINITY ? (l == 0.f ? 0.f : 1.f) : ex2(m - M), their_f = other.x == -INFINITY ? (other.y == 0.f ? 0.f : 1.f) : ex2(other.x - M);
                f[t] = mine_f;
                f[t ^ 1u] = their_f;
                l = t == 0u ? l * mine_f + other.y * their_f : other.y * their_f + l * mine_f;
                m = M;
            }
#pragma unroll
            for (uint32_t g = 0; g < 2u; ++g)
                if (have[g]) {
                    ok = ok && wait_warp(&b.o_full[g], ends[g] & 1u, err);
                    ++ends[g];
                }
            fence_after();
            float *const rec = record_of(a, w.record(), ONE ? kTileRows : 2u * kTileRows) + (base + row) * kDim;
            float2 *const rec_ml = reinterpret_cast<float2 *>(record_of(a, w.record(), ONE ? kTileRows : 2u * kTileRows) + (ONE ? 1u : 2u) * kTileRows * kDim) + base + row;
            const bool leaves = w.leaves(), whole = leaves && w.head && w.tail;
            float fc = 0.f;
            if (w.again && there) {   // the steps before
                const float2 old = __ldcg(rec_ml);
                const float M = fmaxf(m, old.x), g = m == -INFINITY ? (l == 0.f ? 0.f : 1.f) : ex2(m - M);
                fc = old.x == -INFINITY ? (old.y == 0.f ? 0.f : 1.f) : ex2(old.x - M);
                f[0] *= g;
                f[1] *= g;
                l = fmaf(g, l, fc * old.y);
                m = M;
            }
            if (ONE && w.again) meet(1u, 256u);   // both groups have read the state
            if (!ok) l = __int_as_float(0x7fffffff);
            const float inv = whole ? (l == 0.f ? 0.f : 1.0f / l) : 1.0f;
            const uint32_t bad = b.bad[steps & 3u];
            uint16_t *const out = a.out + ((size_t)s * a.r.tokens + mine.x) * a.ldo + (size_t)(h * a.group + mine.y) * kDim;
            constexpr uint32_t kColumns = ONE ? kDim / 2u : kDim;
#pragma unroll 1
            for (uint32_t c = ONE ? t * kColumns : 0u; c < (ONE ? t * kColumns : 0u) + kColumns; c += 16u) {
                float o[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) o[i] = 0.f;
                if (ok) {
#pragma unroll
                    for (uint32_t g = 0; g < 2u; ++g)
                        if (have[g]) {
                            float y[16];
                            tmem_ld(out_at + 128u * g + c, y);
                            tmem_wait_ld(y);
#pragma unroll
                            for (int i = 0; i < 16; ++i) o[i] = f[g] == 0.f ? o[i] : fmaf(f[g], y[i], o[i]);
                        }
                }
                if (!there) continue;
                if (bad == steps) {   // what was taken out of V, to the rows that see it
                    const uint64_t k1 = min((uint64_t)last + 1u, (uint64_t)w.k_end * kTileKeys);
                    for (uint64_t p = max((uint64_t)w.k_begin * kTileKeys, (uint64_t)p0 + divide(row0, a.by_group) + 1u); p < min(k1, (uint64_t)a.c.limit); ++p) {
                        const uint32_t e = (uint32_t)__ldcg(entries + (p >> page_log2));
                        if (e >= a.c.pages) continue;
                        const uint16_t *v = a.c.v + (((((size_t)a.layer * a.c.pages + e) * a.c.kv_heads + h) << page_log2) + (p & ((1u << page_log2) - 1u))) * kDim + c;
                        for (int i = 0; i < 16; ++i) {
                            const float y = unpack1<BF>(__ldcg(v + i));
                            if (!(y - y == 0.f)) o[i] += y;
                        }
                    }
                }
                if (w.again) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) o[i] = fmaf(fc, __ldcg(rec + c + i), o[i]);
                }
                if (whole) {
                    uint32_t y[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) y[i] = pack<BF>(o[2 * i] * inv, o[2 * i + 1] * inv);
                    if (a.wide) {
                        store32(out + c, y);
                    } else {
                        reinterpret_cast<uint4 *>(out + c)[0] = make_uint4(y[0], y[1], y[2], y[3]);
                        reinterpret_cast<uint4 *>(out + c)[1] = make_uint4(y[4], y[5], y[6], y[7]);
                    }
                } else {
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        uint32_t y[8];
#pragma unroll
                        for (int i = 0; i < 8; ++i) y[i] = __float_as_uint(o[8 * k + i]);
                        store32(rec + c + 8 * k, y);
                    }
                }
            }
            fence_before();
            __syncwarp();
            if (lane == 0u)
                for (uint32_t g = 0; g < 2u; ++g)
                    if (have[g]) mbar_arrive(&b.o_free[g]);
            if (!whole && there && (!ONE || t == 0u)) *rec_ml = make_float2(m, l);
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
    p.keep = lanes_keep(a, tiles * p.tokens_per_tile * a.group, kTileKeys);
    p.wide = ((reinterpret_cast<uintptr_t>(a.out) | a.ldo * 2) & 31u) == 0;
    const cudaError_t e = tiles == 1 ? (bf ? launch_prompt_of<true, true>(p, dev, sms, stream) : launch_prompt_of<false, true>(p, dev, sms, stream))
                                     : (bf ? launch_prompt_of<true, false>(p, dev, sms, stream) : launch_prompt_of<false, false>(p, dev, sms, stream));
    if (e != cudaSuccess) return e;
    const uint32_t ctas = std::min((uint32_t)sms, kMaxCtas), per = tiles * p.tokens_per_tile;
    const uint64_t units = (uint64_t)a.c.nseq * a.c.kv_heads * ((a.r.tokens + per - 1) / per);
    if (always_whole(p, units, ctas, kTileKeys, kWorth, kSlots)) return cudaSuccess;
    return launch_merge(a, bf, tiles * kTileRows, ctas, sms, stream);
}

}  // namespace paged
}  // namespace atlas
