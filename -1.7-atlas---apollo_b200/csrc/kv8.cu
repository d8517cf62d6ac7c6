// 8-bit KV cache (sm_100a): quantising append, read-back, and attention over
// the cache for single tokens, dense or over selected blocks. The prompt form
// of the attention is in kv8_prompt.cu.
//
// The reference keeps K and V in fp32 (src/brain_runtime.c:2019-2020) and
// attends per token (gqa_single_token, :1407-1528); this cache takes a quarter
// of the bytes, and the attention over it keeps fp32-level accuracy for the
// values that the codes stand for.
#include <cfloat>
#include <cmath>
#include <algorithm>
#include <atomic>
#include <cuda.h>
#include "../../include/atlas_cuda.h"
#include "common.cuh"
#include "kv8.cuh"

namespace atlas {

int api_fail(int code, const char *fmt, ...);
int api_device(int device, int *sms);

namespace k8 {

// kv8_prompt.cu
PromptCut prompt_cut(const AttnArgs &a, int dev, int sms);
cudaError_t launch_prompt(AttnArgs a, const PromptCut &cut, int dev, int sms, cudaStream_t stream);

namespace {

// --------------------------------------------------------------- append ----

struct AppendArgs {
    Cache c;
    Rows r;
    const float *k, *v;   // [seq][tokens][kv_heads][128], ld floats between tokens
    uint64_t ld;
    uint32_t early;
};

// Nearest integers to x / s (ties to even), exactly, for |x| <= 127.5 s, as the
// low bytes of the results. x * inv + 2^23 + 2^22, rounded once, has the integer
// nearest to x * inv in its low bits; the rounded reciprocal inv = 1 / s puts
// x * inv off by at most 127 * 2^-24 < 2^-17, so that decides everything but
// quotients within 2^-13 of a tie. If one of the four is, they are divided in 64
// bits (two 24-bit values whose quotient is no tie differ from it by 2^-25 or
// more). `slow`: s too small for the reciprocal.
__device__ __forceinline__ void quantise(const float4 &x, float s, float inv, bool slow, uint32_t (&q)[4])
{
    const float v[4] = {x.x, x.y, x.z, x.w};
    constexpr float kInt = 12582912.0f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float u = fmaf(v[j], inv, kInt);
        slow |= fabsf(fmaf(v[j], inv, kInt - u)) > 0.5f - 1.220703125e-4f;
        q[j] = __float_as_uint(u);
    }
    if (slow)
#pragma unroll
        for (int j = 0; j < 4; ++j)
            q[j] = (uint32_t)(int)fmin(fmax(rint((double)v[j] / (double)s), -127.0), 127.0) + 0x4B400000u;
}

// One CTA per (touched block, K or V of a KV head, sequence). Warp w holds
// rows w, w + 8, ... of the block in registers (lane = 4 dimensions), new ones
// as values and earlier ones as codes, so the rows are read once: maximum,
// then codes. scale = max(scale so far, max|new| / 127); rows that were in the
// block before are rounded again where the scale grew. A block that a
// non-finite value joins gets a NaN scale.
// 4 bytes read and 1 written per value: 8192 tokens of 8 heads, K and V, take 18
// to 20 us (84 MB, 4.1 to 4.6 TB/s; 12.9 at the copy rate). Under ncu DRAM is
// busy for 36 % and issue for 66 %, and most stalls wait for loads: a CTA loads,
// converts and stores once, 3.5 waves of them, with nothing of its own to overlap.
template <int B>
__global__ void __launch_bounds__(256) append_kernel(const __grid_constant__ AppendArgs a)
{
    constexpr int kRows = B / 8;
    __shared__ uint32_t s_max[8];
    __shared__ alignas(16) uint32_t s_sum[8][kDim];
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
    wait_predecessor(a.early);
    const uint32_t s = blockIdx.z, h = blockIdx.y >> 1, is_v = blockIdx.y & 1u;
    const uint64_t p0 = __ldcg(a.r.pos0 + s), end = min(p0 + row_count(a.r, s), (uint64_t)a.c.max_context);
    const uint64_t blk = p0 / B + blockIdx.x, b0 = blk * B;
    if (max(p0, b0) >= end) return;                                   // no new row in this block
    const uint32_t lo = b0 < p0 ? (uint32_t)(p0 - b0) : 0u;          // rows [0, lo) were there before
    const uint32_t hi = (uint32_t)min((uint64_t)B, end - b0);        // rows [lo, hi) are new
    const size_t head = (size_t)s * a.c.kv_heads + h;
    int8_t *code = (is_v ? a.c.v : a.c.k) + (head * a.c.max_context + b0) * kDim;
    float *sp = (is_v ? a.c.v_scale : a.c.k_scale) + head * a.c.n_blocks + blk;
    const float *src = (is_v ? a.v : a.k) + (size_t)s * a.r.tokens * a.ld + (size_t)h * kDim;

    float4 x[kRows];   // a row that was there before: its 4 codes in the bits of .x
    uint32_t mx = 0u;
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
        const uint32_t r = warp + 8u * (uint32_t)i;
        x[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (r < lo) x[i].x = __int_as_float(__ldcg(reinterpret_cast<const int *>(code + (size_t)r * kDim) + lane));
        else if (r < hi) x[i] = __ldcg(reinterpret_cast<const float4 *>(src + (b0 + r - p0) * a.ld) + lane);
    }
    const float was = lo ? __ldcg(sp) : 0.f;
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
        const uint32_t r = warp + 8u * (uint32_t)i;
        if (r >= lo && r < hi)   // absolute values order as their bits do, NaN above infinity
            mx = max(max(max(mx, __float_as_uint(x[i].x) & 0x7fffffffu), __float_as_uint(x[i].y) & 0x7fffffffu),
                     max(__float_as_uint(x[i].z) & 0x7fffffffu, __float_as_uint(x[i].w) & 0x7fffffffu));
    }
    mx = __reduce_max_sync(0xffffffffu, mx);
    if (lane == 0) s_max[warp] = mx;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 8; ++w) mx = max(mx, s_max[w]);
    const bool bad = mx >= 0x7f800000u || was != was;
    // divided in 64 bits and rounded once
    const float fresh = (float)((double)__uint_as_float(mx) / 127.0);
    const float now = bad ? __int_as_float(0x7fffffff) : fmaxf(fresh, was);
    const float inv = 1.0f / now;
    const bool slow = now < 7.8886090522101181e-31f, grew = !bad && now > was;
    if (threadIdx.x == 0) *sp = now;
    uint32_t sum[4] = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
        const uint32_t r = warp + 8u * (uint32_t)i;
        if (r >= hi) continue;
        uint32_t q[4];   // 0x4B400000 + code
        if (r < lo) {
            const int w = __float_as_int(x[i].x);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                int c = (int)(int8_t)(w >> (8 * j));
                if (grew) c = (int)rint((double)c * (double)was / (double)now);
                q[j] = (uint32_t)c + 0x4B400000u;
            }
        } else if (bad || now == 0.f) {
            q[0] = q[1] = q[2] = q[3] = 0x4B400000u;
        } else {
            quantise(x[i], now, inv, slow, q);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) sum[j] += q[j] - 0x4B400000u;
        if (r >= lo || grew)
            reinterpret_cast<uint32_t *>(code + (size_t)r * kDim)[lane] =
                __byte_perm(__byte_perm(q[0], q[1], 0x0040), __byte_perm(q[2], q[3], 0x0040), 0x5410);
    }
    if (is_v || !a.c.k_sum) return;
    *reinterpret_cast<uint4 *>(&s_sum[warp][4 * lane]) = make_uint4(sum[0], sum[1], sum[2], sum[3]);
    __syncthreads();
    if (threadIdx.x < kDim) {
        uint32_t t = 0;
#pragma unroll
        for (int w = 0; w < 8; ++w) t += s_sum[w][threadIdx.x];
        a.c.k_sum[(head * a.c.n_blocks + blk) * kDim + threadIdx.x] = (int16_t)t;
    }
}

// ----------------------------------------------------------------- read ----

struct ReadArgs {
    Cache c;
    Rows r;
    float *k, *v;
    uint64_t ld;
    uint32_t early;
};

constexpr int kReadRows = 8;   // rows per warp, all loaded before the first is stored

// value = code * scale, one warp per 8 consecutive rows of a KV head (lane = 4
// dimensions). 1 byte read and 4 written per value: 8192 tokens of 8 heads take 15
// to 18.5 us (84 MB, 4.5 to 5.7 TB/s; 12.9 at the copy rate). Under ncu the stalls
// are waits for the codes, 4 bytes a lane and load.
__global__ void __launch_bounds__(256) read_kernel(const __grid_constant__ ReadArgs a)
{
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
    wait_predecessor(a.early);
    const uint32_t s = blockIdx.z, h = blockIdx.y >> 1, is_v = blockIdx.y & 1u;
    const uint32_t n = row_count(a.r, s), i0 = (blockIdx.x * 8u + warp) * kReadRows;
    if (i0 >= n) return;
    const uint64_t p0 = __ldcg(a.r.pos0 + s);
    const size_t head = (size_t)s * a.c.kv_heads + h;
    const int8_t *code = (is_v ? a.c.v : a.c.k) + head * a.c.max_context * kDim;
    const float *scale = (is_v ? a.c.v_scale : a.c.k_scale) + head * a.c.n_blocks;
    float *dst = (is_v ? a.v : a.k) + (size_t)s * a.r.tokens * a.ld + (size_t)h * kDim;
    int w[kReadRows];
    float sc[kReadRows];
#pragma unroll
    for (int i = 0; i < kReadRows; ++i) {
        const uint64_t p = p0 + i0 + i;
        w[i] = 0;
        sc[i] = __int_as_float(0x7fffffff);   // a position past the cache reads as NaN
        if (i0 + i < n && p < a.c.max_context) {
            w[i] = __ldcg(reinterpret_cast<const int *>(code + p * kDim) + lane);
            sc[i] = __ldcg(scale + (p >> a.c.block_log2));
        }
    }
#pragma unroll
    for (int i = 0; i < kReadRows; ++i)
        if (i0 + i < n)
            reinterpret_cast<float4 *>(dst + (size_t)(i0 + i) * a.ld)[lane] =
                make_float4((float)(int8_t)w[i] * sc[i], (float)(int8_t)(w[i] >> 8) * sc[i],
                            (float)(int8_t)(w[i] >> 16) * sc[i], (float)(w[i] >> 24) * sc[i]);
}


// ------------------------------------------------------ attention, few rows --
//
// One cluster of CTAs per (sequence, KV head, tile of 8 NT query rows; rows
// are (token, head of the group), token-major). The cached positions come in
// chunks of 16, dealt out over all warps of the cluster; each warp keeps a
// softmax state of its own (running maximum, sum, output), and the states
// merge through shared memory, then through the cluster's distributed shared
// memory: one launch, no workspace.
//
// Chunks arrive as two TMA copies (16 rows of K, 16 of V, swizzled) into a ring
// of the warp's own, kStages deep, with a barrier per slot: no CTA-wide step
// until the merge. ldmatrix reads K as the MMAs want it; of V a lane reads the
// 16 dimensions g of rows 2t, 2t + 1, 2t + 8, 2t + 9 (g = lane / 4, t = lane
// % 4), which two byte permutations turn into pairs of rows. Neither has a bank
// conflict. (16-byte cp.async copies by the lanes instead: 4.7 TB/s without any
// arithmetic, bound by the load/store unit.)
//
//   S^T = K Q^T   m16n8k32 integer MMAs straight on the codes (rows are
//                 positions, columns query rows). Q is staged as three int8
//                 planes, q = max|q| / 127 (p0 + p1 / 254 + p2 / 254^2), off by
//                 at most 2^-22 max|q|; the integer sums are exact.
//   O^T += V^T P^T  m16n8k16 binary16 MMAs (rows are dimensions): the codes are
//                 exact in binary16, P is split into two terms hi + lo (22
//                 bits). A chunk lies in one block, so its V scale is a factor
//                 of the chunk's own sums as they join the output: blocks
//                 without weight, or that a row does not see, cost no bits.
//                 P enters as 2^9 p <= 2^15 and is off by 2^-34 of the row's
//                 largest weight where it is small. That would show where a
//                 small weight meets a large V scale, so a chunk whose scale is
//                 more than 64 times the smallest so far takes its weights
//                 against its own maximum (a warp's scales come 32 chunks at a
//                 time, and one ballot marks those chunks; the maximum of every
//                 chunk instead: 108 us where this takes 89, three bfloat16
//                 terms of P: 110).
//
// The maximum is lazy: a row's is raised only when a score passes it by 6 (in
// the exponent's base 2), which is rare after the first chunk, so a chunk
// needs no reduction over lanes.
// Bound by HBM for long caches (256 bytes per position and KV head, read once: 8
// sequences of 32768 positions, 40 heads on 8, 89 us, 6.0 TB/s or 92 % of the
// copy rate), by launch, first-byte latency and the chain of one chunk for short
// ones (640 positions 5.4 us, 8448 10.6 us).

constexpr uint32_t kStages = 3;
constexpr uint32_t kWarps = 8, kThreads = kWarps * 32;   // block selection
constexpr uint32_t kSlot = 8 * 32 * 16;                     // bytes of a chunk: 16 rows of K and V

// The states that a CTA receives at most, C ceil(8 NT / C) over the sizes of a cluster: 16, or 30 at C = 15
constexpr uint32_t received(int NT) { return NT == 1 ? 16u : 30u; }
constexpr uint32_t kRecStride = kDim + 4;                   // output, maximum, sum
constexpr int kSumBits = 0x4B400000;                  // 2^23 + 2^22: integer sums below 2^22 read as floats

__device__ __forceinline__ void mma_s8(int (&d)[4], const int (&a)[4], uint32_t b0, uint32_t b1)
{
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// The first of a sum: onto the constant c in every element
__device__ __forceinline__ void mma_s8_first(int (&d)[4], const int (&a)[4], uint32_t b0, uint32_t b1, int c)
{
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "r"(c));
}

__device__ __forceinline__ void mma_h(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// The transpose of an 8 x 8 matrix of 16-bit values (row = lane / 4, two columns a lane)
__device__ __forceinline__ uint32_t transpose8(uint32_t x)
{
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

// 16 rows of 128 bytes from row `row` of a tensor of codes to shared memory, 16-byte
// chunk c of row r at chunk c ^ (r % 8); rows behind the tensor's end are zeros
__device__ __forceinline__ void load_rows(uint32_t dst, const CUtensorMap *map, uint32_t row, uint64_t *bar)
{
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                 ::"r"(dst), "l"(map), "r"(0), "r"((int)row), "r"(smem_addr(bar))
                 : "memory");
}

// Four 8 x 16-byte matrices: lane i has the address of row i % 8 of matrix i / 8, and gets bytes 4 t .. 4 t + 3 of
// row g of each (g = lane / 4, t = lane % 4)
__device__ __forceinline__ void load_matrices(int (&d)[4], uint32_t addr)
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
                 : "r"(addr)
                 : "memory");
}

__device__ __forceinline__ uint4 ld_shared4(uint32_t addr)
{
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
    return v;
}

// Split: arrive once the CTA runs, wait before the first access to another CTA's shared memory
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.aligned;" ::: "memory"); }
__device__ __forceinline__ void st_cluster(const float *p, uint32_t cta, float4 v)
{
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_addr(p)), "r"(cta));
    asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(r), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w)
                 : "memory");
}
__device__ __forceinline__ void st_cluster(unsigned long long *p, uint32_t cta, unsigned long long v)
{
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_addr(p)), "r"(cta));
    asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(r), "l"(v) : "memory");
}

// The arguments of the few-rows kernels: the codes as tensors of 128-byte rows, too
struct FewArgs : AttnArgs {
    CUtensorMap kmap, vmap;
};

template <int NT, uint32_t W>
struct alignas(1024) Smem {
    union {
        uint8_t ring[W][kStages][kSlot];
        float wrec[W][8 * NT][kRecStride];     // the warps' outputs, once the ring is done with
    } u;
    float rec[W < 8 ? 1 : received(NT)][kRecStride];   // the states that the cluster's CTAs send of this CTA's rows (W < 8: no cluster)
    uint64_t full[W][kStages];                 // a chunk has landed
    uint32_t err;
    float2 wml[W][8 * NT];                     // the warps' maxima and sums
    alignas(16) uint32_t plane[3][8 * NT][kDim / 4 + 16];   // in the order of the B operands (lane t: 8 words from 8 t);
                                               // rows 48 words apart: their reads have no bank conflict
    float qs[8 * NT];                          // what a unit of the first plane is worth in each row
};

// Which positions a tile's keys are: chunk c holds key0(c) .. key0(c) + 15.
struct Dense {
    __device__ __forceinline__ uint32_t key0(uint32_t c) const { return c * kChunk; }
};

// Four dimensions of the output of the tile's row i; NaN where its position lies past the cache
__device__ __forceinline__ void store_row(const AttnArgs &a, const TileRows &tr, uint32_t s, uint32_t h, uint32_t i,
                                          uint64_t p0, uint32_t d4, float4 x)
{
    const uint2 r = tr.at(i);
    const float nan = __int_as_float(0x7fffffff);
    if (p0 + r.x >= a.c.max_context) x = make_float4(nan, nan, nan, nan);
    reinterpret_cast<float4 *>(a.out + ((size_t)s * a.r.tokens + r.x) * a.ldo + (size_t)(h * a.group + r.y) * kDim)[d4] = x;
}

// This warp's query rows warp, warp + 8, ... of the tile (lane = 4 dimensions; warps from 8 on have none; of W < 8
// warps, every W-th row). Rows of tokens that the call does not have are zeros; rows past n_tok are read and their
// results dropped.
constexpr uint32_t row_warps(uint32_t W) { return W < 8u ? W : 8u; }
template <int NT, uint32_t W>
struct Queries {
    float4 x[8 * NT / row_warps(W)];
};
template <int NT, uint32_t W>
__device__ __forceinline__ void load_queries(const AttnArgs &a, const TileRows &tr, uint32_t s, uint32_t h, Queries<NT, W> &q)
{
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
#pragma unroll
    for (uint32_t i = 0; i < 8u * NT / row_warps(W); ++i) {
        const uint2 r = tr.at(warp + row_warps(W) * i);
        float4(&x)[8 * NT / row_warps(W)] = q.x;
        x[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (warp < 8u && r.x < a.r.tokens)
            x[i] = __ldcg(reinterpret_cast<const float4 *>(a.q + ((size_t)s * a.r.tokens + r.x) * a.ldq +
                                                          (size_t)(h * a.group + r.y) * kDim) + lane);
    }
}

// The maximum is raised by a score that passes it by kFewLazy; weights enter their MMAs times kWeightUnit; a V scale
// kSteep times the smallest takes its chunk's own maximum.
constexpr float kFewLazy = 6.0f, kWeightUnit = 0x1p9f, kSteep = 64.0f;

// The ring's barriers, by the lane that will use them; before anything is read
template <int NT, uint32_t W>
__device__ __forceinline__ void init_ring(const FewArgs &a, Smem<NT, W> &sm)
{
    if ((threadIdx.x & 31u) == 0u) {
        for (uint32_t i = 0; i < kStages; ++i) mbar_init(&sm.full[threadIdx.x >> 5][i], 1u);
        fence_mbar_init();
    }
    if (threadIdx.x == 0u) {
        sm.err = kStatusOk;
        asm volatile("prefetch.tensormap [%0];" ::"l"(&a.kmap) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&a.vmap) : "memory");
    }
    __syncthreads();
}

// One (sequence, KV head, tile of query rows) on this cluster. `rows`: the
// tile's rows that exist. KEYS deals chunks [0, chunks). The CTAs of a cluster
// have arrived on its barrier once before.
template <int NT, uint32_t W, class KEYS>
__device__ __forceinline__ void attend(const FewArgs &a, Smem<NT, W> &sm, const KEYS &keys, const Queries<NT, W> &q,
                                       const TileRows &tr, uint32_t s, uint32_t h, uint32_t rows, uint64_t p0,
                                       uint32_t chunks)
{
    constexpr uint32_t R = 8 * NT;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u, g = lane >> 2, t = lane & 3u;
    const uint32_t C = cluster_size(), rank = cluster_rank();
    const size_t head = (size_t)s * a.c.kv_heads + h;
    const uint32_t row0 = (uint32_t)head * a.c.max_context;   // of the tensors of codes
    const float *ksc = a.c.k_scale + head * a.c.n_blocks, *vsc = a.c.v_scale + head * a.c.n_blocks;

    // this warp's chunks are first, first + step, ...
    const uint32_t first = rank + C * warp, step = C * W;
    const uint32_t ring = smem_addr(sm.u.ring[warp][0]);
    uint64_t *const full = sm.full[warp];
    auto issue = [&](uint32_t i, uint32_t slot) {
        const uint32_t c = first + i * step;
        if (c < chunks && lane == 0) {
            const uint32_t row = row0 + keys.key0(c), dst = ring + slot * kSlot;
            mbar_arrive_expect_tx(full + slot, kSlot);
            load_rows(dst, &a.kmap, row, full + slot);
            load_rows(dst + kSlot / 2u, &a.vmap, row, full + slot);
        }
    };
#pragma unroll
    for (uint32_t i = 0; i < kStages - 1; ++i) issue(i, i);
    // K: matrices (rows 0-7, 8-15) x (chunks 2 st, 2 st + 1) of step st; V: rows 2 t, 2 t + 1 (and 8 on), chunk g
    const uint32_t kx = (lane >> 4) ^ (lane & 7u), koff = (lane & 15u) * 128u;
    const uint32_t voff0 = kSlot / 2u + 256u * t + ((g ^ (2u * t)) << 4), voff1 = kSlot / 2u + 256u * t + 128u + ((g ^ (2u * t + 1u)) << 4);
    float ksl, vsl;   // lane: the scales of the warp's chunk 32 (i / 32) + lane
    float least = INFINITY;   // the smallest V scale of the chunks so far and these
    uint32_t far = 0u;        // which of them have one far above it
    auto scales = [&](uint32_t i) {
        const uint32_t b = keys.key0(min(first + (i + lane) * step, chunks - 1u)) >> a.c.block_log2;
        ksl = __ldcg(ksc + b);
        vsl = __ldcg(vsc + b);
    };
    auto mark = [&]() {
        least = fminf(least, __uint_as_float(__reduce_min_sync(0xffffffffu, __float_as_uint(vsl) & 0x7fffffffu)));
        far = __ballot_sync(0xffffffffu, !(fabsf(vsl) <= kSteep * least));
    };
    scales(0u);

    // the query rows as int8 planes; powers of two keep max|q| and its reciprocal away from the ends of the range
    if (warp < 8u)
#pragma unroll
    for (uint32_t i = 0; i < 8u * NT / row_warps(W); ++i) {
        const float v[4] = {q.x[i].x, q.x[i].y, q.x[i].z, q.x[i].w};
        uint32_t mx = 0u;
#pragma unroll
        for (int j = 0; j < 4; ++j) mx = max(mx, __float_as_uint(v[j]) & 0x7fffffffu);
        mx = __reduce_max_sync(0xffffffffu, mx);
        const float amax = __uint_as_float(mx);
        const float up = amax < 0x1p-60f ? 0x1p64f : amax > 0x1p60f ? 0x1p-64f : 1.0f;
        const float r = 127.0f * rcp(amax * up);
        uint32_t w[3] = {0u, 0u, 0u};
        if (mx && mx < 0x7f800000u) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float y = v[j] * up * r;
#pragma unroll
                for (int p = 0; p < 3; ++p) {
                    const float c = rintf(y);
                    y = (y - c) * 254.0f;
                    w[p] |= (uint32_t)((int)c & 255) << (8 * j);
                }
            }
        }
        const uint32_t row = warp + row_warps(W) * i;
#pragma unroll
        for (int p = 0; p < 3; ++p) sm.plane[p][row][8u * (lane & 3u) + (lane >> 2)] = w[p];
        // a row with a non-finite value: every score NaN
        if (lane == 0) sm.qs[row] = mx >= 0x7f800000u ? __int_as_float(0x7fffffff) : mx ? rcp(r) * (amax < 0x1p-60f ? 0x1p-64f : amax > 0x1p60f ? 0x1p64f : 1.0f) : 0.f;
    }
    __syncthreads();

    float qs[NT][2];
    uint32_t last[NT][2];   // the last position that columns 2 t and 2 t + 1 see
    const uint32_t open = (uint32_t)min(p0 + tr.tok, (uint64_t)0x7fffffffu);   // every row sees the positions up to it
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const uint32_t i = 8u * (uint32_t)nt + 2u * t + (uint32_t)e;
            qs[nt][e] = sm.qs[i] * kScoreScale;
            last[nt][e] = i < rows ? (uint32_t)min(p0 + tr.at(i).x, (uint64_t)0x7fffffffu) : open;
        }

    uint64_t o[NT][8][2];   // dimension rows g and g + 8 of MMA j: columns 2 t and 2 t + 1
    float m[NT][2], l[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        m[nt][0] = m[nt][1] = -INFINITY;
        l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) o[nt][j][0] = o[nt][j][1] = 0ull;
    }
    mark();
    uint32_t slot = 0u, phase = 0u;
    bool ok = true;
    for (uint32_t i = 0, c = first; c < chunks; ++i, c += step) {
        if ((i & 31u) == 0u && i) {
            scales(i);
            mark();
        }
        __syncwarp();   // every lane is done with the slot that chunk i - 1 left
        issue(i + kStages - 1, slot ? slot - 1u : kStages - 1u);
        ok = __all_sync(0xffffffffu, mbar_wait(full + slot, phase, &sm.err));
        if (!ok) {   // nothing of this warp is left in flight
            for (uint32_t k = 0; k < kStages && c + k * step < chunks; ++k) {
                const uint64_t w0 = global_ns();
                while (!mbar_try_wait(full + slot, phase) && global_ns() - w0 < kWaitLimitNs) {
                }
                if (++slot == kStages) slot = 0u, phase ^= 1u;
            }
            break;
        }
        const uint32_t key = keys.key0(c), in = ring + slot * kSlot;
        if (++slot == kStages) slot = 0u, phase ^= 1u;
        const float sk = __shfl_sync(0xffffffffu, ksl, i & 31u), sv = __shfl_sync(0xffffffffu, vsl, i & 31u);
        // scores: positions key + g (elements 0, 1) and key + g + 8 (2, 3), columns 2 t and 2 t + 1
        float y[NT][4];
        bool raise = false;
        const uint32_t pa = key + g, pb = key + g + 8u;
        const bool masked = key + kChunk - 1u > open;   // some row does not see all of the chunk
        {
            int ka[4][4];
#pragma unroll
            for (uint32_t st = 0; st < 4; ++st) load_matrices(ka[st], in + koff + ((kx ^ (2u * st)) << 4));
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                int d[3][4];
                // B operands: column g, dimensions 32 st + 4 t on and 32 st + 16 + 4 t on
#pragma unroll
                for (int pl = 0; pl < 3; ++pl) {
                    const uint4 lo = *reinterpret_cast<const uint4 *>(&sm.plane[pl][8 * nt + g][8u * t]);
                    mma_s8_first(d[pl], ka[0], lo.x, lo.y, kSumBits);
                    mma_s8(d[pl], ka[1], lo.z, lo.w);
                }
#pragma unroll
                for (int pl = 0; pl < 3; ++pl) {
                    const uint4 hi = *reinterpret_cast<const uint4 *>(&sm.plane[pl][8 * nt + g][8u * t + 4u]);
                    mma_s8(d[pl], ka[2], hi.x, hi.y);
                    mma_s8(d[pl], ka[3], hi.z, hi.w);
                }
                const uint64_t f = pair(sk * qs[nt][0], sk * qs[nt][1]);
                const uint64_t big = pair(-12582912.0f, -12582912.0f), step = pair(1.0f / 254.0f, 1.0f / 254.0f);
#pragma unroll
                for (int e = 0; e < 4; e += 2) {
                    uint64_t v[3];
#pragma unroll
                    for (int pl = 0; pl < 3; ++pl) v[pl] = add2(pair(__int_as_float(d[pl][e]), __int_as_float(d[pl][e + 1])), big);
                    unpair(mul2(fma2(fma2(v[2], step, v[1]), step, v[0]), f), y[nt][e], y[nt][e + 1]);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if (masked && (e < 2 ? pa : pb) > last[nt][e & 1]) y[nt][e] = -INFINITY;
                    raise |= y[nt][e] > m[nt][e & 1] + kFewLazy;
                }
            }
        }
        float w[NT][2];   // what the weights below count against the row's maximum
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) w[nt][0] = w[nt][1] = 1.0f;
        float unit = sv * (kOutUnit / kWeightUnit);
        const bool steep = far >> (i & 31u) & 1u;
        if (__any_sync(0xffffffffu, raise) || steep) {
            const float poison = sv - sv;   // NaN for a scale that is NaN or infinite: into the rows that see the chunk
            if (poison != 0.f) unit = 0.f;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                float f[2] = {1.0f, 1.0f};
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float x = fmaxf(y[nt][e], y[nt][2 + e]);
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
                    if (x > m[nt][e] + kFewLazy) {   // each row by itself
                        f[e] = m[nt][e] == -INFINITY ? 0.f : ex2(m[nt][e] - x);
                        m[nt][e] = x;
                        l[nt][e] *= f[e];
                    }
                    const float d = !steep || x == -INFINITY ? 0.f : x - m[nt][e];
                    w[nt][e] = ex2(d);
                    y[nt][e] += poison - d;
                    y[nt][2 + e] += poison - d;
                }
                const uint64_t f2 = pair(f[0], f[1]);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    o[nt][j][0] = mul2(o[nt][j][0], f2);
                    o[nt][j][1] = mul2(o[nt][j][1], f2);
                }
            }
        }
        const uint64_t unit2 = pair(unit, unit);
        uint32_t bh[NT][2], bl[NT][2];
        uint64_t by[NT];   // what the chunk's sums count in the output
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            float z[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                z[e] = ex2(y[nt][e] - m[nt][e & 1]);
                // a masked position counts nothing, whatever its block's scales are
                if (masked && (e < 2 ? pa : pb) > last[nt][e & 1]) z[e] = 0.f;
            }
#pragma unroll
            for (int e = 0; e < 2; ++e) l[nt][e] = fmaf(w[nt][e], z[e] + z[2 + e], l[nt][e]);
            by[nt] = mul2(pair(w[nt][0], w[nt][1]), unit2);
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                float hi[2], lo[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    z[2 * half + e] *= kWeightUnit;
                    hi[e] = __uint_as_float(__float_as_uint(z[2 * half + e]) & 0xffffe000u);   // exact in binary16
                    lo[e] = z[2 * half + e] - hi[e];
                }
                bh[nt][half] = transpose8(h2_bits(hi[0], hi[1]));
                bl[nt][half] = transpose8(h2_bits(lo[0], lo[1]));
            }
        }
        // O^T += V^T P^T: rows g and g + 8 of MMA j are dimensions 16 g + 2 j and 16 g + 2 j + 1
        {
            const uint4 v0 = ld_shared4(in + voff0), v1 = ld_shared4(in + voff1), v2 = ld_shared4(in + voff0 + 1024u),
                        v3 = ld_shared4(in + voff1 + 1024u);
            const uint32_t w0[4] = {v0.x, v0.y, v0.z, v0.w}, w1[4] = {v1.x, v1.y, v1.z, v1.w};
            const uint32_t w2[4] = {v2.x, v2.y, v2.z, v2.w}, w3[4] = {v3.x, v3.y, v3.z, v3.w};
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const uint32_t pick = (j & 1) ? 0x7632u : 0x5410u;
                const uint32_t ya = __byte_perm(w0[j >> 1], w1[j >> 1], pick), yb = __byte_perm(w2[j >> 1], w3[j >> 1], pick);
                const uint32_t va[4] = {codes_h2<false>(ya), codes_h2<true>(ya), codes_h2<false>(yb), codes_h2<true>(yb)};
                // the MMAs truncate their sums, so only a chunk's are left to them
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    float x[4] = {0.f, 0.f, 0.f, 0.f};
                    mma_h(x, va, bl[nt][0], bl[nt][1]);
                    mma_h(x, va, bh[nt][0], bh[nt][1]);
                    o[nt][j][0] = fma2(pair(x[0], x[1]), by[nt], o[nt][j][0]);
                    o[nt][j][1] = fma2(pair(x[2], x[3]), by[nt], o[nt][j][1]);
                }
            }
        }
    }
    if (!ok) l[0][0] = l[0][1] = l[NT - 1][0] = l[NT - 1][1] = __int_as_float(0x7fffffff);   // the output will be NaN
    __syncthreads();   // every warp is done with the ring: it takes the warps' outputs

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
            for (int j = 0; j < 8; j += 2) {
                float v[4][2];
#pragma unroll
                for (int k = 0; k < 4; ++k) unpair(o[nt][j + (k >> 1)][k & 1], v[k][0], v[k][1]);
                *reinterpret_cast<float4 *>(&sm.u.wrec[warp][i][16u * g + 2u * (uint32_t)j]) = make_float4(v[0][e], v[1][e], v[2][e], v[3][e]);
            }
        }
    if (C > 1u) cluster_wait();   // the other CTAs run: their shared memory may be written
    __syncthreads();
    // The warps' states -> the CTA's state of each row, straight to the CTA of
    // the cluster that owns the row (row i: CTA i % C, which has `per` slots
    // from each CTA). A state that saw no position (maximum -inf, sum 0) counts
    // nothing.
    const float cinv = rcp((float)C);
    const uint32_t per = (uint32_t)(((float)(R + C) - 0.5f) * cinv);   // ceil(R / C)
    if (threadIdx.x < 256u) {
        constexpr uint32_t kPer = 32u * row_warps(W) / R;   // threads per row, 4 dimensions at a time
        const uint32_t i = threadIdx.x / kPer, part = threadIdx.x % kPer, turn = (uint32_t)(((float)i + 0.5f) * cinv);   // i / C
        float2 ml[W];
        float M = -INFINITY, L = 0.f;
#pragma unroll
        for (uint32_t w = 0; w < W; ++w) {
            ml[w] = sm.wml[w][i];
            M = fmaxf(M, ml[w].x);
        }
#pragma unroll
        for (uint32_t w = 0; w < W; ++w) {
            ml[w].x = ml[w].x == -INFINITY && ml[w].y == 0.f ? 0.f : ex2(ml[w].x - M);
            L = fmaf(ml[w].x, ml[w].y, L);
        }
        const float inv = (1.0f / kOutUnit) / L;
#pragma unroll
        for (uint32_t d = part; d < kDim / 4u; d += kPer) {
            float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (uint32_t w = 0; w < W; ++w) {
                const float4 y = *reinterpret_cast<const float4 *>(&sm.u.wrec[w][i][4u * d]);
                x.x = fmaf(ml[w].x, y.x, x.x);
                x.y = fmaf(ml[w].x, y.y, x.y);
                x.z = fmaf(ml[w].x, y.z, x.z);
                x.w = fmaf(ml[w].x, y.w, x.w);
            }
            if (i >= rows) continue;
            if (C == 1u) store_row(a, tr, s, h, i, p0, d, make_float4(x.x * inv, x.y * inv, x.z * inv, x.w * inv));
            else st_cluster(&sm.rec[rank * per + turn][4u * d], i - turn * C, x);
        }
        if (C > 1u && part == 0u && i < rows)
            st_cluster(&sm.rec[rank * per + turn][kDim], i - turn * C, make_float4(M, L, 0.f, 0.f));
    }
    if (W < 8u || C == 1u) return;
    cluster_sync();   // every record has arrived; nothing remote is touched from here on
    // warp k: row rank + k C; lane: a CTA's maximum and sum, then 4 dimensions
    const uint32_t i = rank + warp * C;
    if (warp >= per || i >= min(rows, R)) return;
    const float *rec = sm.rec[lane * per + warp];
    const float mc = lane < C ? rec[kDim] : -INFINITY, lc = lane < C ? rec[kDim + 1] : 0.f;
    float M = mc;
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o, 16));
    const float f = mc == -INFINITY && lc == 0.f ? 0.f : ex2(mc - M);
    float L = f * lc;
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) L += __shfl_xor_sync(0xffffffffu, L, o, 16);
    L = __shfl_sync(0xffffffffu, L, 0);
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 2
    for (uint32_t c = 0; c < C; ++c) {
        const float4 y = *reinterpret_cast<const float4 *>(&sm.rec[c * per + warp][4u * lane]);
        const float fc = __shfl_sync(0xffffffffu, f, (int)c);
        x.x = fmaf(fc, y.x, x.x);
        x.y = fmaf(fc, y.y, x.y);
        x.z = fmaf(fc, y.z, x.z);
        x.w = fmaf(fc, y.w, x.w);
    }
    const float inv = (1.0f / kOutUnit) / L;
    store_row(a, tr, s, h, i, p0, lane, make_float4(x.x * inv, x.y * inv, x.z * inv, x.w * inv));
}

template <int NT, uint32_t W>
__global__ void __launch_bounds__(W * 32, 1) attn_kernel(const __grid_constant__ FewArgs a)
{
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    Smem<NT, W> &sm = *reinterpret_cast<Smem<NT, W> *>(smem_raw);
    const uint32_t s = blockIdx.z, h = blockIdx.y, r0 = (a.tiles == 1u ? 0u : blockIdx.x / cluster_size()) * 8u * NT;
    if (cluster_size() > 1u) cluster_arrive();
    TileRows tr{0u, 0u, a.group, a.group_inv};
    if (r0) {
        tr.tok = r0 / a.group;
        tr.rem = r0 - tr.tok * a.group;
    }
    init_ring(a, sm);
    wait_predecessor(a.early);
    const uint64_t p0 = __ldcg(a.r.pos0 + s);
    const uint32_t all = row_count(a.r, s) * a.group;
    Queries<NT, W> q;
    load_queries(a, tr, s, h, q);
    if (r0 >= all) {   // the whole cluster leaves
        if (cluster_size() > 1u) cluster_wait();
        return;
    }
    const uint32_t rows = min(all - r0, 8u * NT);
    const uint32_t limit = (uint32_t)min(p0 + tr.at(rows - 1u).x + 1u, (uint64_t)a.c.max_context);
    attend<NT, W>(a, sm, Dense{}, q, tr, s, h, rows, p0, (limit + kChunk - 1u) / kChunk);
}

// ------------------------------------------------- attention, chosen blocks --
//
// One cluster per (sequence, token, KV head): the blocks before the token's own
// are scored, the best n_sel - 1 of them and the token's own block are
// attended. Score of block b: the group's query rows are summed (64 bits) and
// rounded to int8, c = rint(127 qbar / max|qbar|); the score is
// (c . k_sum_b) * k_scale_b, an integer dot product times one fp32 factor.
// Both are exact in 64 bits (28 + 24 bits), so the choice does not depend on
// the order of any sum; equal scores go to the lower block. A NaN score stands
// above every number: a poisoned block is chosen and shows in the output.
// The CTAs of the cluster score every C-th block each, send the keys to all of
// them, and each picks the blocks on its own (a search for the lowest chosen
// key), so the whole operator is one launch.
// Bound by latency: 260 bytes per candidate block, then n_sel blocks.

struct Chosen {
    const uint32_t *list;
    uint32_t per_log2, block_log2;   // chunks per block, positions per block
    __device__ __forceinline__ uint32_t key0(uint32_t c) const
    {
        return (list[c >> per_log2] << block_log2) + (c & ((1u << per_log2) - 1u)) * kChunk;
    }
};

struct PickSmem {
    alignas(16) int8_t code[kDim];
    unsigned long long most[4], least;
    alignas(16) uint4 count[2][kWarps];
    uint32_t scan[kWarps];
};

// The keys lie behind PickSmem in the ring, which the attention fills later.
constexpr uint32_t kMaxBlocks = (uint32_t)((kWarps * kStages * kSlot - sizeof(PickSmem)) / 8u);

// The sum of the group's query rows; thread = dimension (128 of them)
__device__ __forceinline__ double pool_query(const AttnArgs &a, const float *q)
{
    double x = 0.0;
    if (threadIdx.x < kDim)
        for (uint32_t i = 0; i < a.group; i += 8u) {   // eight on their way at a time
            float v[8];
#pragma unroll
            for (uint32_t k = 0; k < 8u; ++k) v[k] = i + k < a.group ? __ldcg(q + (size_t)(i + k) * kDim + threadIdx.x) : 0.f;
#pragma unroll
            for (uint32_t k = 0; k < 8u; ++k) x += (double)v[k];
        }
    return x;
}

// The pooled query as int8 codes. All threads.
__device__ __forceinline__ void code_query(PickSmem &ps, double x)
{
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
    unsigned long long b = (unsigned long long)__double_as_longlong(fabs(x));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) b = max(b, __shfl_xor_sync(0xffffffffu, b, o));
    if (lane == 0 && warp < 4u) ps.most[warp] = b;
    __syncthreads();
    if (warp < 4u) {
#pragma unroll
        for (uint32_t w = 0; w < 4u; ++w) b = max(b, ps.most[w]);
        const double most = __longlong_as_double((long long)b);
        ps.code[threadIdx.x] = most > 0.0 && most < INFINITY ? (int8_t)(int)rint(127.0 * x / most) : (int8_t)0;
    }
    __syncthreads();
}

// A word that orders as the scores do
__device__ __forceinline__ unsigned long long block_key(int d, float sc)
{
    const double x = (double)d * (double)sc + 0.0;   // + 0: one zero
    const unsigned long long k = (unsigned long long)__double_as_longlong(x);
    return x != x ? ~0ull : (k >> 63) ? ~k : k | 1ull << 63;
}

// Keys of blocks rank, rank + C, ... below nb, into every CTA's `key`: 8 lanes per block, 16 dimensions each.
__device__ __forceinline__ void score_blocks(const AttnArgs &a, const PickSmem &ps, size_t head, uint32_t nb,
                                             unsigned long long *key, uint32_t C, uint32_t rank)
{
    const uint32_t part = threadIdx.x & 7u, grp = threadIdx.x >> 3;
    const int4 qc = *reinterpret_cast<const int4 *>(ps.code + 16u * part);
    const int16_t *sums = a.c.k_sum + head * a.c.n_blocks * kDim + 16u * part;
    const float *scale = a.c.k_scale + head * a.c.n_blocks;
    const uint32_t step = C * (kThreads / 8u);
#pragma unroll 4
    for (uint32_t base = rank; base < nb; base += step) {   // uniform over the CTA: the shuffles are whole
        const uint32_t b = base + C * grp;
        int4 u = make_int4(0, 0, 0, 0), v = u;
        float sc = 0.f;
        if (b < nb) {
            const int4 *row = reinterpret_cast<const int4 *>(sums + (size_t)b * kDim);
            u = __ldcg(row);
            v = __ldcg(row + 1);
            sc = __ldcg(scale + b);
        }
        int d = __dp2a_lo(u.x, qc.x, 0);
        d = __dp2a_hi(u.y, qc.x, d);
        d = __dp2a_lo(u.z, qc.y, d);
        d = __dp2a_hi(u.w, qc.y, d);
        d = __dp2a_lo(v.x, qc.z, d);
        d = __dp2a_hi(v.y, qc.z, d);
        d = __dp2a_lo(v.z, qc.w, d);
        d = __dp2a_hi(v.w, qc.w, d);
        d += __shfl_xor_sync(0xffffffffu, d, 1);
        d += __shfl_xor_sync(0xffffffffu, d, 2);
        d += __shfl_xor_sync(0xffffffffu, d, 4);
        const unsigned long long k = block_key(d, sc);
        if (b < nb) {
            if (C == 1u) {
                if (part == 0u) key[b] = k;
            } else {
                for (uint32_t c = part; c < C; c += 8u) st_cluster(key + b, c, k);
            }
        }
    }
}

// The largest value that at least `want` of key[0, nb) reach, 0 < want < nb, or
// one that exactly `want` of them do. One warp, nb <= 512: bit by bit with the
// keys' upper words in registers (a step is 16 comparisons a lane and one sum
// over the warp), mostly 20 steps; the lower words count only where the upper
// ones do not part the keys.
constexpr uint32_t kWarpPick = 512;
__device__ __forceinline__ unsigned long long search_warp(const unsigned long long *key, uint32_t nb, uint32_t want)
{
    constexpr uint32_t kPer = kWarpPick / 32u;
    const uint32_t lane = threadIdx.x & 31u;
    uint32_t k[kPer], least = 0u, n = nb;
    if (nb <= kWarpPick) {
#pragma unroll
        for (uint32_t j = 0; j < kPer; ++j) k[j] = 32u * j + lane < nb ? (uint32_t)(key[32u * j + lane] >> 32) : 0u;
        for (uint32_t bit = 1u << 31; bit && n != want; bit >>= 1) {
            const uint32_t at = least | bit;
            uint32_t c = 0u;
#pragma unroll
            for (uint32_t j = 0; j < kPer; ++j) c += k[j] >= at ? 1u : 0u;
            c = __reduce_add_sync(0xffffffffu, c);
            if (c >= want) least = at, n = c;
        }
    }
    unsigned long long all = (unsigned long long)least << 32;
    for (unsigned long long bit = nb <= kWarpPick ? 1ull << 31 : 1ull << 63; bit && n != want; bit >>= 1) {
        uint32_t c = 0u;
#pragma unroll 8
        for (uint32_t i = lane; i < nb; i += 32u) c += key[i] >= (all | bit) ? 1u : 0u;
        c = __reduce_add_sync(0xffffffffu, c);
        if (c >= want) all |= bit, n = c;
    }
    return all;
}

// The same by all threads, for more blocks: three bits at a time, the keys at or
// above each of their values 1 .. 7 counted in one pass, two counts of 16 bits a word
__device__ __forceinline__ unsigned long long search_all(PickSmem &ps, const unsigned long long *key, uint32_t nb, uint32_t want)
{
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
    unsigned long long least = 0ull;
    for (int bit = 61, turn = 0;; bit = max(bit - 3, 0), turn ^= 1) {   // the last step sees two bits again
        uint32_t c[4] = {0u, 0u, 0u, 0u};
        for (uint32_t i = threadIdx.x; i < nb; i += kThreads) {
            const unsigned long long k = key[i];
#pragma unroll
            for (uint32_t v = 1; v < 8u; ++v)
                if (k >= (least | (unsigned long long)v << bit)) c[v >> 1] += 1u << (16u * (v & 1u));
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) c[j] = __reduce_add_sync(0xffffffffu, c[j]);
        if (lane == 0) ps.count[turn][warp] = make_uint4(c[0], c[1], c[2], c[3]);
        __syncthreads();
        uint4 all = ps.count[turn][0];
#pragma unroll
        for (uint32_t w = 1; w < kWarps; ++w) {
            const uint4 n = ps.count[turn][w];
            all.x += n.x;
            all.y += n.y;
            all.z += n.z;
            all.w += n.w;
        }
        // the largest value that `want` keys reach
        const uint32_t n[8] = {nb, all.x >> 16, all.y & 0xffffu, all.y >> 16, all.z & 0xffffu, all.z >> 16, all.w & 0xffffu,
                               all.w >> 16};
        uint32_t v = 0u, at = nb;
#pragma unroll
        for (uint32_t j = 1; j < 8u; ++j)
            if (n[j] >= want) v = j, at = n[j];
        least |= (unsigned long long)v << bit;
        if (bit == 0 || (v && at == want)) return least;
    }
}

// The `want` largest of key[0, nb), 0 < want < nb, as ascending block numbers
// in list[0, want); equal keys go to the lower number. All threads.
__device__ __forceinline__ void pick_blocks(PickSmem &ps, const unsigned long long *key, uint32_t nb, uint32_t want,
                                            uint32_t *list)
{
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
    unsigned long long least;
    if (nb <= kWarpPick) {
        if (warp == 0) {
            least = search_warp(key, nb, want);
            if (lane == 0) ps.least = least;
        }
        __syncthreads();
        least = ps.least;
    } else {
        least = search_all(ps, key, nb, want);
    }
    // thread: a run of consecutive blocks; (above, equal) counts of the runs before it in one word
    const uint32_t per = (nb + kThreads - 1u) / kThreads, b0 = min(threadIdx.x * per, nb), b1 = min(b0 + per, nb);
    uint32_t cnt = 0u;
    for (uint32_t b = b0; b < b1; ++b) cnt += key[b] > least ? 1u : key[b] == least ? 1u << 16 : 0u;
    uint32_t inc = cnt;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t up = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= (uint32_t)o) inc += up;
    }
    if (lane == 31u) ps.scan[warp] = inc;
    __syncthreads();
    uint32_t before = inc - cnt, all = 0u;
#pragma unroll
    for (uint32_t w = 0; w < kWarps; ++w) {
        if (w < warp) before += ps.scan[w];
        all += ps.scan[w];
    }
    uint32_t gt = before & 0xffffu, eq = before >> 16;
    const uint32_t need = want - (all & 0xffffu);   // of the equal ones, the first
    for (uint32_t b = b0; b < b1; ++b) {
        const unsigned long long k = key[b];
        if (k > least || (k == least && eq < need)) list[gt + min(eq, need)] = b;
        gt += k > least ? 1u : 0u;
        eq += k == least ? 1u : 0u;
    }
    __syncthreads();
}

template <int NT>
__global__ void __launch_bounds__(kThreads, NT == 1 ? 2 : 1) sparse_kernel(const __grid_constant__ FewArgs a)
{
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    Smem<NT, kWarps> &sm = *reinterpret_cast<Smem<NT, kWarps> *>(smem_raw);
    PickSmem &ps = *reinterpret_cast<PickSmem *>(sm.u.ring);
    unsigned long long *key = reinterpret_cast<unsigned long long *>(&ps + 1);
    uint32_t *list = reinterpret_cast<uint32_t *>(smem_raw + sizeof(Smem<NT, kWarps>));
    const uint32_t C = cluster_size(), rank = cluster_rank();
    const uint32_t s = blockIdx.z, h = blockIdx.y, unit = C == 1u ? blockIdx.x : blockIdx.x / C;
    const uint32_t token = a.tiles == 1u ? unit : unit / a.tiles, tile = unit - token * a.tiles;
    const TileRows tr{token, tile * 8u * NT, a.group, a.group_inv};
    if (C > 1u) cluster_arrive();
    init_ring(a, sm);
    wait_predecessor(a.early);
    const uint64_t p0 = __ldcg(a.r.pos0 + s);
    const uint32_t n = row_count(a.r, s);
    const double pooled = pool_query(a, a.q + ((size_t)s * a.r.tokens + token) * a.ldq + (size_t)h * a.group * kDim);
    Queries<NT, kWarps> q;
    load_queries(a, tr, s, h, q);
    if (token >= n) {   // the whole cluster leaves
        if (C > 1u) cluster_wait();
        return;
    }
    const bool inside = p0 + token < a.c.max_context;
    const uint32_t p = inside ? (uint32_t)(p0 + token) : a.c.max_context - 1u;
    const uint32_t own = p >> a.c.block_log2, want = min(own, a.n_sel - 1u);
    const size_t head = (size_t)s * a.c.kv_heads + h;
    if (own > want && want) {
        code_query(ps, pooled);
        // the other CTAs' shared memory is written from here on: they have to run
        if (C > 1u) cluster_wait();
        score_blocks(a, ps, head, own, key, C, rank);
        if (C > 1u) {
            cluster_sync();
            cluster_arrive();
        } else {
            __syncthreads();
        }
        pick_blocks(ps, key, own, want, list);
    } else {
        for (uint32_t i = threadIdx.x; i < want; i += kThreads) list[i] = i;
    }
    if (threadIdx.x == 0) list[want] = own;
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // the ring's copies come after the keys' stores there
    __syncthreads();
    if (rank == 0 && tile == 0) {
        int32_t *sel = a.sel + (((size_t)s * a.r.tokens + token) * a.c.kv_heads + h) * a.n_sel;
        for (uint32_t i = threadIdx.x; i < a.n_sel; i += kThreads) sel[i] = inside && i <= want ? (int32_t)list[i] : -1;
    }
    const uint32_t per = a.c.block_log2 - 4u;
    const uint32_t chunks = (want << per) + ((p & ((1u << a.c.block_log2) - 1u)) / kChunk) + 1u;
    attend<NT, kWarps>(a, sm, Chosen{list, per, a.c.block_log2}, q, tr, s, h, min(a.group - tile * 8u * NT, 8u * NT), p0, chunks);
}

// The same in two launches, for many tokens: a pass that only chooses, eight
// tokens of a KV head per CTA, and one that attends to what `sel` then holds, in
// CTAs of four warps, four of them per SM. The scores of eight tokens are one
// product of integer MMAs (m16n8k32: rows are blocks, columns tokens), in which
// the sums enter as 256 hi + lo, a signed and an unsigned byte; a warp per token
// then searches. Taken where the CTAs of the one launch above, two per SM, do
// not all fit at once: 256 and 516 units (28 heads on 4, 16 of 250 blocks of
// 32) and 4128 (40 on 8, 16 of 125 blocks of 64) take 18.0, 36.1 and 302.6 us
// as one launch, 23.9, 26.6 and 195.7 us as two. Bound by instruction issue
// (400 per 16 positions) and the latency of a unit's short way.

constexpr uint32_t kPickTokens = 8;
struct TokensSmem {
    alignas(16) uint32_t code[kPickTokens][kDim / 4];
};   // then the keys, a row of n_blocks per token

// u8 x s8
__device__ __forceinline__ void mma_u8(int (&d)[4], const int (&a)[4], uint32_t b0, uint32_t b1)
{
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ size_t sel_row(const AttnArgs &a, uint32_t s, uint32_t token, uint32_t h)
{
    return (((size_t)s * a.r.tokens + token) * a.c.kv_heads + h) * a.n_sel;
}

__global__ void __launch_bounds__(32 * kPickTokens) choose_kernel(const __grid_constant__ AttnArgs a)
{
    extern __shared__ __align__(16) uint8_t choose_smem[];
    TokensSmem &sm = *reinterpret_cast<TokensSmem *>(choose_smem);
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u, s = blockIdx.z, h = blockIdx.y;
    const uint32_t first = blockIdx.x * kPickTokens, token = first + warp;
    unsigned long long *const keys = reinterpret_cast<unsigned long long *>(&sm + 1), *const key = keys + (size_t)warp * a.c.n_blocks;
    wait_predecessor(a.early);
    const uint64_t p0 = __ldcg(a.r.pos0 + s);
    const uint32_t n = row_count(a.r, s);
    if (first >= n) return;
    auto own_block = [&](uint32_t tok) { return (uint32_t)min(p0 + tok, (uint64_t)a.c.max_context - 1u) >> a.c.block_log2; };
    const bool inside = p0 + token < a.c.max_context;
    const uint32_t own = own_block(token), want = min(own, a.n_sel - 1u);
    const uint32_t most = own_block(min(first + kPickTokens, n) - 1u);   // blocks that some token scores
    int32_t *sel = a.sel + sel_row(a, s, token, h);
    if (a.n_sel > 1u && most >= a.n_sel) {
        const size_t head = (size_t)s * a.c.kv_heads + h;
        const int4 *const sums = reinterpret_cast<const int4 *>(a.c.k_sum + head * a.c.n_blocks * kDim);
        const float *const scale = a.c.k_scale + head * a.c.n_blocks;
        const uint32_t g = lane >> 2, t = lane & 3u;
        // the pooled query: lane = 4 dimensions
        double x[4] = {0.0, 0.0, 0.0, 0.0};
        if (token < n) {
            const float4 *q = reinterpret_cast<const float4 *>(a.q + ((size_t)s * a.r.tokens + token) * a.ldq + (size_t)h * a.group * kDim) + lane;
            for (uint32_t i = 0; i < a.group; i += 8u) {   // eight on their way at a time
                float4 v[8];
#pragma unroll
                for (uint32_t k = 0; k < 8u; ++k) v[k] = i + k < a.group ? __ldcg(q + (size_t)(i + k) * (kDim / 4u)) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (uint32_t k = 0; k < 8u; ++k) {
                    x[0] += (double)v[k].x;
                    x[1] += (double)v[k].y;
                    x[2] += (double)v[k].z;
                    x[3] += (double)v[k].w;
                }
            }
        }
        unsigned long long top = 0ull;
#pragma unroll
        for (int j = 0; j < 4; ++j) top = max(top, (unsigned long long)__double_as_longlong(fabs(x[j])));
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
        const double amax = __longlong_as_double((long long)top);
        uint32_t word = 0u;
        if (amax > 0.0 && amax < INFINITY)
#pragma unroll
            for (int j = 0; j < 4; ++j) word |= ((uint32_t)(int)rint(127.0 * x[j] / amax) & 255u) << (8 * j);
        sm.code[warp][lane] = word;
        __syncthreads();
        // Step st of the product takes dimensions 8 (4 st + t) + 0 .. 7 of lane t: 16 bytes of a block's sums
        uint2 qc[4];
#pragma unroll
        for (uint32_t st = 0; st < 4u; ++st) qc[st] = *reinterpret_cast<const uint2 *>(&sm.code[g][2u * (4u * st + t)]);
#pragma unroll 2
        for (uint32_t b0 = 16u * warp; b0 < most; b0 += 16u * kPickTokens) {
            const uint32_t ba = min(b0 + g, most - 1u), bb = min(b0 + g + 8u, most - 1u);
            int4 u[4], v[4];
#pragma unroll
            for (uint32_t st = 0; st < 4u; ++st) {
                u[st] = __ldcg(sums + (size_t)ba * (kDim / 8u) + 4u * st + t);
                v[st] = __ldcg(sums + (size_t)bb * (kDim / 8u) + 4u * st + t);
            }
            const float sa = __ldcg(scale + ba), sb = __ldcg(scale + bb);
            int hi[4] = {0, 0, 0, 0}, lo[4] = {0, 0, 0, 0};
#pragma unroll
            for (uint32_t st = 0; st < 4u; ++st) {
                const int l[4] = {(int)__byte_perm(u[st].x, u[st].y, 0x6420u), (int)__byte_perm(v[st].x, v[st].y, 0x6420u),
                                  (int)__byte_perm(u[st].z, u[st].w, 0x6420u), (int)__byte_perm(v[st].z, v[st].w, 0x6420u)};
                const int m[4] = {(int)__byte_perm(u[st].x, u[st].y, 0x7531u), (int)__byte_perm(v[st].x, v[st].y, 0x7531u),
                                  (int)__byte_perm(u[st].z, u[st].w, 0x7531u), (int)__byte_perm(v[st].z, v[st].w, 0x7531u)};
                mma_u8(lo, l, qc[st].x, qc[st].y);
                mma_s8(hi, m, qc[st].x, qc[st].y);
            }
#pragma unroll
            for (uint32_t e = 0; e < 4u; ++e) {
                const uint32_t b = b0 + g + (e < 2u ? 0u : 8u);
                if (b < most) keys[(size_t)(2u * t + (e & 1u)) * a.c.n_blocks + b] = block_key(256 * hi[e] + lo[e], e < 2u ? sa : sb);
            }
        }
    }
    __syncthreads();
    if (token >= n) return;
    if (!inside) {
        for (uint32_t i = lane; i < a.n_sel; i += 32u) sel[i] = -1;
        return;
    }
    if (own > want && want) {
        const unsigned long long least = search_warp(key, own, want);
        uint32_t need = want;   // of the keys equal to `least`, the first
        for (uint32_t b = lane; b - lane < own; b += 32u) need -= __popc(__ballot_sync(0xffffffffu, b < own && key[b] > least));
        const uint32_t below = (1u << lane) - 1u;
        uint32_t at = 0u, equal = 0u;
        for (uint32_t b = lane; b - lane < own; b += 32u) {
            const unsigned long long k = b < own ? key[b] : 0ull;
            const bool same = b < own && k == least;
            const uint32_t sames = __ballot_sync(0xffffffffu, same);
            const bool take = (b < own && k > least) || (same && equal + __popc(sames & below) < need);
            const uint32_t takes = __ballot_sync(0xffffffffu, take);
            if (take) sel[at + __popc(takes & below)] = (int32_t)b;
            at += __popc(takes);
            equal += __popc(sames);
        }
    } else {
        for (uint32_t i = lane; i < want; i += 32u) sel[i] = (int32_t)i;
    }
    for (uint32_t i = want + lane; i < a.n_sel; i += 32u) sel[i] = i == want ? (int32_t)own : -1;
}

constexpr uint32_t kChosenWarps = 4;

template <int NT>
__global__ void __launch_bounds__(32 * kChosenWarps, (NT == 1 ? 16 : 8) / kChosenWarps) chosen_kernel(const __grid_constant__ FewArgs a)
{
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    Smem<NT, kChosenWarps> &sm = *reinterpret_cast<Smem<NT, kChosenWarps> *>(smem_raw);
    uint32_t *list = reinterpret_cast<uint32_t *>(smem_raw + sizeof(Smem<NT, kChosenWarps>));
    const uint32_t s = blockIdx.z, h = blockIdx.y, token = a.tiles == 1u ? blockIdx.x : blockIdx.x / a.tiles;
    const uint32_t tile = blockIdx.x - token * a.tiles;
    const TileRows tr{token, tile * 8u * NT, a.group, a.group_inv};
    init_ring(a, sm);
    wait_predecessor(a.early);
    const uint64_t p0 = __ldcg(a.r.pos0 + s);
    const uint32_t n = row_count(a.r, s);
    if (token >= n) return;
    const int32_t *sel = a.sel + sel_row(a, s, token, h);
    const bool inside = p0 + token < a.c.max_context;   // else one chunk of any block, and NaN
    const uint32_t p = inside ? (uint32_t)(p0 + token) : 0u, own = p >> a.c.block_log2, want = min(own, a.n_sel - 1u);
    for (uint32_t i = threadIdx.x; i <= want; i += 32u * kChosenWarps) list[i] = min((uint32_t)__ldcg(sel + i), own);
    Queries<NT, kChosenWarps> q;
    load_queries(a, tr, s, h, q);
    __syncthreads();
    const uint32_t per = a.c.block_log2 - 4u;
    const uint32_t chunks = (want << per) + ((p & ((1u << a.c.block_log2) - 1u)) / kChunk) + 1u;
    attend<NT, kChosenWarps>(a, sm, Chosen{list, per, a.c.block_log2}, q, tr, s, h, min(a.group - tile * 8u * NT, 8u * NT), p0, chunks);
}

// ------------------------------------------------------------- host side ----

// CTAs per unit of work: the largest cluster of which all units are on the
// device at once (a second wave costs more than the smaller share saves: 8
// units of 8447 positions take 16.2 us as clusters of 16, of which 7 fit, and
// 11.0 us as clusters of 8), with 128 positions per CTA at least.
template <auto KERNEL>
uint32_t cluster_of(int dev, uint32_t threads, size_t smem, uint64_t units, uint64_t positions)
{
    for (uint32_t c = kMaxCluster; c > 1; --c)
        if ((c - 1) * 128ull < positions && clusters_at_once<KERNEL>(dev, c, threads, smem) >= units)
            return c;
    return 1;
}

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

// The checks that all calls share; fills the kernel's view of the cache.
int open_cache(const char *who, const AtlasKv8 *c, uint32_t tokens, const uint32_t *pos0, const uint32_t *n_tok, Cache &out,
               Rows &rows, int &dev, int &sms)
{
    if (!c || !c->k || !c->v || !c->k_scale || !c->v_scale || !pos0)
        return api_fail(ATLAS_EINVAL, "%s: null argument", who);
    if (c->block != 16 && c->block != 32 && c->block != 64 && c->block != 128)
        return api_fail(ATLAS_EINVAL, "%s: blocks of 16, 32, 64 or 128 positions, not %u", who, c->block);
    if (!c->nseq || c->nseq > 65535u || !c->kv_heads || c->kv_heads > 16384u || !c->max_context ||
        c->max_context > 0x7fffff00u)
        return api_fail(ATLAS_EINVAL, "%s: bad cache shape (%u sequences, %u KV heads, %u positions)", who, c->nseq,
                        c->kv_heads, c->max_context);
    if (!aligned(c->k, 16) || !aligned(c->v, 16) || !aligned(c->k_sum, 16) || !aligned(c->k_scale, 4) ||
        !aligned(c->v_scale, 4) || !aligned(pos0, 4) || !aligned(n_tok, 4))
        return api_fail(ATLAS_EINVAL, "%s: codes and sums must be 16-byte aligned, the rest 4-byte", who);
    if (tokens > 0x00ffffffu) return api_fail(ATLAS_EINVAL, "%s: at most 2^24 - 1 tokens, not %u", who, tokens);
    dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || api_device(dev, &sms) != ATLAS_OK)
        return api_fail(ATLAS_ENODEV, "%s: no sm_100 device", who);
    const void *need[] = {c->k, c->v, c->k_scale, c->v_scale, pos0, c->k_sum, n_tok};
    for (const void *p : need)
        if (p && !on_device(p, dev))
            return api_fail(ATLAS_EINVAL, "%s: the cache, pos0 and n_tok must be memory of the current device", who);
    out.k = static_cast<int8_t *>(c->k);
    out.v = static_cast<int8_t *>(c->v);
    out.k_scale = c->k_scale;
    out.v_scale = c->v_scale;
    out.k_sum = c->k_sum;
    out.nseq = c->nseq;
    out.kv_heads = c->kv_heads;
    out.max_context = c->max_context;
    out.block_log2 = c->block == 16 ? 4 : c->block == 32 ? 5 : c->block == 64 ? 6 : 7;
    out.n_blocks = (c->max_context + c->block - 1) / c->block;
    rows.pos0 = pos0;
    rows.n_tok = n_tok;
    rows.tokens = tokens;
    return ATLAS_OK;
}

// Token rows of `heads` x 128 floats, ld floats apart (0: dense).
int check_rows(const char *who, const void *p, const void *q, uint32_t heads, uint64_t &ld, int dev)
{
    if (!p || !q) return api_fail(ATLAS_EINVAL, "%s: null argument", who);
    if (!ld) ld = (uint64_t)heads * kDim;
    if (ld < (uint64_t)heads * kDim || ld % 4 || ld > 0xffffffffull)
        return api_fail(ATLAS_EINVAL, "%s: token rows %llu floats apart: at least heads x 128, a multiple of 4", who,
                        (unsigned long long)ld);
    if (!aligned(p, 16) || !aligned(q, 16)) return api_fail(ATLAS_EINVAL, "%s: token rows must be 16-byte aligned", who);
    if (!on_device(p, dev) || (q != p && !on_device(q, dev)))
        return api_fail(ATLAS_EINVAL, "%s: token rows must be memory of the current device", who);
    return ATLAS_OK;
}

// The codes as tensors of 128-byte rows, for copies of 16 rows into swizzled shared memory
int map_codes(const char *who, FewArgs &a)
{
    using Encode = decltype(&cuTensorMapEncodeTiled);
    static std::atomic<Encode> known{nullptr};
    Encode encode = known.load(std::memory_order_acquire);
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
    const cuuint64_t rows = (cuuint64_t)a.c.nseq * a.c.kv_heads * a.c.max_context;
    if (rows > 0x7fffffffull) return api_fail(ATLAS_EINVAL, "%s: more than 2^31 - 1 rows of codes", who);
    const cuuint64_t dims[2] = {kDim, rows}, strides[1] = {kDim};
    const cuuint32_t box[2] = {kDim, kChunk}, steps[2] = {1, 1};
    for (int i = 0; i < 2; ++i)
        if (encode(i ? &a.vmap : &a.kmap, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, i ? a.c.v : a.c.k, dims, strides, box, steps,
                   CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_NONE,
                   CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
            return api_fail(ATLAS_ECUDA, "%s: the codes cannot be described to the copy engine", who);
    return ATLAS_OK;
}

int done(const char *who, cudaError_t e)
{
    if (e == cudaSuccess) return ATLAS_OK;
    cudaGetLastError();
    return api_fail(ATLAS_ECUDA, "%s: %s", who, cudaGetErrorString(e));
}

// CTAs that share a unit's positions; the kernel is allowed its shared memory before
template <int NT, uint32_t W>
uint32_t attn_cluster(const FewArgs &a, int dev)
{
    const uint64_t units = (uint64_t)a.c.nseq * a.c.kv_heads * a.tiles;
    return cluster_of<attn_kernel<NT, W>>(dev, W * 32, sizeof(Smem<NT, W>), units, a.c.max_context);
}

template <int NT, uint32_t W>
cudaError_t launch_attn(const FewArgs &a, int dev, int sms, cudaStream_t stream)
{
    cudaError_t e = allow<attn_kernel<NT, W>>(dev, (int)kMaxSmem);
    if (e != cudaSuccess) return e;
    const uint32_t C = attn_cluster<NT, W>(a, dev);
    return launch(attn_kernel<NT, W>, dim3(C * a.tiles, a.c.kv_heads, a.c.nseq), W * 32, sizeof(Smem<NT, W>), C, a, sms, stream);
}

// The longest CTA's time in cycles (1.8 per ns) for more than eight rows, to be
// compared with the prompt form's: 18.5 per position of a tile of 16 rows (8
// warps), 9000 before and after. Rows: this form, the prompt form, in us: one
// sequence of 28 heads on 4, 500 positions, 112: 6.7, 15.3; 8000, 42 and 112:
// 15.4, 28 and 27, 30; 40 heads on 8, 30000, 20 and 65: 57, 81 and 107, 82; 8
// sequences of them, 2000, 20 and 35: 26, 32 and 51, 32; 16000: 166, 197 and 325,
// 197.
uint64_t few_cycles(const FewArgs &a, int dev)
{
    constexpr auto kernel = attn_kernel<2, 8>;
    if (allow<kernel>(dev, (int)kMaxSmem) != cudaSuccess) return 0;   // the launch will say so
    const uint64_t units = (uint64_t)a.c.nseq * a.c.kv_heads * a.tiles;
    const uint32_t C = attn_cluster<2, 8>(a, dev);
    const uint64_t at_once = std::max(clusters_at_once<kernel>(dev, C, 256, sizeof(Smem<2, 8>)), 1u);
    return (units + at_once - 1) / at_once * ((a.c.max_context + C - 1) / C) * 37 / 2 + 9000;
}

template <int NT>
cudaError_t launch_sparse(const FewArgs &a, int dev, int sms, cudaStream_t stream)
{
    const uint64_t units = (uint64_t)a.c.nseq * a.c.kv_heads * a.r.tokens * a.tiles;
    const size_t keys = sizeof(TokensSmem) + (size_t)kPickTokens * a.c.n_blocks * 8u;
    cudaError_t e;
    if (units > 2u * (uint32_t)sms && keys <= kMaxSmem) {
        if ((e = allow<choose_kernel>(dev, (int)kMaxSmem)) != cudaSuccess || (e = allow<chosen_kernel<NT>>(dev, (int)kMaxSmem)) != cudaSuccess)
            return e;
        e = launch(choose_kernel, dim3((a.r.tokens + kPickTokens - 1) / kPickTokens, a.c.kv_heads, a.c.nseq), 32 * kPickTokens, keys, 1,
                   static_cast<AttnArgs>(a), sms, stream);
        if (e != cudaSuccess) return e;
        return launch(chosen_kernel<NT>, dim3(a.r.tokens * a.tiles, a.c.kv_heads, a.c.nseq), 32 * kChosenWarps,
                      sizeof(Smem<NT, kChosenWarps>) + (size_t)a.n_sel * 4u, 1, a, sms, stream);
    }
    if ((e = allow<sparse_kernel<NT>>(dev, (int)kMaxSmem)) != cudaSuccess) return e;
    const size_t smem = sizeof(Smem<NT, kWarps>) + (size_t)a.n_sel * 4u;
    const uint32_t C = cluster_of<sparse_kernel<NT>>(dev, kThreads, smem, units,
                                                     std::max<uint64_t>((uint64_t)a.n_sel << a.c.block_log2, a.c.max_context / 8));
    return launch(sparse_kernel<NT>, dim3(C * a.r.tokens * a.tiles, a.c.kv_heads, a.c.nseq), kThreads,
                  smem, C, a, sms, stream);
}

}  // namespace
}  // namespace k8
}  // namespace atlas

using namespace atlas;
using namespace atlas::k8;

extern "C" int atlas_cuda_kv8_append(const AtlasKv8 *cache, uint32_t tokens, const uint32_t *d_pos0, const uint32_t *d_ntok,
                                     const float *d_k, const float *d_v, uint64_t ld, void *stream)
{
    const char *who = "kv8_append";
    AppendArgs a{};
    int dev, sms, rc = open_cache(who, cache, tokens, d_pos0, d_ntok, a.c, a.r, dev, sms);
    if (rc == ATLAS_OK) rc = check_rows(who, d_k, d_v, cache->kv_heads, ld, dev);
    if (rc != ATLAS_OK || !tokens) return rc;
    a.k = d_k;
    a.v = d_v;
    a.ld = ld;
    // the first row may be the last of its block
    const dim3 grid((tokens + 2 * cache->block - 2) / cache->block, 2 * cache->kv_heads, cache->nseq);
    auto *kernel = cache->block == 16   ? append_kernel<16>
                   : cache->block == 32 ? append_kernel<32>
                   : cache->block == 64 ? append_kernel<64>
                                        : append_kernel<128>;
    return done(who, launch(kernel, grid, 256, 0, 1, a, sms, (cudaStream_t)stream));
}

extern "C" int atlas_cuda_kv8_read(const AtlasKv8 *cache, uint32_t tokens, const uint32_t *d_pos0, const uint32_t *d_ntok,
                                   float *d_k, float *d_v, uint64_t ld, void *stream)
{
    const char *who = "kv8_read";
    ReadArgs a{};
    int dev, sms, rc = open_cache(who, cache, tokens, d_pos0, d_ntok, a.c, a.r, dev, sms);
    if (rc == ATLAS_OK) rc = check_rows(who, d_k, d_v, cache->kv_heads, ld, dev);
    if (rc != ATLAS_OK || !tokens) return rc;
    a.k = d_k;
    a.v = d_v;
    a.ld = ld;
    const dim3 grid((tokens + 8 * kReadRows - 1) / (8 * kReadRows), 2 * cache->kv_heads, cache->nseq);
    return done(who, launch(read_kernel, grid, 256, 0, 1, a, sms, (cudaStream_t)stream));
}

namespace {

int attn_args(const char *who, const AtlasKv8 *cache, uint32_t q_heads, uint32_t tokens, const uint32_t *d_pos0,
              const uint32_t *d_ntok, const float *d_q, uint64_t ldq, float *d_out, uint64_t ldo, AttnArgs &a, int &dev,
              int &sms)
{
    // a row of `out` may be written before another CTA has read its neighbours in `q`
    if (d_q && d_q == d_out) return api_fail(ATLAS_EINVAL, "%s: out must not be q", who);
    int rc = open_cache(who, cache, tokens, d_pos0, d_ntok, a.c, a.r, dev, sms);
    if (rc != ATLAS_OK) return rc;
    if (!q_heads || q_heads % cache->kv_heads || q_heads > 32768u || (uint64_t)q_heads * tokens > 0x3fffffffull)
        return api_fail(ATLAS_EINVAL, "%s: %u query heads over %u KV heads, %u tokens", who, q_heads, cache->kv_heads, tokens);
    if ((rc = check_rows(who, d_q, d_q, q_heads, ldq, dev)) != ATLAS_OK) return rc;
    if ((rc = check_rows(who, d_out, d_out, q_heads, ldo, dev)) != ATLAS_OK) return rc;
    a.q = d_q;
    a.out = d_out;
    a.ldq = ldq;
    a.ldo = ldo;
    a.q_heads = q_heads;
    a.group = q_heads / cache->kv_heads;
    a.group_inv = 1.000001f / (float)a.group;
    return ATLAS_OK;
}

}  // namespace

namespace {

// The form of a call: `one` (up to eight rows per KV head), else prompt or not; fills a.tiles for the few-rows forms
struct AttnForm {
    bool one, prompt;
    PromptCut cut;
};

AttnForm attn_form(FewArgs &a, int dev, int sms)
{
    const uint32_t rows = a.r.tokens * a.group;
    AttnForm f{rows <= 8, false, {}};
    a.tiles = f.one ? 1 : (rows + 15) / 16;
    if (!f.one) {
        f.cut = prompt_cut(a, dev, sms);
        f.prompt = f.cut.cycles < few_cycles(a, dev);
    }
    return f;
}

}  // namespace

extern "C" int atlas_cuda_kv8_attn_form(const AtlasKv8 *cache, uint32_t q_heads, uint32_t tokens, uint32_t *rows, uint32_t *ctas)
{
    const char *who = "kv8_attn_form";
    FewArgs a{};
    int dev, sms;
    if (!cache || !rows || !ctas) return api_fail(ATLAS_EINVAL, "%s: null argument", who);
    // rows and positions are not looked at: any memory that passes as theirs
    const int rc = attn_args(who, cache, q_heads, tokens, reinterpret_cast<const uint32_t *>(cache->k_scale), nullptr,
                             static_cast<const float *>(cache->k), 0, static_cast<float *>(cache->k) + 4, 0, a, dev, sms);
    if (rc != ATLAS_OK) return rc;
    if (!tokens) return api_fail(ATLAS_EINVAL, "%s: no tokens", who);
    const AttnForm f = attn_form(a, dev, sms);
    const cudaError_t e = allow<attn_kernel<1, 16>>(dev, (int)kMaxSmem);
    if (e != cudaSuccess) return done(who, e);
    *rows = f.one ? 8 : f.prompt ? 128 * f.cut.tiles : 16;
    *ctas = f.one ? attn_cluster<1, 16>(a, dev) : f.prompt ? f.cut.split : attn_cluster<2, 8>(a, dev);
    return ATLAS_OK;
}

extern "C" int atlas_cuda_kv8_attn(const AtlasKv8 *cache, uint32_t q_heads, uint32_t tokens, const uint32_t *d_pos0,
                                   const uint32_t *d_ntok, const float *d_q, uint64_t ldq, float *d_out, uint64_t ldo,
                                   void *stream)
{
    const char *who = "kv8_attn";
    FewArgs a{};
    int dev, sms;
    int rc = attn_args(who, cache, q_heads, tokens, d_pos0, d_ntok, d_q, ldq, d_out, ldo, a, dev, sms);
    if (rc != ATLAS_OK || !tokens) return rc;
    const AttnForm f = attn_form(a, dev, sms);
    if (f.prompt) return done(who, launch_prompt(a, f.cut, dev, sms, (cudaStream_t)stream));
    if ((rc = map_codes(who, a)) != ATLAS_OK) return rc;
    return done(who, f.one ? launch_attn<1, 16>(a, dev, sms, (cudaStream_t)stream)
                         : launch_attn<2, 8>(a, dev, sms, (cudaStream_t)stream));
}

extern "C" int atlas_cuda_kv8_attn_sparse(const AtlasKv8 *cache, uint32_t q_heads, uint32_t tokens, uint32_t n_sel,
                                          const uint32_t *d_pos0, const uint32_t *d_ntok, const float *d_q, uint64_t ldq,
                                          float *d_out, uint64_t ldo, int32_t *d_sel, void *stream)
{
    const char *who = "kv8_attn_sparse";
    FewArgs a{};
    int dev, sms;
    int rc = attn_args(who, cache, q_heads, tokens, d_pos0, d_ntok, d_q, ldq, d_out, ldo, a, dev, sms);
    if (rc != ATLAS_OK) return rc;
    if (!cache->k_sum) return api_fail(ATLAS_EINVAL, "%s: the cache has no k_sum", who);
    if (!d_sel || !aligned(d_sel, 4) || !on_device(d_sel, dev))
        return api_fail(ATLAS_EINVAL, "%s: sel must be 4-byte aligned memory of the current device", who);
    if (!n_sel || n_sel > 4096u) return api_fail(ATLAS_EINVAL, "%s: 1 to 4096 blocks per token, not %u", who, n_sel);
    if (a.c.n_blocks > kMaxBlocks)
        return api_fail(ATLAS_EINVAL, "%s: a cache of %u blocks: %u can be scored; take larger blocks", who, a.c.n_blocks,
                        kMaxBlocks);
    const bool one = a.group <= 8;
    a.tiles = one ? 1 : (a.group + 15) / 16;
    if ((uint64_t)tokens * a.tiles > 0x7ffffffull) return api_fail(ATLAS_EINVAL, "%s: too many rows", who);
    if (!tokens) return ATLAS_OK;
    if ((rc = map_codes(who, a)) != ATLAS_OK) return rc;
    a.n_sel = n_sel;
    a.sel = d_sel;
    return done(who, one ? launch_sparse<1>(a, dev, sms, (cudaStream_t)stream)
                         : launch_sparse<2>(a, dev, sms, (cudaStream_t)stream));
}
