// What the kernels of the 8-bit KV cache share (kv8.cu, kv8_prompt.cu).
#pragma once
#include <atomic>
#include "common.cuh"
#include "kv8.h"

namespace atlas {
namespace k8 {
namespace {

// Every kernel here is launched with programmatic stream serialization: it
// may start while its predecessor drains, so it first waits for it. Inputs are
// then read through L2 (__ldcg, cp.async.cg): this SM's L1 may hold lines from
// before the predecessor wrote them.
// `early`: let the successor start at once (it waits in turn). Only where all
// of this grid fits on the device with room to spare: CTAs of a successor that
// take the first slots to fall free would crowd on a few SMs.
__device__ __forceinline__ void wait_predecessor(uint32_t early)
{
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (early) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

constexpr float kScoreScale = (float)(1.4426950408889634 / 11.313708498984761);   // log2(e) / sqrt(128)
constexpr float kLazy = 8.0f;                 // a running maximum is raised once a score passes it by this (base 2)
// Outputs are kept times this until the last division: the sum of 2^16 weights of 1 and any finite values stays finite,
// and V scales of 2^-100 and more keep all their bits.
constexpr float kOutUnit = 0x1p-16f;

__device__ __forceinline__ float ex2(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ float rcp(float x)
{
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ uint32_t h2_bits(float lo, float hi)
{
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
}

// Signed bytes 0 and 2 (odd: 1 and 3) of y as two binary16 numbers: 0x6400 | u
// is 1024 + u, and u = code + 128 with the sign bit flipped.
template <bool ODD>
__device__ __forceinline__ uint32_t codes_h2(uint32_t y)
{
    const uint32_t u = ((ODD ? y >> 8 : y) & 0x00ff00ffu) ^ 0x64806480u;
    const __half2 c = __hsub2(*reinterpret_cast<const __half2 *>(&u), __float2half2_rn(1152.0f));
    return *reinterpret_cast<const uint32_t *>(&c);
}

// Query rows of a tile: row i is head `rem + i` of token `tok`, counted on through the group (no division: the
// factor is 1 / group, a little high, and exact for rem + i < group + 256).
struct TileRows {
    uint32_t tok, rem, group;
    float inv;
    __device__ __forceinline__ uint2 at(uint32_t i) const   // (token, head of the group)
    {
        const uint32_t t = rem + i, q = (uint32_t)((float)t * inv);
        return make_uint2(tok + q, t - q * group);
    }
};

__device__ __forceinline__ uint32_t cluster_size()
{
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t cluster_rank()
{
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync()
{
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Two floats in one register pair, for the packed fp32 instructions
__device__ __forceinline__ uint64_t pair(float a, float b)
{
    uint64_t d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(a), "f"(b));
    return d;
}
__device__ __forceinline__ void unpair(uint64_t d, float &a, float &b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(d)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c)
{
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b)
{
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b)
{
    uint64_t d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}

// A launch that may overlap its predecessor's end (the kernels wait for it), in clusters of `cluster` CTAs along x.
template <class ARGS>
cudaError_t launch(void (*kernel)(ARGS), dim3 grid, uint32_t threads, size_t smem, uint32_t cluster, ARGS a, int sms,
                   cudaStream_t stream)
{
    a.early = (uint64_t)grid.x * grid.y * grid.z <= (uint64_t)sms;
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = cluster;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cfg.attrs = at;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, a);
}

// Lets a kernel take up to the device's shared memory and clusters of 16, once per device.
template <auto KERNEL>
cudaError_t allow(int dev, int bytes)
{
    static std::atomic<bool> done[64];
    if (done[dev].load(std::memory_order_acquire)) return cudaSuccess;
    cudaError_t e = cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(KERNEL, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e == cudaSuccess) done[dev].store(true, std::memory_order_release);
    return e;
}

constexpr size_t kMaxSmem = 232448;   // shared memory a CTA may have
constexpr uint32_t kMaxCluster = 16;

// How many clusters of `c` CTAs of a kernel are on the device at once; asked once per device and size, for shared memory
// that leaves an SM room for two CTAs (228 KB, of which each takes 1 KB more) and that does not.
template <auto KERNEL>
uint32_t clusters_at_once(int dev, uint32_t c, uint32_t threads, size_t smem)
{
    static std::atomic<uint32_t> known[2][64][kMaxCluster + 1];   // + 1; 0: not asked yet
    std::atomic<uint32_t> &entry = known[smem > 113 * 1024][dev][c];
    uint32_t n = entry.load(std::memory_order_relaxed);
    if (!n) {
        cudaLaunchConfig_t cfg{};
        cudaLaunchAttribute at;
        at.id = cudaLaunchAttributeClusterDimension;
        at.val.clusterDim.x = c;
        at.val.clusterDim.y = at.val.clusterDim.z = 1;
        cfg.gridDim = dim3(c);
        cfg.blockDim = dim3(threads);
        cfg.dynamicSmemBytes = smem;
        cfg.attrs = &at;
        cfg.numAttrs = 1;
        int most = 0;
        if (cudaOccupancyMaxActiveClusters(&most, KERNEL, &cfg) != cudaSuccess) cudaGetLastError();
        n = (uint32_t)std::max(most, 0) + 1;
        entry.store(n, std::memory_order_relaxed);
    }
    return n - 1;
}

}  // namespace
}  // namespace k8
}  // namespace atlas
