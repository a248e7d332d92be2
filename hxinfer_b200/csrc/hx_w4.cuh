// hx_w4.cuh — what the 4-bit linear kernels share: the shape of a packed
// weight, the product's arguments and the conversion's steps.  The layout is
// described in w4_linear.cu.
#pragma once

#include "hx_common.cuh"

namespace hx {

constexpr int kW4Rows = 16;
constexpr int kW4Unit = 128;   // inputs one warp takes at a time: two 64-input blocks

struct W4Shape {
    int out, in, group;
    int tiles, units;           // of the padded weight
    int record;                 // bytes of a unit of a row tile
    size_t bytes;
};

struct W4Params {
    W4Shape s;
    const __half* x;
    const char* packed;
    const __half* bias;
    void* y;
    int n, y_f32;
    int* status;
};

__device__ __forceinline__ uint32_t lop_and_or(uint32_t a, uint32_t mask, uint32_t orv)
{
    uint32_t d;
    asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(d) : "r"(a), "r"(mask), "r"(orv));  // (a & mask) | orv
    return d;
}

__device__ __forceinline__ uint32_t h2_sub(uint32_t a, uint32_t b)
{
    const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
}

// Untiled bulk copy global -> shared (16-byte aligned, a multiple of 16 bytes).
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar, uint64_t policy)
{
    asm volatile(
        "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1], %2, [%3], %4;" ::"r"(
            smem_u32(dst)),
        "l"(src), "r"(bytes), "r"(smem_u32(bar)), "l"(policy)
        : "memory");
}

// The product on the 5th-generation tensor cores (w4_tile.cu).
int launch_w4_tile(const W4Params& p, bool zeros, cudaStream_t stream);

}  // namespace hx
