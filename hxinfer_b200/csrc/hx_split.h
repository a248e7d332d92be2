// hx_split.h — an even cut of a list of items into n consecutive parts, for
// host and device.
#pragma once

#include <stdint.h>

#ifdef __CUDACC__
#define HX_HD __host__ __device__ __forceinline__
#else
#define HX_HD static inline
#endif

namespace hx {

// Part c of n holds items [first(c), first(c + 1)), first(c) = items c / n.
// The products fit 32 bits in most calls, where the division is the short one.
HX_HD int64_t split_first(int64_t items, int n, int c)
{
    const int64_t x = items * c;
    return x >> 32 ? x / n : (int64_t)((uint32_t)x / (uint32_t)n);
}

// The part that holds an item: the largest k with items k / n <= item, i.e.
// items k < (item + 1) n.
HX_HD int split_owner(int64_t items, int n, int64_t item)
{
    const int64_t x = (item + 1) * n - 1;
    return (int)((x | items) >> 32 ? x / items : (int64_t)((uint32_t)x / (uint32_t)items));
}

}  // namespace hx
