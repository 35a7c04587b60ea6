// What the kernels of the paged key-value cache share.
#pragma once
#include "twm_device.h"

namespace twm {

// Rows of queries and of fused projections begin at any element; the memory takes vectors there too
typedef half8 half8_any __attribute__((aligned(2)));
typedef float4v float4v_any __attribute__((aligned(4)));

// The first element of (page, head) in a cache's array
__device__ __forceinline__ size_t kv_chunk(const KvView &kv, uint32_t page, uint32_t head)
{
    return (((size_t)page * kv.kv_heads + head) << kv.page_shift) * kv.dim;
}

}  // namespace twm
