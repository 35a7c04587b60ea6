// Attention of one new token per sequence over a paged key-value cache.
#include "twm_attn_rows.h"

namespace twm {

template <bool E4M3> __global__ __launch_bounds__(64) void k_attn_decode(const AttnArgs a)
{
    attend_row<E4M3>(a, blockIdx.x, blockIdx.y, (int)blockIdx.x, a.seqs.lengths[blockIdx.x] - 1);
}

hipError_t launch_attn_decode(hipStream_t s, const AttnArgs &a, void *, size_t)
{
    hipLaunchKernelGGL(a.kv.e4m3 ? k_attn_decode<true> : k_attn_decode<false>, dim3(a.rows, a.q_heads), dim3(64), 0, s, a);
    return hipGetLastError();
}

}  // namespace twm
