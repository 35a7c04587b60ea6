// Causal attention of packed rows over a paged key-value cache.
#include "twm_attn_rows.h"

namespace twm {

template <bool E4M3> __global__ __launch_bounds__(64) void k_attn_prompt(const AttnArgs a)
{
    const int row = (int)blockIdx.x;
    int seq = -1;
    for (uint32_t s = 0; s < a.seqs.seqs; s++)
        if (a.seqs.starts[s] <= row && row < a.seqs.starts[s + 1]) seq = (int)s;
    if (seq < 0) return;
    attend_row<E4M3>(a, blockIdx.x, blockIdx.y, seq, a.seqs.lengths[seq] - (a.seqs.starts[seq + 1] - row));
}

hipError_t launch_attn_prompt(hipStream_t s, const AttnArgs &a)
{
    hipLaunchKernelGGL(a.kv.e4m3 ? k_attn_prompt<true> : k_attn_prompt<false>, dim3(a.rows, a.q_heads), dim3(64), 0, s, a);
    return hipGetLastError();
}

}  // namespace twm
