// Attention of single query rows, a wave each: the simplest form.
#pragma once
#include "twm_kv.h"

namespace twm {

__device__ __forceinline__ float e4m3_value(uint8_t code) { return __builtin_amdgcn_cvt_f32_fp8((int)code, 0); }

// Sixty-four tokens at a time: a lane's token's score, the running maximum and sum, then the values, a lane's columns over the tokens.
template <bool E4M3> __device__ __forceinline__ void attend_row(const AttnArgs &a, uint32_t row, uint32_t head, int seq, int position)
{
    const uint32_t lane = threadIdx.x, dim = a.kv.dim, kv_head = head / a.group, page_tokens = 1u << a.kv.page_shift;
    const int capacity = (int)(a.seqs.table_stride << a.kv.page_shift), end = min(position + 1, capacity);
    const int begin = a.window ? max(0, position + 1 - (int)a.window) : 0;   // (position is -1 or more rows before the first token)
    const float k_scale = (a.kv.k_scales ? a.kv.k_scales[kv_head] : 1.0f) * a.scale * 1.44269504f, v_scale = a.kv.v_scales ? a.kv.v_scales[kv_head] : 1.0f;
    const _Float16 *q = a.q + (size_t)row * a.q_stride + head * dim;
    float top = -INFINITY, total = 0.f, sum[4] = {};
    for (int t0 = begin; t0 < end; t0 += 64) {
        const int t = t0 + (int)lane;
        int page = t < end ? a.seqs.tables[(size_t)seq * a.seqs.table_stride + ((uint32_t)t >> a.kv.page_shift)] : -1;
        const bool seen = (uint32_t)page < a.kv.pages;
        float score = -INFINITY;
        size_t at = 0;
        if (seen) {
            at = kv_chunk(a.kv, (uint32_t)page, kv_head) + (size_t)((uint32_t)t & (page_tokens - 1u)) * dim;
            float dot = 0.f;
            for (uint32_t d = 0; d < dim; d++)
                dot = fmaf((float)q[d], E4M3 ? e4m3_value(((const uint8_t *)a.kv.k)[at + d]) : (float)((const _Float16 *)a.kv.k)[at + d], dot);
            score = dot * k_scale;
        }
        float most = score;
        for (int i = 1; i < 64; i *= 2) most = fmaxf(most, __shfl_xor(most, i));
        const float next = fmaxf(top, most), base = next == -INFINITY ? 0.f : next, keep = exp2f(top - base);
        float p = seen ? exp2f(score - base) : 0.f;
        top = next;
        total = total * keep;
        for (uint32_t c = 0; c < 4; c++) sum[c] *= keep;
        for (int j = 0; j < 64; j++) {
            if (!__shfl((int)seen, j)) continue;
            const float weight = __shfl(p, j);
            const size_t from = (size_t)__shfl((long long)at, j);
            total += weight;
            for (uint32_t c = 0; c < 4; c++)
                if (64u * c < dim)
                    sum[c] = fmaf(weight, E4M3 ? e4m3_value(((const uint8_t *)a.kv.v)[from + 64u * c + lane]) : (float)((const _Float16 *)a.kv.v)[from + 64u * c + lane], sum[c]);
        }
    }
    for (uint32_t c = 0; c < 4; c++)
        if (64u * c < dim) a.out[(size_t)row * a.out_stride + head * dim + 64u * c + lane] = (_Float16)(total != 0.f ? sum[c] / total * v_scale : 0.f);
}

}  // namespace twm
