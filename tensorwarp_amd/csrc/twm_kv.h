// What the kernels of the paged key-value cache share.
#pragma once
#include "twm_device.h"

#include <cfloat>

namespace twm {

// Rows of queries and of fused projections begin at any element; the memory takes vectors there too
typedef half8 half8_any __attribute__((aligned(2)));
typedef float4v float4v_any __attribute__((aligned(4)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef half4 half4_any __attribute__((aligned(2)));
typedef short short4v __attribute__((ext_vector_type(4)));
#define TWM_LDS(T) __attribute__((address_space(3))) T

// The first element of (page, head) in a cache's array
__device__ __forceinline__ size_t kv_chunk(const KvView &kv, uint32_t page, uint32_t head)
{
    return (((size_t)page * kv.kv_heads + head) << kv.page_shift) * kv.dim;
}

// What a difference of scores is multiplied by, to base 2.  The product of three numbers passes what f32 holds although the two on the host's side
// are finite: it is made in 64 bits, and kept within f32's range, where no weight differs from what lies beyond it (at the largest, the least
// difference of two f16 rows' scores is 2^80 of an exponent, at the least the largest one 2^-80), and where it times -infinity is that.
__device__ __forceinline__ float exponent_factor(const KvView &kv, float scale, uint32_t head)
{
    const float c = (float)((double)scale * 1.4426950408889634 * (kv.k_scales ? (double)kv.k_scales[head] : 1.0));
    return c > FLT_MAX ? FLT_MAX : c < FLT_MIN ? FLT_MIN : c;   // (a NaN stays)
}

// eight codes as f16 (exact)
__device__ __forceinline__ half8 to_f16(unsigned lo, unsigned hi)
{
    const half2v a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)lo, 1.0f, false), b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)lo, 1.0f, true);
    const half2v c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)hi, 1.0f, false), d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)hi, 1.0f, true);
    return half8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// What sums are multiplied by where the score that they refer to becomes another: 2^(c (from - to)).  Never 0, so that an infinite sum stays one; 2^-126
// of what is finite counts for nothing, nor does that of nothing, where from is -infinity.
__device__ __forceinline__ float shrink(float from, float to, float c) { return __builtin_amdgcn_exp2f(fmaxf((from - to) * c, -126.0f)); }

// v of this lane and of those before it, added up (by moves within rows of sixteen lanes, then across them)
__device__ __forceinline__ uint32_t wave_sum_up_to(uint32_t v)
{
#define TWM_ADD_STEP(CONTROL, ROWS) v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CONTROL, ROWS, 0xf, false)
    TWM_ADD_STEP(0x111, 0xf);   // row_shr:1, 2, 4, 8
    TWM_ADD_STEP(0x112, 0xf);
    TWM_ADD_STEP(0x114, 0xf);
    TWM_ADD_STEP(0x118, 0xf);
    TWM_ADD_STEP(0x142, 0xa);   // row_bcast:15 to rows 1 and 3, row_bcast:31 to rows 2 and 3
    TWM_ADD_STEP(0x143, 0xc);
#undef TWM_ADD_STEP
    return v;
}

// Division by a number that a launch knows: n / d for n below 2^31 as (n * factor) >> shift, factor = ceil(2^shift / d) with
// shift = 31 + ceil(log2 d).  (factor d is less than 2^shift + d, so that n factor / 2^shift is less than n / d + n / 2^shift, and the
// last term is at most 1 / d.)
struct Divisor {
    uint32_t d, factor, shift;
    explicit __host__ Divisor(uint32_t by) : d(by)
    {
        uint32_t log = 0;
        while ((1ull << log) < by) log++;
        shift = 31 + log;
        factor = (uint32_t)(((1ull << shift) + by - 1) / by);
    }
    Divisor() = default;
    __device__ __forceinline__ uint32_t operator()(uint32_t n) const { return (uint32_t)((uint64_t)n * factor >> shift); }
};

}  // namespace twm
