// Activation rows in 8-bit floating point (e4m3, one f32 scale per row and 128 columns): the residual's addition and the
// root-mean-square norm, the gate of fused gate/up rows, or the rows as they are.
//
//   scale[row][b] = max(max |y| over the block, 1e-30) / 448,   q = e4m3(y / scale)   (448: the largest e4m3 value)
//
// A block that holds an infinity or a NaN gets a NaN scale (and NaN codes), so that what is multiplied with it is NaN, as it
// would be with the f32 values.
//
// Sixteen lanes hold a block, eight columns each: the largest magnitude is found by four DPP steps within those lanes, on the
// bit patterns (which order as the magnitudes do and put NaN above infinity above all numbers).
#include "twm_device.h"

namespace twm {

namespace {

constexpr uint32_t kFp8Each = 8;       // columns per lane
constexpr float kFp8Max = 448.0f;
constexpr float kFp8LeastAmax = 1e-30f;  // (448 / amax stays finite, a block of zeros gets codes of zero)

// the largest of sixteen lanes' values, in each of them
__device__ __forceinline__ uint32_t max_of_16(uint32_t v)
{
#define TWM_MAX_STEP(N) v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x120 + N, 0xf, 0xf, true))   // row_ror:N
    TWM_MAX_STEP(8);
    TWM_MAX_STEP(4);
    TWM_MAX_STEP(2);
    TWM_MAX_STEP(1);
#undef TWM_MAX_STEP
    return v;
}

// Columns col .. col + 7 of a row that ends at `cols`; zeros behind the end.  VEC: eight columns are 16 (f16) or 32 (f32)
// aligned bytes, wholly inside the row or outside.
template <bool F16, bool VEC> __device__ __forceinline__ void load_8(float (&v)[8], const void *row, uint32_t col, uint32_t cols)
{
    if constexpr (VEC) {
        if (col < cols) {
            if constexpr (F16) {
                const half8 h = *(const half8 *)((const _Float16 *)row + col);
#pragma unroll
                for (int j = 0; j < 8; j++) v[j] = (float)h[j];
            } else {
                const float4v a = *(const float4v *)((const float *)row + col), b = *(const float4v *)((const float *)row + col + 4);
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    v[j] = a[j];
                    v[4 + j] = b[j];
                }
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++) v[j] = 0.f;
        }
    } else {
#pragma unroll
        for (uint32_t j = 0; j < 8; j++) {
            v[j] = 0.f;
            if (col + j < cols) v[j] = F16 ? (float)((const _Float16 *)row)[col + j] : ((const float *)row)[col + j];
        }
    }
}

template <bool VEC> __device__ __forceinline__ void store_f32_8(float *row, uint32_t col, uint32_t cols, const float (&v)[8])
{
    if constexpr (VEC) {
        if (col < cols) {
            *(float4v *)(row + col) = float4v{v[0], v[1], v[2], v[3]};
            *(float4v *)(row + col + 4) = float4v{v[4], v[5], v[6], v[7]};
        }
    } else {
#pragma unroll
        for (uint32_t j = 0; j < 8; j++)
            if (col + j < cols) row[col + j] = v[j];
    }
}

template <bool VEC> __device__ __forceinline__ void store_f16_8(_Float16 *row, uint32_t col, uint32_t cols, const float (&v)[8])
{
    if constexpr (VEC) {
        half8 h;
#pragma unroll
        for (int j = 0; j < 8; j++) h[j] = (_Float16)v[j];
        if (col < cols) *(half8 *)(row + col) = h;
    } else {
#pragma unroll
        for (uint32_t j = 0; j < 8; j++)
            if (col + j < cols) row[col + j] = (_Float16)v[j];
    }
}

// The codes of eight values whose block spans this lane's sixteen, and from its first lane the block's scale (null where the
// block lies behind the row's end).  q: column 0 of the row.
template <bool VEC> __device__ __forceinline__ void store_codes(uint8_t *q, float *scale, uint32_t col, uint32_t cols, const float (&v)[8])
{
    uint32_t bits = 0;
#pragma unroll
    for (int j = 0; j < 8; j++) bits = max(bits, __float_as_uint(v[j]) & 0x7FFFFFFFu);
    bits = max_of_16(bits);
    float amax = __uint_as_float(bits);
    // (fmaxf would drop a NaN)
    amax = bits >= 0x7F800000u ? __uint_as_float(0x7FC00000u) : amax < kFp8LeastAmax ? kFp8LeastAmax : amax;
    const float to_code = kFp8Max / amax;
    if (scale && (col & 127u) == 0) *scale = amax / kFp8Max;
    // (|v| * to_code is at most 448 and a rounding, which the conversion rounds to 448)
    int lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[0] * to_code, v[1] * to_code, 0, false);
    lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[2] * to_code, v[3] * to_code, lo, true);
    int hi = __builtin_amdgcn_cvt_pk_fp8_f32(v[4] * to_code, v[5] * to_code, 0, false);
    hi = __builtin_amdgcn_cvt_pk_fp8_f32(v[6] * to_code, v[7] * to_code, hi, true);
    if constexpr (VEC) {
        if (col < cols) *(uint2v *)(q + col) = uint2v{(uint32_t)lo, (uint32_t)hi};
    } else {
#pragma unroll
        for (uint32_t j = 0; j < 8; j++)
            if (col + j < cols) q[col + j] = (uint8_t)((uint32_t)(j < 4 ? lo : hi) >> (8 * (j & 3u)));
    }
}

}  // namespace

// Sixteen lanes per (row, block).  GATE: y = act(gate) * up of a row of 2 * cols columns, gate columns then up columns or in the
// paired order; otherwise y = x.
template <bool F16, bool VEC, bool GATE>
__global__ __launch_bounds__(256) void k_fp8_rows(const void *__restrict__ in, uint32_t cols, uint32_t blocks, uint64_t items, uint32_t act,
                                                  uint32_t paired, uint8_t *__restrict__ q, float *__restrict__ scales)
{
    const uint64_t item = ((uint64_t)blockIdx.x * 256u + threadIdx.x) >> 4;
    if (item >= items) return;   // (all sixteen lanes of an item)
    const uint64_t row = item / blocks;
    const uint32_t block = (uint32_t)(item - row * blocks), col = block * 128u + (threadIdx.x & 15u) * kFp8Each;
    constexpr size_t kEach = F16 ? 2 : 4;
    const char *src = (const char *)in + (size_t)row * cols * (GATE ? 2 * kEach : kEach);
    float v[8];
    if constexpr (GATE) {
        // (a run of 32 paired columns is whole: eight columns never cross into the up half)
        const uint32_t g_col = paired ? paired_col(col) : col, u_col = paired ? g_col + kPairWidth : col + cols;
        const bool in_row = col < cols;
        float g[8], u[8];
        load_8<F16, VEC>(g, src, in_row ? g_col : 2u * cols, paired ? 2u * cols : cols);
        load_8<F16, VEC>(u, src, in_row ? u_col : 2u * cols, 2u * cols);
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = gated_mul(act, g[j], u[j]);
    } else {
        load_8<F16, VEC>(v, src, col, cols);
    }
    store_codes<VEC>(q + (size_t)row * cols, scales + item, col, cols, v);
}

// A workgroup per row.  s = x (+ residual) stays in registers up to 8 * THREADS * HELD columns; a longer row is read again for its
// second pass.  sum: where s goes, or null; it may be the residual itself, whose elements are read by the lane that writes them.
template <bool F16, bool VEC, uint32_t THREADS, uint32_t HELD>
__global__ __launch_bounds__(THREADS) void k_fp8_norm(const void *x, const float *residual, const float *__restrict__ weight, float eps,
                                                      uint32_t cols, uint32_t blocks, float *sum, uint8_t *__restrict__ q,
                                                      float *__restrict__ scales, _Float16 *__restrict__ normed)
{
    constexpr uint32_t kWaves = THREADS / 64, kSpan = THREADS * kFp8Each;
    __shared__ double parts[kWaves];
    const size_t row = blockIdx.x;
    const void *x_row = (const char *)x + row * cols * (F16 ? 2 : 4);
    const float *r_row = residual ? residual + row * cols : nullptr;
    float *s_row = sum ? sum + row * cols : nullptr;
    const uint32_t col0 = threadIdx.x * kFp8Each;

    float v[HELD][8];
    double squares = 0.0;   // (a lane's eight in 32 bits, their sum over a row of any length in 64)
    auto take = [&](float (&s)[8], uint32_t col) {
        load_8<F16, VEC>(s, x_row, col, cols);
        if (r_row) {
            float r[8];
            load_8<false, VEC>(r, r_row, col, cols);
#pragma unroll
            for (int j = 0; j < 8; j++) s[j] += r[j];
        }
    };
    auto add = [&](const float (&s)[8]) {
        float part = 0.f;
#pragma unroll
        for (int j = 0; j < 8; j++) part += s[j] * s[j];
        squares += (double)part;
    };
#pragma unroll
    for (uint32_t h = 0; h < HELD; h++) take(v[h], col0 + h * kSpan);
#pragma unroll
    for (uint32_t h = 0; h < HELD; h++) {
        add(v[h]);
        if (s_row) store_f32_8<VEC>(s_row, col0 + h * kSpan, cols, v[h]);
    }
    for (uint64_t at = (uint64_t)kSpan * HELD; at < cols; at += kSpan) {
        const uint64_t col = at + col0;
        if (col >= cols) break;
        float s[8];
        take(s, (uint32_t)col);
        add(s);
        if (s_row) store_f32_8<VEC>(s_row, (uint32_t)col, cols, s);
    }
#pragma unroll
    for (int step = 32; step; step >>= 1) squares += __shfl_xor(squares, step);
    if ((threadIdx.x & 63u) == 0) parts[threadIdx.x >> 6] = squares;
    __syncthreads();
    squares = 0.0;
#pragma unroll
    for (uint32_t w = 0; w < kWaves; w++) squares += parts[w];
    const float scale = 1.0f / sqrtf((float)(squares / cols) + eps);

    // (whole groups of sixteen lanes: the columns of a block behind the row's end count as zeros)
    auto finish = [&](float (&s)[8], uint64_t col) {
        if (col >= (uint64_t)blocks * 128u) return;
        float w[8];
        load_8<false, VEC>(w, weight, (uint32_t)col, cols);
#pragma unroll
        for (int j = 0; j < 8; j++) s[j] = s[j] * scale * w[j];
        if (normed) store_f16_8<VEC>(normed + row * cols, (uint32_t)col, cols, s);
        store_codes<VEC>(q + row * cols, scales + row * blocks + (uint32_t)(col >> 7), (uint32_t)col, cols, s);
    };
#pragma unroll
    for (uint32_t h = 0; h < HELD; h++) finish(v[h], col0 + h * kSpan);
    for (uint64_t at = (uint64_t)kSpan * HELD; at < cols; at += kSpan) {
        const uint64_t col = at + col0;
        if (col >= (uint64_t)blocks * 128u) break;
        float s[8];
        // (what this lane wrote, where the residual may have been written over)
        if (s_row) load_8<false, VEC>(s, s_row, (uint32_t)col, cols);
        else take(s, (uint32_t)col);
        finish(s, col);
    }
}

hipError_t launch_fp8_rows(hipStream_t s, const void *in, bool f16, uint32_t rows, uint32_t cols, int gate, bool paired, uint8_t *q, float *scales)
{
    if (rows == 0 || cols == 0) return hipSuccess;
    const uint32_t blocks = (cols + 127u) / 128u;
    const uint64_t items = (uint64_t)rows * blocks;
    const bool vec = cols % 8 == 0 && ((uintptr_t)in & 15) == 0 && ((uintptr_t)q & 7) == 0;
    auto kernel = gate ? (f16 ? (vec ? k_fp8_rows<true, true, true> : k_fp8_rows<true, false, true>) : (vec ? k_fp8_rows<false, true, true> : k_fp8_rows<false, false, true>))
                       : (f16 ? (vec ? k_fp8_rows<true, true, false> : k_fp8_rows<true, false, false>) : (vec ? k_fp8_rows<false, true, false> : k_fp8_rows<false, false, false>));
    hipLaunchKernelGGL(kernel, dim3((unsigned)((items + 15) / 16)), dim3(256), 0, s, in, cols, blocks, items, gate == 1 ? 1u : 0u, paired ? 1u : 0u, q, scales);
    return hipGetLastError();
}

hipError_t launch_fp8_norm(hipStream_t s, const void *x, bool f16, const float *residual, const float *weight, float eps, uint32_t rows,
                           uint32_t cols, float *sum, uint8_t *q, float *scales, uint16_t *normed)
{
    if (rows == 0 || cols == 0) return hipSuccess;
    const uint32_t blocks = (cols + 127u) / 128u;
    const uintptr_t quads = (uintptr_t)x | (uintptr_t)residual | (uintptr_t)weight | (uintptr_t)sum | (uintptr_t)normed;
    const bool vec = cols % 8 == 0 && (quads & 15) == 0 && ((uintptr_t)q & 7) == 0;
    auto kernel = f16 ? (vec ? k_fp8_norm<true, true, 256, 2> : k_fp8_norm<true, false, 256, 2>) : (vec ? k_fp8_norm<false, true, 256, 2> : k_fp8_norm<false, false, 256, 2>);
    hipLaunchKernelGGL(kernel, dim3(rows), dim3(256), 0, s, x, residual, weight, eps, cols, blocks, sum, q, scales, (_Float16 *)normed);
    return hipGetLastError();
}

}  // namespace twm
