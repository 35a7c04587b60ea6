// Activation rows in 8-bit floating point (e4m3, one f32 scale per row and 128 columns): the residual's addition and the
// root-mean-square norm, the gate of fused gate/up rows, or the rows as they are.
//
//   scale[row][b] = max(max |y| over the block, 1e-30) / 448,   q = e4m3(y / scale)   (448: the largest e4m3 value; both quotients in f32)
//
// A block that holds an infinity or a NaN gets a NaN scale (and NaN codes), so that what is multiplied with it is NaN, as it
// would be with the f32 values.
//
// Sixteen lanes hold a block, eight columns each: the largest magnitude is found by four DPP steps within those lanes, on the
// bit patterns (which order as the magnitudes do and put NaN above infinity above all numbers).
#include "twm_device.h"
#include "twm_e4m3.h"
#include "twm_slices.h"

#include <type_traits>

namespace twm {

namespace {

constexpr uint32_t kFp8Each = 8;       // columns per lane
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

// act(g) * u with silu(g) = g / (1 + e^-g), or gelu's tanh form, g / (1 + e^-2z) with z = sqrt(2 / pi) (g + 0.044715 g^3) (which is
// 0.5 g (1 + tanh z) without the difference of nearly equal numbers).  e^-x = 2^t with t = -x log2(e) in two f32 terms and the
// hardware's exponential and reciprocal, each within a unit in the last place: silu is within 2^-21 of itself.  gelu's t is g times a
// polynomial of g^2 whose roundings -- of g^2, of the polynomial, of its constants -- count 2z times over: within 2^-21 + 2^-22.7 |2z|
// (measured 2^-19.6 at g = -5 and 2^-17 at g = -9, where gelu is 5e-8 and 2e-29 of g).  The polynomial in 64 bits would keep it at
// 2^-21 and takes a 2048 x 11008 f16 gate from 25.6 to 27.8 us.  (GATE: 1 gelu, 2 silu; g above far_gate.)
template <int GATE, bool F16> __device__ __forceinline__ float gate_rows(float g, float u)
{
    float t, low;   // (finite for any f16 g, and for an f32 one between the limits)
    if constexpr (GATE == 1) {
        constexpr double c = -1.5957691216057308 * 1.4426950408889634;   // -2 sqrt(2 / pi) log2(e)
        const float x = F16 ? g : __builtin_amdgcn_fmed3f(g, -9.0f, 100.0f), p = fmaf(x * x, (float)(0.044715 * c), (float)c);
        t = x * p;
        low = fmaf(x, p, -t);
    } else {
        const float x = F16 ? g : __builtin_amdgcn_fmed3f(g, -80.0f, 1e4f);
        t = x * -1.44269502f;
        low = fmaf(x, -1.92596303e-8f, fmaf(x, -1.44269502f, -t));
    }
    const float e = __builtin_amdgcn_exp2f(t);
    // (act(g) first: it is small where g u may be beyond f32)
    return g * __builtin_amdgcn_rcpf(fmaf(e, low * 0.693147182f, e) + 1.0f) * u;
}

// Below this the gate is g e^x and less than 2^-95 of g: 1 / (1 + e^-x) leaves what f32 holds at x = -87, act(g) soon after, while its
// product with u need not.  There the product is taken in 64 bits, 2^-t as a power of two and the rest.  (One comparison for eight
// gates, and t without clamps in f16: 2048 x 11008 rows 25.2 us, gelu 25.6; clamped and without this 25.5 and 26.0.)
template <int GATE> constexpr float far_gate = GATE == 1 ? -9.0f : -80.0f;
template <int GATE> __device__ __forceinline__ float gate_far(float g, float u)
{
    const double d = g, x = GATE == 1 ? 1.5957691216057308 * (d + 0.044715 * d * d * d) : d;
    const double t = fmax(x * 1.4426950408889634, -1000.0), whole = rint(t);   // (g u e^-693 is nothing for any g and u)
    return (float)(d * u * ldexp((double)__builtin_amdgcn_exp2f((float)(t - whole)), (int)whole));
}

// Rows begin where the ones before them end, on any element's boundary; the memory takes vectors there too (2048 x 11007 f16 gate
// 64.6 us element by element, 27.6 so; 2048 x 4095 f16 norm with every output 68.4 and 31.2)
typedef half8 half8_any __attribute__((aligned(2)));
typedef float4v float4v_any __attribute__((aligned(4)));
typedef uint2v uint2v_any __attribute__((aligned(1)));

// Columns col .. col + 7 of a row that ends at `cols`; zeros behind the end.  WHOLE: the eight are wholly inside the row or outside
// (cols is a multiple of eight).
template <bool F16, bool WHOLE> __device__ __forceinline__ void load_8(float (&v)[8], const void *row, uint32_t col, uint32_t cols)
{
    if (WHOLE ? col < cols : (uint64_t)col + 8u <= cols) {
        if constexpr (F16) {
            const half8 h = *(const half8_any *)((const _Float16 *)row + col);
#pragma unroll
            for (int j = 0; j < 8; j++) v[j] = (float)h[j];
        } else {
            const float4v a = *(const float4v_any *)((const float *)row + col), b = *(const float4v_any *)((const float *)row + col + 4);
#pragma unroll
            for (int j = 0; j < 4; j++) {
                v[j] = a[j];
                v[4 + j] = b[j];
            }
        }
        return;
    }
#pragma unroll
    for (uint32_t j = 0; j < 8; j++) {
        v[j] = 0.f;
        if (!WHOLE && col + j < cols) v[j] = F16 ? (float)((const _Float16 *)row)[col + j] : ((const float *)row)[col + j];
    }
}

template <bool WHOLE> __device__ __forceinline__ void store_f32_8(float *row, uint32_t col, uint32_t cols, const float (&v)[8])
{
    if (WHOLE ? col < cols : (uint64_t)col + 8u <= cols) {
        *(float4v_any *)(row + col) = float4v{v[0], v[1], v[2], v[3]};
        *(float4v_any *)(row + col + 4) = float4v{v[4], v[5], v[6], v[7]};
    } else if (!WHOLE) {
#pragma unroll
        for (uint32_t j = 0; j < 8; j++)
            if (col + j < cols) row[col + j] = v[j];
    }
}

template <bool WHOLE> __device__ __forceinline__ void store_f16_8(_Float16 *row, uint32_t col, uint32_t cols, const float (&v)[8])
{
    if (WHOLE ? col < cols : (uint64_t)col + 8u <= cols) {
        half8 h;
#pragma unroll
        for (int j = 0; j < 8; j++) h[j] = (_Float16)v[j];
        *(half8_any *)(row + col) = h;
    } else if (!WHOLE) {
#pragma unroll
        for (uint32_t j = 0; j < 8; j++)
            if (col + j < cols) row[col + j] = (_Float16)v[j];
    }
}

// The codes of eight values whose block spans this lane's sixteen, and from its first lane the block's scale (null where the
// block lies behind the row's end).  q: column 0 of the row.
template <bool WHOLE> __device__ __forceinline__ void store_codes(uint8_t *q, float *scale, uint32_t col, uint32_t cols, const float (&v)[8])
{
    uint32_t bits = 0;
#pragma unroll
    for (int j = 0; j < 8; j++) bits = max(bits, __float_as_uint(v[j]) & 0x7FFFFFFFu);
    bits = max_of_16(bits);
    float amax = __uint_as_float(bits);
    // (fmaxf would drop a NaN)
    amax = bits >= 0x7F800000u ? __uint_as_float(0x7FC00000u) : amax < kFp8LeastAmax ? kFp8LeastAmax : amax;
    const float block_scale = amax / kFp8Max;
    if (scale && (col & 127u) == 0) *scale = block_scale;
    const float inverse = kFp8Max / amax;   // (not 1 / block_scale, which would wait for it: 1 x 896 norm's kernel 3.1 us, so 3.3)
    // (2048 x 11008 f16 gate 25.2 us, with eight divisions 27.8, with the product with the inverse alone 24.6)
    float c[8];
    if (__builtin_expect(block_scale < kFp8LeastExact, 0)) {
#pragma unroll
        for (int j = 0; j < 8; j++) c[j] = v[j] / block_scale;
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++) c[j] = units_of(v[j], block_scale, inverse);
    }
    // (at most 448 and a rounding, which the conversion rounds to 448)
    int lo = __builtin_amdgcn_cvt_pk_fp8_f32(c[0], c[1], 0, false);
    lo = __builtin_amdgcn_cvt_pk_fp8_f32(c[2], c[3], lo, true);
    int hi = __builtin_amdgcn_cvt_pk_fp8_f32(c[4], c[5], 0, false);
    hi = __builtin_amdgcn_cvt_pk_fp8_f32(c[6], c[7], hi, true);
    if (WHOLE ? col < cols : (uint64_t)col + 8u <= cols) {
        *(uint2v_any *)(q + col) = uint2v{(uint32_t)lo, (uint32_t)hi};
    } else if (!WHOLE) {
#pragma unroll
        for (uint32_t j = 0; j < 8; j++)
            if (col + j < cols) q[col + j] = (uint8_t)((uint32_t)(j < 4 ? lo : hi) >> (8 * (j & 3u)));
    }
}

}  // namespace

// Sixteen lanes per (row, block).  GATE 1, 2: y = gelu(gate) * up, silu(gate) * up of a row of 2 * cols columns, gate columns then up
// columns or in the paired order; 0: y = x.  Bound: the rows' way through memory.
template <bool F16, bool WHOLE, int GATE>
__global__ __launch_bounds__(256) void k_fp8_rows(const void *__restrict__ in, uint32_t cols, uint32_t blocks, uint32_t items, uint32_t paired, uint8_t *__restrict__ q, float *__restrict__ scales)
{
    const uint32_t item = blockIdx.x * 16u + (threadIdx.x >> 4);
    if (item >= items) return;   // (all sixteen lanes of an item)
    const uint32_t row = item / blocks, block = item - row * blocks, col = block * 128u + (threadIdx.x & 15u) * kFp8Each;
    constexpr size_t kEach = F16 ? 2 : 4;
    const char *src = (const char *)in + (size_t)row * cols * (GATE ? 2 * kEach : kEach);
    float v[8];
    if constexpr (GATE != 0) {
        // (a run of 32 paired columns is whole: eight columns never cross into the up half)
        const uint32_t g_col = paired ? paired_col(col) : col, u_col = paired ? g_col + kPairWidth : col + cols;
        const bool in_row = col < cols;
        float g[8], u[8];
        load_8<F16, WHOLE>(g, src, in_row ? g_col : 2u * cols, paired ? 2u * cols : cols);
        load_8<F16, WHOLE>(u, src, in_row ? u_col : 2u * cols, 2u * cols);
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = gate_rows<GATE, F16>(g[j], u[j]);
        const float least = fminf(fminf(fminf(g[0], g[1]), fminf(g[2], g[3])), fminf(fminf(g[4], g[5]), fminf(g[6], g[7])));
        if (__builtin_expect(least < far_gate<GATE>, 0)) {
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (g[j] < far_gate<GATE>) v[j] = gate_far<GATE>(g[j], u[j]);
        }
    } else {
        load_8<F16, WHOLE>(v, src, col, cols);
    }
    store_codes<WHOLE>(q + (size_t)row * cols, scales + item, col, cols, v);
}

// A workgroup per row.  Bound: the rows' way through memory (2048 x 4096 f16 rows with every output 26.6 us, 4.1 TB/s of four arrays in
// and out; a copy reaches 4.7).  s = x (+ residual) stays in registers up to 8 * THREADS * HELD columns; a longer row is read again for its
// second pass.  sum: where s goes, or null; it may be the residual itself, whose elements are read by the lane that writes them.
template <bool F16, bool WHOLE, uint32_t THREADS, uint32_t HELD>
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
    double squares = 0.0;   // (in 64 bits, which hold the square of any f32 and the sum over a row of any length)
    auto take = [&](float (&s)[8], uint32_t col) {
        load_8<F16, WHOLE>(s, x_row, col, cols);
        if (r_row) {
            float r[8];
            load_8<false, WHOLE>(r, r_row, col, cols);
#pragma unroll
            for (int j = 0; j < 8; j++) s[j] += r[j];
        }
    };
    auto add = [&](const float (&s)[8]) {
#pragma unroll
        for (int j = 0; j < 8; j++) squares = fma((double)s[j], (double)s[j], squares);
    };
#pragma unroll
    for (uint32_t h = 0; h < HELD; h++) take(v[h], col0 + h * kSpan);
#pragma unroll
    for (uint32_t h = 0; h < HELD; h++) {
        add(v[h]);
        if (s_row) store_f32_8<WHOLE>(s_row, col0 + h * kSpan, cols, v[h]);
    }
    for (uint64_t at = (uint64_t)kSpan * HELD; at < cols; at += kSpan) {
        const uint64_t col = at + col0;
        if (col >= cols) break;
        float s[8];
        take(s, (uint32_t)col);
        add(s);
        if (s_row) store_f32_8<WHOLE>(s_row, (uint32_t)col, cols, s);
    }
#pragma unroll
    for (int step = 32; step; step >>= 1) squares += __shfl_xor(squares, step);
    if ((threadIdx.x & 63u) == 0) parts[threadIdx.x >> 6] = squares;
    __syncthreads();
    squares = 0.0;
#pragma unroll
    for (uint32_t w = 0; w < kWaves; w++) squares += parts[w];
    // 1 / sqrt(mean + eps) as a power of two, which takes a row of any magnitude half way to one, and the rest: neither need be beyond f32
    // where the result is not
    const double whole = 1.0 / sqrt(squares / cols + (double)eps);
    const int half_way = __builtin_amdgcn_frexp_exp(whole) / 2;
    const float power = ldexpf(1.0f, half_way), scale = (float)ldexp(whole, -half_way);

    // (whole groups of sixteen lanes: the columns of a block behind the row's end count as zeros)
    auto finish = [&](float (&s)[8], uint64_t col) {
        if (col >= (uint64_t)blocks * 128u) return;
        float w[8];
        load_8<false, WHOLE>(w, weight, (uint32_t)col, cols);
#pragma unroll
        for (int j = 0; j < 8; j++) s[j] = s[j] * power * scale * w[j];
        if (normed) store_f16_8<WHOLE>(normed + row * cols, (uint32_t)col, cols, s);
        store_codes<WHOLE>(q + row * cols, scales + row * blocks + (uint32_t)(col >> 7), (uint32_t)col, cols, s);
    };
#pragma unroll
    for (uint32_t h = 0; h < HELD; h++) finish(v[h], col0 + h * kSpan);
    for (uint64_t at = (uint64_t)kSpan * HELD; at < cols; at += kSpan) {
        const uint64_t col = at + col0;
        if (col >= (uint64_t)blocks * 128u) break;
        float s[8];
        // (what this lane wrote, where the residual may have been written over)
        if (s_row) load_8<false, WHOLE>(s, s_row, (uint32_t)col, cols);
        else take(s, (uint32_t)col);
        finish(s, col);
    }
}

hipError_t launch_fp8_rows(hipStream_t s, const void *in, bool f16, uint32_t rows, uint32_t cols, int gate, bool paired, uint8_t *q, float *scales)
{
    if (rows == 0 || cols == 0) return hipSuccess;
    const uint32_t blocks = (cols + 127u) / 128u;
    const bool whole = cols % 8 == 0;
    auto kernel_of = [&](auto which) {
        constexpr int GATE = decltype(which)::value;
        return f16 ? (whole ? k_fp8_rows<true, true, GATE> : k_fp8_rows<true, false, GATE>) : (whole ? k_fp8_rows<false, true, GATE> : k_fp8_rows<false, false, GATE>);
    };
    auto kernel = gate == 0   ? kernel_of(std::integral_constant<int, 0>{})
                  : gate == 1 ? kernel_of(std::integral_constant<int, 1>{})
                              : kernel_of(std::integral_constant<int, 2>{});
    const size_t row_bytes = (size_t)cols * (gate ? 2 : 1) * (f16 ? 2 : 4);
    return in_slices(rows, most_workgroups(256) * 16u / blocks, [&](uint32_t row, uint32_t here) {
        const uint32_t items = here * blocks;
        hipLaunchKernelGGL(kernel, dim3((items + 15) / 16), dim3(256), 0, s, (const char *)in + row * row_bytes, cols, blocks, items, paired ? 1u : 0u,
                           q + (size_t)row * cols, scales + (size_t)row * blocks);
        return hipGetLastError();
    });
}

hipError_t launch_fp8_norm(hipStream_t s, const void *x, bool f16, const float *residual, const float *weight, float eps, uint32_t rows,
                           uint32_t cols, float *sum, uint8_t *q, float *scales, uint16_t *normed)
{
    if (rows == 0 || cols == 0) return hipSuccess;
    const uint32_t blocks = (cols + 127u) / 128u;
    const bool whole = cols % 8 == 0;
    // Sixteen waves for a row where four would hold less than all of it, or there are fewer rows than CUs (1024 x 8192 f16 rows with every
    // output 26.8 us on four, 24.2 on sixteen; in a graph 1 x 8192 5.6 and 4.1, 1 x 4096 3.5 and 3.1, 256 x 4096 5.2 and 4.9; but 2048 x 4096
    // f32 rows without a residual 10.0 and 13.7), and two for short rows (9362 x 896 such rows 14.7 us on four, 10.4 on two)
    const bool wide = cols > 4096 || (rows <= 256 && cols > 2048), brief = cols <= 1024;
    auto kernel_of = [&](auto threads, auto held) {
        constexpr uint32_t THREADS = decltype(threads)::value, HELD = decltype(held)::value;
        return f16 ? (whole ? k_fp8_norm<true, true, THREADS, HELD> : k_fp8_norm<true, false, THREADS, HELD>)
                   : (whole ? k_fp8_norm<false, true, THREADS, HELD> : k_fp8_norm<false, false, THREADS, HELD>);
    };
    auto kernel = wide    ? kernel_of(std::integral_constant<uint32_t, 1024>{}, std::integral_constant<uint32_t, 1>{})
                  : brief ? kernel_of(std::integral_constant<uint32_t, 128>{}, std::integral_constant<uint32_t, 1>{})
                          : kernel_of(std::integral_constant<uint32_t, 256>{}, std::integral_constant<uint32_t, 2>{});
    const uint32_t threads = wide ? 1024 : brief ? 128 : 256;
    return in_slices(rows, most_workgroups(threads), [&](uint32_t row, uint32_t here) {
        const size_t at = (size_t)row * cols;
        hipLaunchKernelGGL(kernel, dim3(here), dim3(threads), 0, s, (const char *)x + at * (f16 ? 2 : 4), residual ? residual + at : nullptr, weight, eps, cols, blocks,
                           sum ? sum + at : nullptr, q + at, scales + (size_t)row * blocks, normed ? (_Float16 *)normed + at : nullptr);
        return hipGetLastError();
    });
}

}  // namespace twm
