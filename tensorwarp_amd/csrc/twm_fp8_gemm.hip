// C[M,N] = A[M,K] x W[N,K]^T in 8-bit floating point (e4m3) with f32 scales, one per row and 128 features of A and one per
// 128 x 128 block of W:
//
//   C[m][n] = sum over blocks b of a_scales[m][b] * w_scales[n / 128][b] * (sum over the block's k of A[m][k] * W[n][k])
//
// The matrix unit's 8-bit instructions are not used where sums are to hold 32 bits: they cut every product of eight
// neighbouring features off below 2^-13 of the largest one's power of two before they add (measured: 2^14 + 2^0 is 2^14 within a
// group of eight and exact across two, against the exact sum results were off by 1.2e-5 of their norm on bell-shaped values and
// 5e-5 on evenly drawn codes).  The codes become f16 instead, which holds each exactly, as do the f32 products of
// v_mfma_f32_16x16x32_f16.  A block's sum is scaled by one f32 factor per lane (the rows of A are the lanes' columns of the
// result, those of W lie in its registers) and added to the f32 sum.  Both arrays are read as the caller holds them, row by
// row: a lane's operand is 32 consecutive bytes of a row, and which of the 128 features a lane holds does not matter as long as
// both operands agree.
#include "twm_device.h"

namespace twm {

typedef int int8v __attribute__((ext_vector_type(8)));

namespace {

struct Fp8Gemm {
    const uint8_t *a, *w;
    const float *a_scales, *w_scales;
    uint32_t m, n, k, kb;    // kb = blocks of 128 features, the last one possibly cut short (k is a multiple of 16)
    void *c;
    uint32_t c_f16;
};

// eight codes as f16 (exact)
__device__ __forceinline__ half8 to_f16(int lo, int hi)
{
    const half2v a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, false), b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, true);
    const half2v c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, false), d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, true);
    return half8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// the sum over a block of 128 features of 16 rows of each operand
__device__ __forceinline__ float4v block_sum(const int8v &w, const int8v &a)
{
    float4v d = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 8; i += 2) d = __builtin_amdgcn_mfma_f32_16x16x32_f16(to_f16(w[i], w[i + 1]), to_f16(a[i], a[i + 1]), d, 0, 0, 0);
    return d;
}

// 32 bytes of a row; a 16-byte piece behind the row's end is zeros (and is not read)
template <bool TAIL> __device__ __forceinline__ int8v load_32(const uint8_t *row, uint32_t k0, uint32_t k)
{
    uint4v lo, hi;
    if constexpr (TAIL) {
        lo = *(const uint4v *)(row + (k0 < k ? k0 : 0u));
        hi = *(const uint4v *)(row + (k0 + 16u < k ? k0 + 16u : 0u));
        const uint4v zero = {0u, 0u, 0u, 0u};
        lo = k0 < k ? lo : zero;
        hi = k0 + 16u < k ? hi : zero;
    } else {
        lo = *(const uint4v *)(row + k0);
        hi = *(const uint4v *)(row + k0 + 16u);
    }
    return int8v{(int)lo[0], (int)lo[1], (int)lo[2], (int)lo[3], (int)hi[0], (int)hi[1], (int)hi[2], (int)hi[3]};
}

// columns n .. n + 3 of row m; VEC: N is a multiple of four and C aligned to four columns
__device__ __forceinline__ void store_quad(const Fp8Gemm &g, bool vec, uint32_t m, uint32_t n, const float4v &v)
{
    if (m >= g.m || n >= g.n) return;
    const size_t at = (size_t)m * g.n + n;
    if (g.c_f16) {
        _Float16 *c = (_Float16 *)g.c + at;
        if (vec) {
            typedef _Float16 half4 __attribute__((ext_vector_type(4)));
            *(half4 *)c = half4{(_Float16)v[0], (_Float16)v[1], (_Float16)v[2], (_Float16)v[3]};
        } else {
#pragma unroll
            for (uint32_t j = 0; j < 4; j++)
                if (n + j < g.n) c[j] = (_Float16)v[j];
        }
    } else {
        float *c = (float *)g.c + at;
        if (vec) {
            *(float4v *)c = v;
        } else {
#pragma unroll
            for (uint32_t j = 0; j < 4; j++)
                if (n + j < g.n) c[j] = v[j];
        }
    }
}

bool fp8_vec_store(const Fp8Gemm &g) { return g.n % 4 == 0 && ((uintptr_t)g.c & (g.c_f16 ? 7 : 15)) == 0; }

}  // namespace

// 16 columns x 16 * MT rows per workgroup, K shared out among its waves block by block; the waves' sums are added in LDS in wave
// order.
template <int MT, int WAVES>
__global__ __launch_bounds__(WAVES * 64) void k_fp8_gemm_simple(const Fp8Gemm g, uint32_t vec)
{
    __shared__ float4v sums[WAVES][MT][64];
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63u;
    const uint32_t n0 = blockIdx.x * 16u, m0 = blockIdx.y * (16u * MT), part = (lane >> 4) * 32u;
    // rows behind the end replay the last one and are not stored
    const uint32_t n_row = min(n0 + (lane & 15u), g.n - 1u);
    const uint8_t *w_row = g.w + (size_t)n_row * g.k;
    const uint8_t *a_row[MT];
    const float *as_row[MT];
#pragma unroll
    for (int t = 0; t < MT; t++) {
        const uint32_t m_row = min(m0 + 16u * t + (lane & 15u), g.m - 1u);
        a_row[t] = g.a + (size_t)m_row * g.k;
        as_row[t] = g.a_scales + (size_t)m_row * g.kb;
    }
    const float *ws_row = g.w_scales + (size_t)(n0 >> 7) * g.kb;
    float4v acc[MT] = {};
    for (uint32_t b = wave; b < g.kb; b += WAVES) {
        const uint32_t k0 = b * 128u + part;
        const bool tail = b * 128u + 128u > g.k;
        const int8v w = tail ? load_32<true>(w_row, k0, g.k) : load_32<false>(w_row, k0, g.k);
        const float ws = ws_row[b];
#pragma unroll
        for (int t = 0; t < MT; t++) {
            const int8v a = tail ? load_32<true>(a_row[t], k0, g.k) : load_32<false>(a_row[t], k0, g.k);
            const float4v d = block_sum(w, a);
            acc[t] += d * (as_row[t][b] * ws);
        }
    }
#pragma unroll
    for (int t = 0; t < MT; t++) sums[wave][t][lane] = acc[t];
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < MT * 64u; i += WAVES * 64u) {
        const uint32_t t = i >> 6, l = i & 63u;
        float4v s = sums[0][t][l];
#pragma unroll
        for (int w = 1; w < WAVES; w++) s += sums[w][t][l];
        store_quad(g, vec, m0 + 16u * t + (l & 15u), n0 + (l >> 4) * 4u, s);
    }
}

hipError_t launch_fp8_gemm(hipStream_t s, const uint8_t *a, const float *a_scales, const uint8_t *w, const float *w_scales, uint32_t m,
                           uint32_t n, uint32_t k, void *c, bool c_f16, float *ws, size_t ws_bytes)
{
    if (m == 0 || n == 0) return hipSuccess;
    const Fp8Gemm g = {a, w, a_scales, w_scales, m, n, k, (k + 127u) / 128u, c, c_f16 ? 1u : 0u};
    const uint32_t tiles_m = (m + 15u) / 16u, tiles_n = (n + 15u) / 16u;
    if (tiles_m == 1) hipLaunchKernelGGL((k_fp8_gemm_simple<1, 8>), dim3(tiles_n, 1), dim3(512), 0, s, g, fp8_vec_store(g));
    else hipLaunchKernelGGL((k_fp8_gemm_simple<4, 4>), dim3(tiles_n, (tiles_m + 3u) / 4u), dim3(256), 0, s, g, fp8_vec_store(g));
    return hipGetLastError();
}

}  // namespace twm
