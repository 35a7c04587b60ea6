// The paged key-value cache: new tokens' rows into their pages, and whole pages to other pages.
#include "twm_kv.h"

#include <algorithm>
#include <cmath>

namespace twm {

namespace {

struct Append {
    KvView kv;
    KvSeqs seqs;
    const void *qkv;
    const float *cos_sin;
    _Float16 *q_out;
    uint32_t qkv_stride, q_heads, positions, rotary_dim, interleaved;
};

template <bool F16> __device__ __forceinline__ void load_8(float (&v)[8], const void *row, uint32_t col)
{
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
}

__device__ __forceinline__ half8 rounded_8(const float (&v)[8])
{
    half8 h;
#pragma unroll
    for (int j = 0; j < 8; j++) h[j] = (_Float16)v[j];
    return h;
}

// eight values as e4m3 codes: the quotient as f32 rounds it, cut off at the largest code (a NaN is neither above nor below), and the
// nearest code, ties to the even one
__device__ __forceinline__ uint2v codes_8(const float (&v)[8], float scale)
{
    float u[8];
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const float x = v[j] / scale;
        u[j] = x > 448.0f ? 448.0f : x < -448.0f ? -448.0f : x;
    }
    int lo = __builtin_amdgcn_cvt_pk_fp8_f32(u[0], u[1], 0, false), hi = __builtin_amdgcn_cvt_pk_fp8_f32(u[4], u[5], 0, false);
    lo = __builtin_amdgcn_cvt_pk_fp8_f32(u[2], u[3], lo, true);
    hi = __builtin_amdgcn_cvt_pk_fp8_f32(u[6], u[7], hi, true);
    return uint2v{(unsigned)lo, (unsigned)hi};
}

}  // namespace

// A workgroup per row.  A thread holds sixteen values of one head: the two runs of eight that a rotation of halves turns into each other,
// or sixteen neighbours.  The row's sequence is the last one that starts up to it, found among as many at once as there are threads.
// One row is a launch and the way from the starts by the length and the table to the store (4.0 - 4.8 us); 2048 rows of 36 heads of 128 f16 values
// into e4m3, 37 MB, take 11.8 us (3.1 TB/s), into f16 10.3 (3.8), of f32 values 15.6 and 15.1: one round of workgroups, whose loads wait for their sequence.
template <bool F16> __global__ void k_kv_append(const Append a)
{
    const uint32_t row = blockIdx.x, dim = a.kv.dim, each = dim >> 4, units = (a.q_heads + 2u * a.kv.kv_heads) * each;
    int seq = (int)row, behind = 0;   // behind: the rows of the sequence from this one on
    if (a.seqs.starts) {
        uint32_t base = 0, among = a.seqs.seqs;
        for (uint32_t stride = 0; stride != 1; among = min(stride, a.seqs.seqs - base)) {
            stride = (among + blockDim.x - 1) / blockDim.x;
            const uint32_t s = threadIdx.x * stride;
            const uint32_t begun = (uint32_t)__syncthreads_count(s < among && a.seqs.starts[base + s] <= (int)row);
            if (begun == 0) return;
            base += (begun - 1) * stride;
        }
        seq = (int)base;
        behind = a.seqs.starts[seq + 1] - (int)row;
    } else {
        behind = 1;
    }
    const int position = max(a.seqs.lengths[seq], 0) - behind;
    if (behind <= 0 || position < 0) return;
    const uint32_t in_table = (uint32_t)position >> a.kv.page_shift;
    const int page = in_table < a.seqs.table_stride ? a.seqs.tables[(size_t)seq * a.seqs.table_stride + in_table] : -1;
    const uint32_t token = (uint32_t)position & ((1u << a.kv.page_shift) - 1u), half = a.rotary_dim >> 1;
    const char *from = (const char *)a.qkv + (size_t)row * a.qkv_stride * (F16 ? 2 : 4);
    for (uint32_t unit = threadIdx.x; unit < units; unit += blockDim.x) {
        const uint32_t head = unit / each, part = unit - head * each;
        const bool turned = head < a.q_heads + a.kv.kv_heads && 16u * part < a.rotary_dim, halves = turned && !a.interleaved;
        const uint32_t first = halves ? 8u * part : 16u * part, second = halves ? first + half : first + 8u;
        float x[8], y[8];
        load_8<F16>(x, from, head * dim + first);
        load_8<F16>(y, from, head * dim + second);
        if (turned) {
            const float *angles = a.cos_sin + (size_t)position * a.rotary_dim;
            float c[8], s[8];
            if ((uint32_t)position < a.positions) {
                load_8<false>(c, angles, 8u * part);
                load_8<false>(s, angles, half + 8u * part);
            } else {
#pragma unroll
                for (int j = 0; j < 8; j++) c[j] = s[j] = NAN;
            }
            if (halves) {
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const float p = x[j], r = y[j];
                    x[j] = fmaf(p, c[j], -(r * s[j]));
                    y[j] = fmaf(r, c[j], p * s[j]);
                }
            } else {
#pragma unroll
                for (int j = 0; j < 8; j += 2) {
                    const float p = x[j], r = x[j + 1], t = y[j], u = y[j + 1], c0 = c[j / 2], s0 = s[j / 2], c1 = c[4 + j / 2], s1 = s[4 + j / 2];
                    x[j] = fmaf(p, c0, -(r * s0));
                    x[j + 1] = fmaf(r, c0, p * s0);
                    y[j] = fmaf(t, c1, -(u * s1));
                    y[j + 1] = fmaf(u, c1, t * s1);
                }
            }
        }
        if (head < a.q_heads) {
            _Float16 *to = a.q_out + ((size_t)row * a.q_heads + head) * dim;
            *(half8_any *)(to + first) = rounded_8(x);
            *(half8_any *)(to + second) = rounded_8(y);
        } else if ((uint32_t)page < a.kv.pages) {
            const bool value = head >= a.q_heads + a.kv.kv_heads;
            const uint32_t h = head - a.q_heads - (value ? a.kv.kv_heads : 0u);
            const size_t at = kv_chunk(a.kv, (uint32_t)page, h) + (size_t)token * dim;
            void *to = value ? a.kv.v : a.kv.k;
            if (a.kv.e4m3) {
                const float *scales = value ? a.kv.v_scales : a.kv.k_scales;
                const float scale = scales ? scales[h] : 1.0f;
                *(uint2v *)((uint8_t *)to + at + first) = codes_8(x, scale);
                *(uint2v *)((uint8_t *)to + at + second) = codes_8(y, scale);
            } else {
                *(half8 *)((_Float16 *)to + at + first) = rounded_8(x);
                *(half8 *)((_Float16 *)to + at + second) = rounded_8(y);
            }
        }
    }
}

hipError_t launch_kv_append(hipStream_t s, const KvView &kv, const KvSeqs &seqs, const void *qkv, bool f16, uint32_t rows, uint32_t qkv_stride,
                            uint32_t q_heads, const float *cos_sin, uint32_t positions, uint32_t rotary_dim, bool interleaved, _Float16 *q_out)
{
    const Append a{kv, seqs, qkv, cos_sin, q_out, qkv_stride, q_heads, positions, rotary_dim, interleaved};
    const uint32_t units = (q_heads + 2 * kv.kv_heads) * (kv.dim / 16), threads = std::min(512u, (units + 63u) / 64u * 64u);
    hipLaunchKernelGGL(f16 ? k_kv_append<true> : k_kv_append<false>, dim3(rows), dim3(threads), 0, s, a);
    return hipGetLastError();
}

// ---- whole pages ------------------------------------------------------------------------------------------------------

namespace {

// What a launch takes along: pages and arrays travel as arguments of the kernel, so that a call needs no memory of its own and a
// captured one keeps what it was given.
constexpr uint32_t kCopyArrays = 128, kCopyPairs = 320, kCopyPiece = 256 * 16 * 4;   // bytes per workgroup
struct Copy {
    uint32_t page_bytes, pieces;
    void *array[kCopyArrays];
    uint32_t source[kCopyPairs], target[kCopyPairs];
};
static_assert(sizeof(Copy) <= 4000, "arguments of a kernel end at 4 KB");

}  // namespace

// A workgroup per 16 KB piece, four loads of 16 bytes a lane on their way.  Bound by memory where pages are many (500 of 16 KB, keys and values of 28
// layers, 918 MB read and written: 187 us, 4.9 TB/s, a large copy's 5.1), by the host where they are few (one page 4.6 - 5.7 us, of which the kernel takes 2.9).
__global__ __launch_bounds__(256) void k_kv_copy_pages(const Copy c)
{
    char *base = (char *)c.array[blockIdx.z];
    const uint32_t at = blockIdx.x * kCopyPiece + threadIdx.x * 16u;
    const uint4v *from = (const uint4v *)(base + (size_t)c.source[blockIdx.y] * c.page_bytes + at);
    uint4v *to = (uint4v *)(base + (size_t)c.target[blockIdx.y] * c.page_bytes + at);
    uint4v v[4];
#pragma unroll
    for (uint32_t i = 0; i < 4; i++)
        if (at + i * 4096u < c.page_bytes) v[i] = from[i * 256u];
#pragma unroll
    for (uint32_t i = 0; i < 4; i++)
        if (at + i * 4096u < c.page_bytes) to[i * 256u] = v[i];
}

hipError_t launch_kv_copy_pages(hipStream_t s, const KvView *caches, uint32_t count, const uint32_t *sources, const uint32_t *targets, uint32_t pairs)
{
    Copy c;
    c.page_bytes = (caches->kv_heads << caches->page_shift) * caches->dim * (caches->e4m3 ? 1u : 2u);
    c.pieces = (c.page_bytes + kCopyPiece - 1) / kCopyPiece;
    // as few launches as hold them, all of a size
    const uint32_t sets = (pairs + kCopyPairs - 1) / kCopyPairs, each = (pairs + sets - 1) / sets;
    for (uint32_t first = 0; first < count; first += kCopyArrays / 2) {
        const uint32_t layers = std::min(kCopyArrays / 2, count - first);
        for (uint32_t i = 0; i < layers; i++) {
            c.array[2 * i] = caches[first + i].k;
            c.array[2 * i + 1] = caches[first + i].v;
        }
        for (uint32_t pair = 0; pair < pairs; pair += each) {
            const uint32_t here = std::min(each, pairs - pair);
            std::copy(sources + pair, sources + pair + here, c.source);
            std::copy(targets + pair, targets + pair + here, c.target);
            hipLaunchKernelGGL(k_kv_copy_pages, dim3(c.pieces, here, 2 * layers), dim3(256), 0, s, c);
            if (const hipError_t error = hipGetLastError(); error != hipSuccess) return error;
        }
    }
    return hipSuccess;
}

}  // namespace twm
