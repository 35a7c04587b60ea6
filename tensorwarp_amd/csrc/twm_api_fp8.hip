// C ABI of libtwmarlin_hip.so (declared in include/twmarlin.h), part: linear layers in 8-bit floating point, the rows that feed
// them, and token sampling.
#include "twm_api_impl.h"

using namespace twm;

namespace {

constexpr uint32_t kFp8MostDim = 1u << 24;   // rows and columns of one call
constexpr uint32_t kFp8MostK = 1u << 20;     // features of a product (256 rows of codes are within a buffer's 32-bit offsets)

bool row_type(int dtype) { return dtype == TWM_F32 || dtype == TWM_F16; }

// what the calls that write e4m3 rows check alike; 1: nothing to do
int check_rows(const char *who, const twm_ctx *ctx, const void *in, int dtype, uint32_t rows, uint32_t cols, const void *q, const void *scales)
{
    if (!ctx) return api_fail(TWM_INVALID_HANDLE, "%s: null context", who);
    if (!row_type(dtype)) return api_fail(TWM_UNSUPPORTED_OP, "%s: rows must be f16 or f32", who);
    if (rows > kFp8MostDim || cols > kFp8MostDim) return api_fail(TWM_SHAPE_ERROR, "%s: %u x %u is beyond 2^24 rows or columns", who, rows, cols);
    if (rows == 0 || cols == 0) return -1;
    if (!in || !q || !scales) return api_fail(TWM_INVALID_HANDLE, "%s: null pointer", who);
    if (misaligned(in, dtype == TWM_F16 ? 2 : 4) || misaligned(scales, 4)) return api_fail(TWM_SHAPE_ERROR, "%s: a pointer is not aligned to its elements", who);
    return TWM_OK;
}

int gated_rows(const char *who, twm_ctx *ctx, const void *gate_up_dev, int dtype, uint32_t batch, uint32_t dim, int paired, int act, uint8_t *q_dev,
               float *scales_dev)
{
    if (int rc = check_rows(who, ctx, gate_up_dev, dtype, batch, dim, q_dev, scales_dev)) return rc < 0 ? TWM_OK : rc;
    if (paired && dim % kPairWidth != 0) return api_fail(TWM_SHAPE_ERROR, "%s: the paired order needs a multiple of %u columns, got %u", who, kPairWidth, dim);
    DeviceGuard on(ctx);
    HIP_TRY(on.status, TWM_DEVICE_ERROR, who);
    HIP_TRY(launch_fp8_rows(ctx->stream, gate_up_dev, dtype == TWM_F16, batch, dim, act, paired != 0, q_dev, scales_dev), TWM_DEVICE_ERROR, who);
    return TWM_OK;
}

}  // namespace

extern "C" {

static int check_gemm_fp8(const char *who, uint32_t m, uint32_t n, uint32_t k, int c_dtype)
{
    if (!row_type(c_dtype)) return api_fail(TWM_UNSUPPORTED_OP, "%s: results must be f16 or f32", who);
    if (k % 16 != 0) return api_fail(TWM_SHAPE_ERROR, "%s: K (%u) must be divisible by 16", who, k);
    if (m > kFp8MostDim || n > kFp8MostDim) return api_fail(TWM_SHAPE_ERROR, "%s: %u x %u is beyond 2^24 rows or columns", who, m, n);
    if ((uint64_t)m * n > 1ull << 36) return api_fail(TWM_SHAPE_ERROR, "%s: %u x %u results are more than 2^36", who, m, n);
    if (k > kFp8MostK) return api_fail(TWM_SHAPE_ERROR, "%s: K (%u) is beyond 2^20", who, k);
    return TWM_OK;
}

int twm_gemm_fp8(twm_ctx *ctx, const uint8_t *a_dev, const float *a_scales_dev, const uint8_t *w_dev, const float *w_scales_dev, uint32_t m, uint32_t n,
                 uint32_t k, void *c_dev, int c_dtype)
{
    const char *who = "twm_gemm_fp8";
    if (!ctx) return api_fail(TWM_INVALID_HANDLE, "%s: null context", who);
    if (int rc = check_gemm_fp8(who, m, n, k, c_dtype)) return rc;
    if (m == 0 || n == 0) return TWM_OK;
    if (!c_dev || (k != 0 && (!a_dev || !a_scales_dev || !w_dev || !w_scales_dev))) return api_fail(TWM_INVALID_HANDLE, "%s: null pointer", who);
    if (misaligned(a_dev, 16) || misaligned(w_dev, 16)) return api_fail(TWM_SHAPE_ERROR, "%s: A and W must be 16-byte aligned", who);
    if (misaligned(a_scales_dev, 4) || misaligned(w_scales_dev, 4) || misaligned(c_dev, c_dtype == TWM_F16 ? 2 : 4))
        return api_fail(TWM_SHAPE_ERROR, "%s: a pointer is not aligned to its elements", who);
    DeviceGuard on(ctx);
    HIP_TRY(on.status, TWM_DEVICE_ERROR, who);
    HIP_TRY(launch_fp8_gemm(ctx->stream, a_dev, a_scales_dev, w_dev, w_scales_dev, m, n, k, c_dev, c_dtype == TWM_F16, ctx->ws, ctx->ws_bytes),
            TWM_DEVICE_ERROR, who);
    return TWM_OK;
}

int twm_plan_describe_fp8(uint32_t m, uint32_t n, uint32_t k, int c_dtype, char *text, size_t bytes)
{
    const char *who = "twm_plan_describe_fp8";
    if (!text || bytes == 0) return api_fail(TWM_INVALID_HANDLE, "%s: null buffer", who);
    if (int rc = check_gemm_fp8(who, m, n, k, c_dtype)) return rc;
    describe_fp8_gemm(m, n, k, c_dtype == TWM_F16, kWsBytes, text, bytes);
    return TWM_OK;
}

int twm_quantize_rows_fp8(twm_ctx *ctx, const void *x_dev, int x_dtype, uint32_t rows, uint32_t cols, uint8_t *q_dev, float *scales_dev)
{
    const char *who = "twm_quantize_rows_fp8";
    if (int rc = check_rows(who, ctx, x_dev, x_dtype, rows, cols, q_dev, scales_dev)) return rc < 0 ? TWM_OK : rc;
    DeviceGuard on(ctx);
    HIP_TRY(on.status, TWM_DEVICE_ERROR, who);
    HIP_TRY(launch_fp8_rows(ctx->stream, x_dev, x_dtype == TWM_F16, rows, cols, 0, false, q_dev, scales_dev), TWM_DEVICE_ERROR, who);
    return TWM_OK;
}

int twm_swiglu_rows_fp8(twm_ctx *ctx, const void *gate_up_dev, int dtype, uint32_t batch, uint32_t ffn_dim, int paired, uint8_t *q_dev, float *scales_dev)
{
    return gated_rows("twm_swiglu_rows_fp8", ctx, gate_up_dev, dtype, batch, ffn_dim, paired, 2, q_dev, scales_dev);
}

int twm_geglu_rows_fp8(twm_ctx *ctx, const void *gate_up_dev, int dtype, uint32_t batch, uint32_t dim, int paired, uint8_t *q_dev, float *scales_dev)
{
    return gated_rows("twm_geglu_rows_fp8", ctx, gate_up_dev, dtype, batch, dim, paired, 1, q_dev, scales_dev);
}

int twm_add_rms_norm_fp8(twm_ctx *ctx, const void *x_dev, int x_dtype, const float *residual_dev, const float *weight_dev, float eps, uint32_t rows,
                         uint32_t cols, float *sum_dev, uint8_t *q_dev, float *scales_dev, uint16_t *normed_dev_f16)
{
    const char *who = "twm_add_rms_norm_fp8";
    if (int rc = check_rows(who, ctx, x_dev, x_dtype, rows, cols, q_dev, scales_dev)) return rc < 0 ? TWM_OK : rc;
    if (!weight_dev) return api_fail(TWM_INVALID_HANDLE, "%s: null pointer", who);
    if (misaligned(residual_dev, 4) || misaligned(weight_dev, 4) || misaligned(sum_dev, 4) || misaligned(normed_dev_f16, 2))
        return api_fail(TWM_SHAPE_ERROR, "%s: a pointer is not aligned to its elements", who);
    if (!(eps >= 0.0f)) return api_fail(TWM_SHAPE_ERROR, "%s: eps must not be negative or NaN", who);
    DeviceGuard on(ctx);
    HIP_TRY(on.status, TWM_DEVICE_ERROR, who);
    HIP_TRY(launch_fp8_norm(ctx->stream, x_dev, x_dtype == TWM_F16, residual_dev, weight_dev, eps, rows, cols, sum_dev, q_dev, scales_dev, normed_dev_f16),
            TWM_DEVICE_ERROR, who);
    return TWM_OK;
}

int twm_sample_f32(twm_ctx *ctx, const float *logits_dev, uint32_t rows, uint32_t cols, const float *uniform_dev, const float *temperature_dev,
                   const int32_t *top_k_dev, const float *top_p_dev, const float *min_p_dev, int32_t *out_dev)
{
    const char *who = "twm_sample_f32";
    if (!ctx) return api_fail(TWM_INVALID_HANDLE, "%s: null context", who);
    if (rows > kFp8MostDim || cols > kFp8MostDim) return api_fail(TWM_SHAPE_ERROR, "%s: %u x %u is beyond 2^24 rows or columns", who, rows, cols);
    if (rows == 0) return TWM_OK;
    if (!out_dev || !uniform_dev || (cols != 0 && !logits_dev)) return api_fail(TWM_INVALID_HANDLE, "%s: null pointer", who);
    if (misaligned(logits_dev, 4) || misaligned(uniform_dev, 4) || misaligned(temperature_dev, 4) || misaligned(top_k_dev, 4) || misaligned(top_p_dev, 4) ||
        misaligned(min_p_dev, 4) || misaligned(out_dev, 4))
        return api_fail(TWM_SHAPE_ERROR, "%s: a pointer is not aligned to its elements", who);
    DeviceGuard on(ctx);
    HIP_TRY(on.status, TWM_DEVICE_ERROR, who);
    HIP_TRY(launch_sample(ctx->stream, logits_dev, rows, cols, uniform_dev, temperature_dev, top_k_dev, top_p_dev, min_p_dev, out_dev, ctx->ws, ctx->ws_bytes,
                          ctx->counters, ctx->n_counters),
            TWM_DEVICE_ERROR, who);
    return TWM_OK;
}

}  // extern "C"
