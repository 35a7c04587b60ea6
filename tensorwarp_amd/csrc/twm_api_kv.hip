// C ABI of libtwmarlin_hip.so (declared in include/twmarlin.h), part: the paged key-value cache and the attention that reads it.
#include "twm_api_impl.h"

#include <algorithm>
#include <cmath>

using namespace twm;

namespace {

constexpr uint32_t kKvMostRows = 1u << 20, kKvMostHeads = 1024, kKvMostPages = 1u << 28;
constexpr uint64_t kKvMostTokens = 1ull << 30;   // of one sequence: positions are 32-bit numbers

// A cache's description, checked.  (The arrays may be null where there is nothing to do with them: pages = 0.)
int check_cache(const char *who, const twm_kv_cache *c, KvView *view)
{
    if (!c) return api_fail(TWM_INVALID_HANDLE, "%s: null cache", who);
    if (c->dtype != TWM_F16 && c->dtype != TWM_U8) return api_fail(TWM_UNSUPPORTED_OP, "%s: a cache holds f16 or e4m3 codes (TWM_U8)", who);
    if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256)
        return api_fail(TWM_UNSUPPORTED_OP, "%s: heads of %u values (64, 128 and 256 are built)", who, c->head_dim);
    if (c->page_tokens < 16 || c->page_tokens > 256 || (c->page_tokens & (c->page_tokens - 1)) != 0)
        return api_fail(TWM_UNSUPPORTED_OP, "%s: pages of %u tokens (16, 32, 64, 128 and 256 are built)", who, c->page_tokens);
    if (c->kv_heads == 0 || c->kv_heads > kKvMostHeads) return api_fail(TWM_SHAPE_ERROR, "%s: %u key-value heads (1 to 1024)", who, c->kv_heads);
    if (c->pages > kKvMostPages) return api_fail(TWM_SHAPE_ERROR, "%s: %u pages are beyond 2^28", who, c->pages);
    if (c->pages != 0 && (!c->k_dev || !c->v_dev)) return api_fail(TWM_INVALID_HANDLE, "%s: null pointer", who);
    if (misaligned(c->k_dev, 16) || misaligned(c->v_dev, 16)) return api_fail(TWM_SHAPE_ERROR, "%s: a cache's arrays must be 16-byte aligned", who);
    if (misaligned(c->k_scales_dev, 4) || misaligned(c->v_scales_dev, 4)) return api_fail(TWM_SHAPE_ERROR, "%s: a pointer is not aligned to its elements", who);
    const bool e4m3 = c->dtype == TWM_U8;
    *view = KvView{c->k_dev, c->v_dev, e4m3 ? c->k_scales_dev : nullptr, e4m3 ? c->v_scales_dev : nullptr, e4m3, c->pages,
                   (uint32_t)__builtin_ctz(c->page_tokens), c->kv_heads, c->head_dim};
    return TWM_OK;
}

int check_seqs(const char *who, const twm_kv_cache *c, const twm_kv_seqs *s, bool starts, KvSeqs *view)
{
    if (!s) return api_fail(TWM_INVALID_HANDLE, "%s: null sequences", who);
    if (s->seqs > kKvMostRows) return api_fail(TWM_SHAPE_ERROR, "%s: %u sequences are beyond 2^20", who, s->seqs);
    if ((uint64_t)s->table_stride * c->page_tokens > kKvMostTokens) return api_fail(TWM_SHAPE_ERROR, "%s: a table's row of more than 2^30 tokens", who);
    if (s->seqs != 0 && (!s->lengths_dev || (s->table_stride != 0 && !s->tables_dev) || (starts && !s->starts_dev)))
        return api_fail(TWM_INVALID_HANDLE, "%s: null pointer", who);
    if (misaligned(s->tables_dev, 4) || misaligned(s->lengths_dev, 4) || misaligned(s->starts_dev, 4))
        return api_fail(TWM_SHAPE_ERROR, "%s: a pointer is not aligned to its elements", who);
    *view = KvSeqs{s->tables_dev, s->lengths_dev, s->starts_dev, s->seqs, s->table_stride};
    return TWM_OK;
}

int check_heads(const char *who, const twm_kv_cache *c, uint32_t q_heads)
{
    if (q_heads == 0 || q_heads > kKvMostHeads || q_heads % c->kv_heads != 0)
        return api_fail(TWM_SHAPE_ERROR, "%s: %u query heads for %u key-value heads (a multiple of them, at most 1024)", who, q_heads, c->kv_heads);
    return TWM_OK;
}

int attention(const char *who, twm_ctx *ctx, const twm_kv_cache *cache, const twm_kv_seqs *seqs, const uint16_t *q_dev, uint32_t q_stride, uint32_t rows,
              uint32_t q_heads, float scale, uint32_t window, uint16_t *out_dev, uint32_t out_stride, bool prompt)
{
    if (!ctx) return api_fail(TWM_INVALID_HANDLE, "%s: null context", who);
    AttnArgs a;
    if (int rc = check_cache(who, cache, &a.kv)) return rc;
    if (int rc = check_seqs(who, cache, seqs, prompt, &a.seqs)) return rc;
    if (int rc = check_heads(who, cache, q_heads)) return rc;
    if (!prompt) rows = seqs->seqs;
    if (rows > kKvMostRows) return api_fail(TWM_SHAPE_ERROR, "%s: %u rows are beyond 2^20", who, rows);
    if (!(scale > 0.0f) || !std::isfinite(scale)) return api_fail(TWM_SHAPE_ERROR, "%s: scale must be above 0 and finite", who);
    const uint32_t width = q_heads * cache->head_dim;
    if ((q_stride != 0 && q_stride < width) || (out_stride != 0 && out_stride < width))
        return api_fail(TWM_SHAPE_ERROR, "%s: a row stride below a row's %u values", who, width);
    if (rows == 0 || seqs->seqs == 0) return TWM_OK;
    if (!q_dev || !out_dev) return api_fail(TWM_INVALID_HANDLE, "%s: null pointer", who);
    if (misaligned(q_dev, 2) || misaligned(out_dev, 2)) return api_fail(TWM_SHAPE_ERROR, "%s: a pointer is not aligned to its elements", who);
    a.q = (const _Float16 *)q_dev;
    a.out = (_Float16 *)out_dev;
    a.rows = rows;
    a.q_stride = q_stride ? q_stride : width;
    a.out_stride = out_stride ? out_stride : width;
    a.q_heads = q_heads;
    a.group = q_heads / cache->kv_heads;
    a.scale = scale;
    a.window = std::min(window, 0x7FFFFFFFu);   // (as far as a position goes)
    DeviceGuard on(ctx);
    HIP_TRY(on.status, TWM_DEVICE_ERROR, who);
    HIP_TRY((prompt ? launch_attn_prompt : launch_attn_decode)(ctx->stream, a, ctx->ws, ctx->ws_bytes), TWM_DEVICE_ERROR, who);
    return TWM_OK;
}

}  // namespace

extern "C" {

int twm_kv_append(twm_ctx *ctx, const twm_kv_cache *cache, const twm_kv_seqs *seqs, const void *qkv_dev, int qkv_dtype, uint32_t rows,
                  uint32_t qkv_stride, uint32_t q_heads, const float *cos_sin_dev, uint32_t positions, uint32_t rotary_dim, int interleaved,
                  uint16_t *q_out_dev)
{
    const char *who = "twm_kv_append";
    if (!ctx) return api_fail(TWM_INVALID_HANDLE, "%s: null context", who);
    KvView kv;
    KvSeqs sq;
    if (int rc = check_cache(who, cache, &kv)) return rc;
    if (int rc = check_seqs(who, cache, seqs, false, &sq)) return rc;
    if (int rc = check_heads(who, cache, q_heads)) return rc;
    if (qkv_dtype != TWM_F16 && qkv_dtype != TWM_F32) return api_fail(TWM_UNSUPPORTED_OP, "%s: rows must be f16 or f32", who);
    if (rows > kKvMostRows) return api_fail(TWM_SHAPE_ERROR, "%s: %u rows are beyond 2^20", who, rows);
    if (!seqs->starts_dev && rows > seqs->seqs) return api_fail(TWM_SHAPE_ERROR, "%s: %u rows for %u sequences of one row each", who, rows, seqs->seqs);
    if (rotary_dim % 16 != 0 || rotary_dim > cache->head_dim)
        return api_fail(TWM_SHAPE_ERROR, "%s: rotary_dim (%u) must be a multiple of 16 up to the head's %u values", who, rotary_dim, cache->head_dim);
    const uint32_t width = (q_heads + 2 * cache->kv_heads) * cache->head_dim;
    if (qkv_stride != 0 && qkv_stride < width) return api_fail(TWM_SHAPE_ERROR, "%s: a row stride below a row's %u values", who, width);
    if (rows == 0 || seqs->seqs == 0) return TWM_OK;
    if (!qkv_dev || !q_out_dev || (rotary_dim != 0 && positions != 0 && !cos_sin_dev)) return api_fail(TWM_INVALID_HANDLE, "%s: null pointer", who);
    if (misaligned(qkv_dev, qkv_dtype == TWM_F16 ? 2 : 4) || misaligned(cos_sin_dev, 4) || misaligned(q_out_dev, 2))
        return api_fail(TWM_SHAPE_ERROR, "%s: a pointer is not aligned to its elements", who);
    DeviceGuard on(ctx);
    HIP_TRY(on.status, TWM_DEVICE_ERROR, who);
    HIP_TRY(launch_kv_append(ctx->stream, kv, sq, qkv_dev, qkv_dtype == TWM_F16, rows, qkv_stride ? qkv_stride : width, q_heads, cos_sin_dev, positions,
                             rotary_dim, interleaved != 0, (_Float16 *)q_out_dev),
            TWM_DEVICE_ERROR, who);
    return TWM_OK;
}

int twm_attn_decode(twm_ctx *ctx, const twm_kv_cache *cache, const twm_kv_seqs *seqs, const uint16_t *q_dev, uint32_t q_stride, uint32_t q_heads,
                    float scale, uint32_t window, uint16_t *out_dev, uint32_t out_stride)
{
    return attention("twm_attn_decode", ctx, cache, seqs, q_dev, q_stride, 0, q_heads, scale, window, out_dev, out_stride, false);
}

int twm_attn_prompt(twm_ctx *ctx, const twm_kv_cache *cache, const twm_kv_seqs *seqs, const uint16_t *q_dev, uint32_t q_stride, uint32_t rows,
                    uint32_t q_heads, float scale, uint32_t window, uint16_t *out_dev, uint32_t out_stride)
{
    return attention("twm_attn_prompt", ctx, cache, seqs, q_dev, q_stride, rows, q_heads, scale, window, out_dev, out_stride, true);
}

int twm_kv_copy_pages(twm_ctx *ctx, const twm_kv_cache *caches, uint32_t count, const uint32_t *sources, const uint32_t *targets, uint32_t pairs)
{
    const char *who = "twm_kv_copy_pages";
    if (!ctx) return api_fail(TWM_INVALID_HANDLE, "%s: null context", who);
    if (count == 0 || pairs == 0) return TWM_OK;
    if (!caches) return api_fail(TWM_INVALID_HANDLE, "%s: null cache", who);
    if (!sources || !targets) return api_fail(TWM_INVALID_HANDLE, "%s: null pointer", who);
    if (count > kKvMostRows) return api_fail(TWM_SHAPE_ERROR, "%s: %u caches are beyond 2^20", who, count);
    try {
        std::vector<KvView> views(count);
        for (uint32_t i = 0; i < count; i++) {
            if (int rc = check_cache(who, caches + i, &views[i])) return rc;
            const twm_kv_cache &c = caches[i], &first = caches[0];
            if (c.dtype != first.dtype || c.pages != first.pages || c.page_tokens != first.page_tokens || c.kv_heads != first.kv_heads ||
                c.head_dim != first.head_dim)
                return api_fail(TWM_SHAPE_ERROR, "%s: the caches are not of one shape and type", who);
        }
        // a target may be named once, and not as a source: found among the sorted pages of both, targets ahead of sources
        std::vector<uint64_t> named;
        named.reserve(2 * (size_t)pairs);
        for (uint32_t i = 0; i < pairs; i++) {
            if (sources[i] >= caches[0].pages || targets[i] >= caches[0].pages)
                return api_fail(TWM_SHAPE_ERROR, "%s: page %u to page %u of %u", who, sources[i], targets[i], caches[0].pages);
            named.push_back(2ull * targets[i]);
            named.push_back(2ull * sources[i] + 1);
        }
        std::sort(named.begin(), named.end());
        for (size_t i = 1; i < named.size(); i++)
            if ((named[i - 1] & 1) == 0 && named[i] >> 1 == named[i - 1] >> 1)
                return api_fail(TWM_SHAPE_ERROR, "%s: page %u is a target and named again", who, (unsigned)(named[i] >> 1));
        DeviceGuard on(ctx);
        HIP_TRY(on.status, TWM_DEVICE_ERROR, who);
        HIP_TRY(launch_kv_copy_pages(ctx->stream, views.data(), count, sources, targets, pairs), TWM_DEVICE_ERROR, who);
        return TWM_OK;
    } catch (const std::bad_alloc &) {
        return api_fail(TWM_MEMORY_ERROR, "%s: out of host memory", who);
    }
}

}  // extern "C"
