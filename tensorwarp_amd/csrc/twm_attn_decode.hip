// Attention of one new token per sequence over a paged key-value cache.
//
//   out[h] = sum_t w_t v_t / sum_t w_t,   w_t = 2^(15 + c (s_t - m)),   s_t = q[h] . k_t,   c = scale * log2(e) * the head's scale of keys
//
// with m the largest s_t so far; whatever was summed is multiplied by 2^(c (m - m')) when it grows to m'.  (The difference comes before the
// product: c m by itself would be rounded, and where scores are large its rounding would be a power of two in the weight.)
//
// Keys and values are read once, from memory to registers, whatever the number of query heads that share them: up to sixteen heads are the
// columns of the matrix instructions (16 x 16 x 32), thirty-two tokens at a time.  Scores come transposed, S^T = K Q^T, which leaves a lane
// with eight neighbouring tokens of one head: the operand that O^T = V^T P^T asks for, without an exchange between lanes.  The instruction
// takes the tokens in any order that both operands agree on, so rows 4 g + i of its two blocks are tokens 8 g + i and 8 g + 4 + i.  V^T comes from
// LDS through the transposing reads; every wave has a buffer of its own there and no other wave is waited for.
//
// Weights enter the product as two f16 terms, the first one cut off and the second what it leaves.  A term that is 0 times an infinite value is NaN,
// where the formula has that infinity: a wave whose sums have come to NaN goes over its tokens once more with terms of at least the smallest f16 number
// (both 2^-38 of the largest weight; what is not seen has values of 0).
//
// All tokens of all sequences, in steps of 128, are dealt out evenly among as many workgroups for each key-value head as the chip holds at once,
// which find their share from the lengths by themselves: a long sequence is cut into many shares, several short ones make one.  What a share
// holds of a sequence that others hold too goes to scratch, and a second kernel joins it.  (Joining by the last workgroup to arrive cost the same
// 5 us.)  Where no sequence is long, each sequence and unit has a workgroup of more waves to itself and nothing is joined.
//
// Bound by the reading of the cache where it is long: 32 sequences of up to 8192 tokens, 28 heads on 4 of 128 f16 values, 60 us (4.6 TB/s; a copy
// reaches 5.1); 48 of up to 4096, 32 heads on 32, e4m3, 152 us (5.5 TB/s); 32 of up to 4096, 16 heads on 8 of 256, 106 us (5.2 TB/s), e4m3 64 (4.3); one
// sequence of 131072 58 us, of 32768 20.7 - 22.9 (two launches and eight steps a share are what is left), and of 777 tokens, 14 heads of 64
// values, 9.2 us, which are the chain from the length by the table and the keys to the sums.
#include "twm_kv.h"
#include "twm_slices.h"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace twm {

namespace {

typedef int int2v __attribute__((ext_vector_type(2)));

constexpr uint32_t kDecodeHeads = 16;   // query heads of one unit: columns of a matrix instruction
constexpr uint32_t kDecodeWaves = 4, kDecodeStep = 32 * kDecodeWaves;   // of shares
constexpr int kNoScore = 0xFF800000;   // -infinity

struct Decode {
    AttnArgs a;
    float *parts;          // [2 * workgroups][heads of a unit][dim]
    float2 *part_sums;     // [2 * workgroups][heads of a unit]: largest score, sum of weights
    uint32_t units, tiles;   // units: tiles of up to sixteen heads for each key-value head
    uint32_t heads;          // of a unit
    uint32_t shares;         // of each unit: workgroup unit * shares + share of the first kernel
    Divisor by_shares, by_tiles, by_group;
};

// The tokens that a sequence sees, from `first`, the multiple of 32 at or below the first one, in steps of 128
struct Span {
    int lo, hi, first;
    uint32_t steps;
};
__device__ __forceinline__ Span span_of(const Decode &d, int length)
{
    Span s;
    s.hi = min(length, (int)(d.a.seqs.table_stride << d.a.kv.page_shift));
    s.lo = d.a.window ? max(0, max(length, 0) - (int)d.a.window) : 0;
    s.first = s.lo & ~31;
    s.steps = s.hi > s.lo && d.a.kv.pages ? (uint32_t)(s.hi - s.first + (int)kDecodeStep - 1) / kDecodeStep : 0u;
    return s;
}

// The steps of 64 sequences, a lane each, and the sums up to it (64 sequences have less than 2^29)
struct Lengths {
    int length;
    uint32_t steps, up_to, all;
};
__device__ __forceinline__ Lengths lengths_from(const Decode &d, uint32_t base)
{
    const uint32_t s = base + (threadIdx.x & 63u);
    Lengths l;
    l.length = s < d.a.seqs.seqs ? d.a.seqs.lengths[s] : 0;
    l.steps = span_of(d, l.length).steps;
    l.up_to = wave_sum_up_to(l.steps);
    l.all = __builtin_amdgcn_readlane(l.up_to, 63);
    return l;
}

// Share w of a unit's `total` steps begins here; every share has a step at least, where there are as many.  (In 64 bits beyond 2^20: any
// rounding would do that is the same for all who ask.)
__device__ __forceinline__ uint64_t share_begin(const Decode &d, uint64_t total, uint32_t w)
{
    if (total <= d.shares) return min((uint64_t)w, total);
    if (total < 1u << 20) return d.by_shares((uint32_t)total * w);
    return w == d.shares ? total : (uint64_t)((double)total * w / d.shares);
}

__device__ __forceinline__ float max_over_quarters(float v)
{
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float sum_over_quarters(float v)
{
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// Workgroups of four waves that share a compute unit, by their registers; waves of a workgroup that has a sequence to itself
template <int D, bool E4M3> constexpr uint32_t kDecodePerUnit = D == 256 ? (E4M3 ? 2 : 1) : D == 128 ? (E4M3 ? 3 : 2) : 3;
template <int D, bool E4M3> constexpr uint32_t kDecodeWholeWaves = D == 64 ? 16 : D == 128 || E4M3 ? 8 : 4;

}  // namespace

// WHOLE: a workgroup has a sequence and unit to itself, sequence first_seq + blockIdx.x / units
template <int D, bool E4M3, uint32_t WAVES, bool WHOLE>
__global__ __launch_bounds__(64 * WAVES, (WHOLE ? WAVES / 4 : kDecodePerUnit<D, E4M3>)) void k_attn_decode(const Decode d, uint32_t first_seq)
{
    constexpr uint32_t THREADS = 64 * WAVES, STEP = 32 * WAVES;
    constexpr uint32_t kRow = D * (E4M3 ? 1 : 2);          // bytes of a token
    constexpr uint32_t kStride = kRow + 32;                // in LDS: four rows that are read at once lie in different banks
    constexpr uint32_t kBuffer = 32 * kStride > kDecodeHeads * D * 4 ? 32 * kStride : kDecodeHeads * D * 4;   // also a wave's results
    constexpr int NK = kRow / 64, NV = 32 * kRow / 1024;   // loads per lane: of each block of 16 keys, of 32 values
    constexpr uint32_t kLanesPerRow = kRow / 16, kRowsPerLoad = 64 / kLanesPerRow;
    __shared__ __align__(16) char buffers[WAVES][kBuffer];
    __shared__ half8 queries[D / 32 * 64];
    __shared__ float tops[WAVES][kDecodeHeads], sums[WAVES][kDecodeHeads];
    const AttnArgs &a = d.a;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63u, quarter = lane >> 4, col = lane & 15u;
    char *const buffer = buffers[wave];

    const uint32_t pair = d.by_shares(blockIdx.x), unit = WHOLE ? blockIdx.x - pair * d.shares : pair, share = WHOLE ? 0u : blockIdx.x - unit * d.shares;
    const uint32_t kv_head = d.by_tiles(unit), head0 = kv_head * a.group + (unit - kv_head * d.tiles) * kDecodeHeads;
    const uint32_t heads = min(kDecodeHeads, (kv_head + 1) * a.group - head0);
    auto clear = [&](uint32_t s) {   // a row without tokens
        for (uint32_t i = threadIdx.x; i < heads * D / 8; i += THREADS) *(half8_any *)(a.out + (size_t)s * a.out_stride + head0 * D + 8u * i) = half8{};
    };
    Lengths l;
    uint64_t total = 0, at = 0, end = 1, before = 0;
    uint32_t base = 0, seq = first_seq + pair;
    if constexpr (WHOLE) {
        l.length = a.seqs.lengths[seq];
        if (span_of(d, l.length).steps == 0) {
            clear(seq);
            return;
        }
    } else {
        // Up to 64 sequences are looked up once
        l = lengths_from(d, 0);
        total = l.all;
        for (uint32_t b = 64; b < a.seqs.seqs; b += 64) total += lengths_from(d, b).all;
        for (uint32_t s = share; s < a.seqs.seqs; s += d.shares)   // (every share sees to some)
            if (span_of(d, a.seqs.lengths[s]).steps == 0) clear(s);
        at = share_begin(d, total, share);
        end = share_begin(d, total, share + 1);
        if (at >= end) return;
        // the sequence in which the share begins
        for (;;) {
            const uint64_t past = __ballot(before + l.up_to > at);
            if (past) {
                const uint32_t lane_of = (uint32_t)__builtin_ctzll(past);
                seq = base + lane_of;
                before += lane_of == 0 ? 0u : (uint32_t)__builtin_amdgcn_readlane(l.up_to, lane_of - 1);
                break;
            }
            before += l.all;
            base += 64;
            l = lengths_from(d, base);
        }
    }
    const uint32_t part = 2 * blockIdx.x;
    const uint32_t page_mask = (1u << a.kv.page_shift) - 1u;
    for (bool first_of_share = true; at < end; first_of_share = false) {
        if (!WHOLE && seq - base >= 64) {
            base += 64;
            l = lengths_from(d, base);
        }
        const Span span = span_of(d, WHOLE ? l.length : __builtin_amdgcn_readlane(l.length, seq - base));
        if (!WHOLE && span.steps == 0) {
            seq++;
            continue;
        }
        // this share's steps of the sequence
        const uint32_t step0 = (uint32_t)(at - before), step1 = (uint32_t)min((uint64_t)span.steps, step0 + (end - at));
        const float c = exponent_factor(a.kv, a.scale, kv_head);

        // Q^T: a lane's head's values, in the order in which it holds keys
        for (uint32_t x = threadIdx.x; x < D / 32 * 64; x += THREADS) {
            const uint32_t i = x >> 6, head = min(x & 15u, heads - 1), g = x >> 4 & 3u;
            queries[x] = *(const half8_any *)(a.q + (size_t)seq * a.q_stride + (head0 + head) * D + (E4M3 ? (i / 2) * 64 + g * 16 + (i % 2) * 8 : i * 32 + g * 8));
        }

        float top, sum;
        float4v o[D / 16];

        // Pages of this wave's tokens, 32 a step: a lane looks one of a step's halves up, the wave those of 32 steps at once
        const int *table = a.seqs.tables + (size_t)seq * a.seqs.table_stride;
        const char *const k_base = (const char *)a.kv.k, *const v_base = (const char *)a.kv.v;
        int page_of = -1, page0 = -1, page1 = -1;
        uint32_t looked_up;
        auto pages_of = [&](int t) {
            if ((looked_up & 31u) == 0) {
                const int64_t token = t + (int64_t)(lane >> 1) * (int)STEP + (int)(lane & 1u) * 16;
                page_of = token < span.hi ? table[(uint32_t)token >> a.kv.page_shift] : -1;
            }
            page0 = __builtin_amdgcn_readlane(page_of, 2 * (looked_up & 31u));
            page1 = __builtin_amdgcn_readlane(page_of, 2 * (looked_up & 31u) + 1);
            looked_up++;
        };
        uint4v k[2][NK], v[NV];
        bool k_there = false;   // whether both pages are inside the pool
        auto load = [&](int t) {
            const bool in0 = (uint32_t)page0 < a.kv.pages, in1 = (uint32_t)page1 < a.kv.pages;
            k_there = in0 && in1;
            // what lies outside is read from the pool's first page, and left out
            const size_t chunk0 = kv_chunk(a.kv, in0 ? (uint32_t)page0 : 0u, kv_head) + ((uint32_t)t & page_mask) * D;
            const size_t chunk1 = kv_chunk(a.kv, in1 ? (uint32_t)page1 : 0u, kv_head) + ((uint32_t)(t + 16) & page_mask) * D;
            const size_t bytes0 = chunk0 * (E4M3 ? 1 : 2), bytes1 = chunk1 * (E4M3 ? 1 : 2);
            const char *key = k_base + (col < 8 ? bytes0 : bytes1) + (8u * ((col >> 2) & 1u) + (col & 3u)) * kRow + quarter * 16u;
#pragma unroll
            for (int b = 0; b < 2; b++)
#pragma unroll
                for (int i = 0; i < NK; i++) k[b][i] = *(const uint4v *)(key + b * 4 * kRow + i * 64);
            const uint32_t v_off = lane / kLanesPerRow * kRow + lane % kLanesPerRow * 16u;
#pragma unroll
            for (int i = 0; i < NV; i++) {
                const uint32_t row = i * kRowsPerLoad;   // (a load's rows lie in one half)
                v[i] = *(const uint4v *)(v_base + (row < 16 ? bytes0 + row * kRow : bytes1 + (row - 16) * kRow) + v_off);
            }
        };
        const int stop = WHOLE ? span.hi : min(span.hi, span.first + (int)(step1 * STEP));
        for (uint32_t least = 0;; least = 0x00010001u) {   // the least of two f16 terms: 0, or 2^-24
            top = -INFINITY;
            sum = 0.f;
#pragma unroll
            for (int i = 0; i < D / 16; i++) o[i] = float4v{0.f, 0.f, 0.f, 0.f};
            looked_up = 0;
            int t = span.first + (int)(step0 * STEP + wave * 32u);
            if (t < stop) {
                pages_of(t);
                load(t);
            }
            if (least == 0) __syncthreads();
            for (; t < stop; t += (int)STEP) {
                const bool whole = k_there && t >= span.lo && t + 32 <= span.hi;
                const bool in0 = (uint32_t)page0 < a.kv.pages, in1 = (uint32_t)page1 < a.kv.pages;
                // values to LDS; what is not seen is zeros there, whatever it may be in memory
#pragma unroll
                for (int i = 0; i < NV; i++) {
                    const uint32_t row = i * kRowsPerLoad + lane / kLanesPerRow;
                    if (!whole) {
                        const int token = t + (int)row;
                        const bool seen = token >= span.lo && token < span.hi && (row < 16 ? in0 : in1);
                        v[i] = seen ? v[i] : uint4v{0u, 0u, 0u, 0u};
                    }
                    *(uint4v *)(buffer + row * kStride + lane % kLanesPerRow * 16u) = v[i];
                }
                float4v s[2];
#pragma unroll
                for (int b = 0; b < 2; b++) {
                    s[b] = float4v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int i = 0; i < D / 32; i++) {
                        half8 key;
                        if constexpr (E4M3)
                            key = to_f16(k[b][i / 2][(i % 2) * 2], k[b][i / 2][(i % 2) * 2 + 1]);
                        else
                            key = __builtin_bit_cast(half8, k[b][i]);
                        s[b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(key, queries[i * 64 + lane], s[b], 0, 0, 0);
                    }
                }
                const int next = t + (int)STEP;
                if (next < stop) {
                    pages_of(next);
                    load(next);
                }
                // scores of tokens t + 8 quarter + 4 b + i
                if (!whole) {
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        const int token = t + 8 * (int)quarter + i;
                        const bool one = token >= span.lo && token < span.hi && (quarter < 2 ? in0 : in1);
                        s[i / 4][i % 4] = one ? s[i / 4][i % 4] : __int_as_float(kNoScore);
                    }
                }
                float most = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])), fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
                most = fmaxf(top, max_over_quarters(most));
                if (__any(most > top)) {
                    const float by = shrink(top, most, c);
                    sum *= by;
#pragma unroll
                    for (int i = 0; i < D / 16; i++) o[i] *= by;
                    top = most;
                }
                const float from = top == -INFINITY ? 0.f : top;
                half2v p_hi[4], p_lo[4];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float x = __builtin_amdgcn_exp2f(fmaf(s[i / 2][(2 * i) % 4] - from, c, 15.0f)), y = __builtin_amdgcn_exp2f(fmaf(s[i / 2][(2 * i) % 4 + 1] - from, c, 15.0f));
                    sum += x + y;
                    p_hi[i] = __builtin_bit_cast(half2v, __builtin_amdgcn_cvt_pkrtz(x, y));
                    p_lo[i] = __builtin_bit_cast(half2v, __builtin_amdgcn_cvt_pkrtz(x - (float)p_hi[i][0], y - (float)p_hi[i][1]));
                    if constexpr (!E4M3) {
                        p_hi[i] = __builtin_elementwise_max(p_hi[i], __builtin_bit_cast(half2v, least));
                        p_lo[i] = __builtin_elementwise_max(p_lo[i], __builtin_bit_cast(half2v, least));
                    }
                }
                const half8 hi = {p_hi[0][0], p_hi[0][1], p_hi[1][0], p_hi[1][1], p_hi[2][0], p_hi[2][1], p_hi[3][0], p_hi[3][1]};
                const half8 lo = {p_lo[0][0], p_lo[0][1], p_lo[1][0], p_lo[1][1], p_lo[2][0], p_lo[2][1], p_lo[3][0], p_lo[3][1]};
                // (the wave's own stores have reached LDS: its reads come after them, in order)
#pragma unroll
                for (int i = 0; i < D / 16; i++) {
                    half8 value;
                    if constexpr (E4M3) {
                        const int2v codes = __builtin_amdgcn_ds_read_tr8_b64_v2i32(
                            (TWM_LDS(int2v) *)(buffer + (8u * quarter + (col >> 1)) * kStride + 16u * i + 8u * (col & 1u)));
                        value = to_f16((unsigned)codes[0], (unsigned)codes[1]);
                    } else {
                        const char *from = buffer + (8u * quarter + (col >> 2)) * kStride + 32u * i + 8u * (col & 3u);
                        const half4 x = __builtin_bit_cast(half4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((TWM_LDS(short4v) *)from));
                        const half4 y = __builtin_bit_cast(half4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((TWM_LDS(short4v) *)(from + 4 * kStride)));
                        value = half8{x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
                    }
                    o[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(value, hi, o[i], 0, 0, 0);
                    o[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(value, lo, o[i], 0, 0, 0);
                }
            }
            if (E4M3 || least != 0) break;   // (e4m3 has no infinity)
            float4v all = o[0];
#pragma unroll
            for (int i = 1; i < D / 16; i++) all += o[i];
            const float one = (all[0] + all[1]) + (all[2] + all[3]);
            if (!__any(one != one)) break;
        }

        // the waves' sums, brought to the largest score of all and added in wave order
        sum = sum_over_quarters(sum);
        if (lane < 16) {
            tops[wave][col] = top;
            sums[wave][col] = sum;
        }
        __syncthreads();
        float most = top;
#pragma unroll
        for (uint32_t w = 0; w < WAVES; w++) most = fmaxf(most, tops[w][col]);
        const float by = shrink(top, most, c);
#pragma unroll
        for (int i = 0; i < D / 16; i++) *(float4v *)(buffer + (col * D + 16 * i + 4 * quarter) * 4) = o[i] * by;
        __syncthreads();
        const bool all = WHOLE || (step0 == 0 && step1 == span.steps);
        const float v_scale = E4M3 && a.kv.v_scales ? a.kv.v_scales[kv_head] : 1.0f;
        for (uint32_t i = threadIdx.x; i < heads * (D / 4); i += THREADS) {
            const uint32_t h = i / (D / 4), x = i % (D / 4) * 4;
            float4v r = *(const float4v *)(buffers[0] + (h * D + x) * 4);
#pragma unroll
            for (uint32_t w = 1; w < WAVES; w++) r += *(const float4v *)(buffers[w] + (h * D + x) * 4);
            float m = tops[0][h], l = 0.f;
#pragma unroll
            for (uint32_t w = 1; w < WAVES; w++) m = fmaxf(m, tops[w][h]);
#pragma unroll
            for (uint32_t w = 0; w < WAVES; w++) l += sums[w][h] * shrink(tops[w][h], m, c);
            if (all) {
                const float to = l == 0.f ? 0.f : v_scale / l;
                if (l == 0.f) r = float4v{0.f, 0.f, 0.f, 0.f};   // (all scores are -infinity, whatever the values)
                *(half4_any *)(a.out + (size_t)seq * a.out_stride + (head0 + h) * D + x) =
                    half4{(_Float16)(r[0] * to), (_Float16)(r[1] * to), (_Float16)(r[2] * to), (_Float16)(r[3] * to)};
            } else {
                // a share holds at most two parts: of the unit in which it begins, and of the one in which it ends
                const size_t slot = (size_t)(first_of_share ? part : part + 1) * d.heads + h;
                *(float4v *)(d.parts + slot * D + x) = r;
                if (x == 0) d.part_sums[slot] = float2{m, l};
            }
        }
        if (WHOLE) return;
        __syncthreads();   // (the buffers are the waves' own again)
        at += step1 - step0;
        before += span.steps;
        seq++;
    }
}

// Joins what several shares hold of a unit: a workgroup per query head and sequence.  D / 4 lanes hold a part, as many at a time as THREADS do, four
// on their way.
template <int D, uint32_t THREADS> __global__ __launch_bounds__(THREADS) void k_attn_join(const Decode d)
{
    constexpr uint32_t kLanes = D / 4, kAtOnce = THREADS / kLanes, kAhead = 4;
    __shared__ float4v results[kAtOnce][kLanes];
    __shared__ float2 sums[kAtOnce];
    const AttnArgs &a = d.a;
    const uint32_t seq = blockIdx.x, head = blockIdx.y, kv_head = d.by_group(head), in_group = head - kv_head * a.group;
    const uint32_t unit = kv_head * d.tiles + in_group / kDecodeHeads, h = in_group % kDecodeHeads;
    uint64_t total = 0, begin = 0;
    uint32_t steps = 0;
    for (uint32_t base = 0; base < a.seqs.seqs; base += 64) {
        const Lengths l = lengths_from(d, base);
        if (seq - base < 64u) {
            steps = __builtin_amdgcn_readlane(l.steps, seq - base);
            begin = total + __builtin_amdgcn_readlane(l.up_to, seq - base) - steps;
        }
        total += l.all;
    }
    if (steps == 0) return;
    const uint64_t end = begin + steps;
    // the shares that hold its first and its last step
    auto share_of = [&](uint64_t at) {
        // (where steps are fewer than shares, step and share are one)
        uint32_t w = total <= d.shares ? (uint32_t)at : (uint32_t)min((uint64_t)(d.shares - 1), (uint64_t)((float)at / (float)total * d.shares));
        while (share_begin(d, total, w) > at) w--;
        while (share_begin(d, total, w + 1) <= at) w++;
        return w;
    };
    const uint32_t first = share_of(begin), last = share_of(end - 1);
    if (first == last) return;
    const uint32_t first_slot = 2 * (unit * d.shares + first) + (share_begin(d, total, first) < begin ? 1u : 0u);
    auto slot_of = [&](uint32_t w) { return (size_t)(w == first ? first_slot : 2 * (unit * d.shares + w)) * d.heads + h; };
    const float c = exponent_factor(a.kv, a.scale, kv_head), v_scale = a.kv.v_scales ? a.kv.v_scales[kv_head] : 1.0f;
    const uint32_t group = threadIdx.x / kLanes, lane = threadIdx.x % kLanes;
    float top = -INFINITY, sum = 0.f;
    float4v o = {0.f, 0.f, 0.f, 0.f};
    auto add = [&](const float2 &s, const float4v &part) {
        const float most = fmaxf(top, s.x), keep = shrink(top, most, c), by = shrink(s.x, most, c);
        sum = sum * keep + s.y * by;
        o = o * keep + part * by;
        top = most;
    };
    for (uint32_t w = first + group; w <= last; w += kAtOnce * kAhead) {
        float2 s[kAhead];
        float4v part[kAhead];
#pragma unroll
        for (uint32_t i = 0; i < kAhead; i++) {
            const size_t slot = slot_of(min(w + kAtOnce * i, last));
            s[i] = d.part_sums[slot];
            part[i] = *(const float4v *)(d.parts + slot * D + 4u * lane);
        }
#pragma unroll
        for (uint32_t i = 0; i < kAhead; i++)
            if (w + kAtOnce * i <= last) add(s[i], part[i]);
    }
    // the upper half of those that hold something joins the lower one (one after the other: 32768 tokens 21.4 us, now 20.8, of heads of 64 15.2 and 13.3)
#pragma unroll
    for (uint32_t half = kAtOnce / 2; half != 0; half /= 2) {
        if (group >= half && group < 2 * half) {
            results[group][lane] = o;
            if (lane == 0) sums[group] = float2{top, sum};
        }
        __syncthreads();
        if (group < half) add(sums[group + half], results[group + half][lane]);
    }
    if (group != 0) return;
    const float to = sum == 0.f ? 0.f : v_scale / sum;
    if (sum == 0.f) o = float4v{0.f, 0.f, 0.f, 0.f};
    *(half4_any *)(a.out + (size_t)seq * a.out_stride + head * D + 4u * lane) =
        half4{(_Float16)(o[0] * to), (_Float16)(o[1] * to), (_Float16)(o[2] * to), (_Float16)(o[3] * to)};
}

hipError_t launch_attn_decode(hipStream_t s, const AttnArgs &a, void *scratch, size_t scratch_bytes)
{
    Decode d;
    d.a = a;
    d.tiles = (a.group + kDecodeHeads - 1) / kDecodeHeads;
    d.units = a.kv.kv_heads * d.tiles;
    d.heads = std::min(a.group, kDecodeHeads);
    d.by_tiles = Divisor(d.tiles);
    d.by_group = Divisor(a.group);
    const uint64_t capacity = (uint64_t)a.seqs.table_stride << a.kv.page_shift, seen = std::min(capacity, a.window ? (uint64_t)a.window + 31 : capacity);
    auto launch = [&](auto dim, auto e4m3) {
        constexpr int D = decltype(dim)::value;
        constexpr bool E4M3 = decltype(e4m3)::value;
        constexpr uint32_t WHOLE_WAVES = kDecodeWholeWaves<D, E4M3>;
        // No shares, and nothing to join, where no sequence can be long by the table's width, by as much more as there are many.  28 heads on 4 of 128 values:
        // one sequence of 100 tokens 6.6 us, 10.7 in shares; 32 sequences up to 512 11.0 and 13.1, 200 35 and 40; up to 2048, 200 sequences 90 and 98;
        // but one of 512 10.0 and 9.9, up to 4096 200 sequences 166 either way, 48 of 32 heads in e4m3 160 and 155, and one of 1024 tokens, four steps of eight
        // waves, 14.4 and 9.9.  And none among so many sequences that each share's way through their lengths costs more than most waits: 1023
        // up to 512 tokens 179 in shares, 1024 154 without, up to 8192 1485 and 1454, 16384 up to 64 (7 heads on one) 2384 and 352.  The price
        // is one that is much longer than the others: one of 16384 tokens among 1024 of 100 189 (among 1023, in shares, 121), of 131072 1390 (177).
        if (seen <= std::min<uint64_t>(8, 2 + (uint64_t)a.seqs.seqs * d.units / 64) * (32 * WHOLE_WAVES) || a.seqs.seqs >= 1024) {
            d.shares = d.units;
            d.by_shares = Divisor(d.units);
            return in_slices(a.seqs.seqs, most_workgroups(64 * WHOLE_WAVES) / d.units, [&](uint32_t seq, uint32_t here) {
                hipLaunchKernelGGL((k_attn_decode<D, E4M3, WHOLE_WAVES, true>), dim3(here * d.units), dim3(64 * WHOLE_WAVES), 0, s, d, seq);
                return hipGetLastError();
            });
        }
        // as many workgroups as the chip holds at once, or as there may be steps
        const uint64_t most_steps = (seen + kDecodeStep - 1) / kDecodeStep * a.seqs.seqs;
        d.shares = (uint32_t)std::max<uint64_t>(1, std::min<uint64_t>(256 * kDecodePerUnit<D, E4M3> / d.units, most_steps));
        d.by_shares = Divisor(d.shares);
        const size_t slots = 2 * (size_t)d.shares * d.units * d.heads;
        d.part_sums = (float2 *)scratch;
        d.parts = (float *)((char *)scratch + (slots * sizeof(float2) + 255) / 256 * 256);
        if ((size_t)((char *)(d.parts + slots * D) - (char *)scratch) > scratch_bytes) return hipErrorOutOfMemory;   // (at most 17 MB of 256)
        hipLaunchKernelGGL((k_attn_decode<D, E4M3, kDecodeWaves, false>), dim3(d.shares * d.units), dim3(64 * kDecodeWaves), 0, s, d, 0u);
        if (const hipError_t error = hipGetLastError(); error != hipSuccess) return error;
        // sixteen parts of 128 values at once for few sequences, which have many, four otherwise (32 sequences up to 1024 tokens 20.7 us with
        // sixteen, 18.9 with four; one of 32768 21.3 and 25.3; both before the halves joined)
        if (a.seqs.seqs < 8)
            hipLaunchKernelGGL((k_attn_join<D, 512>), dim3(a.seqs.seqs, a.q_heads), dim3(512), 0, s, d);
        else
            hipLaunchKernelGGL((k_attn_join<D, 128>), dim3(a.seqs.seqs, a.q_heads), dim3(128), 0, s, d);
        return hipGetLastError();
    };
    auto of_type = [&](auto dim) { return a.kv.e4m3 ? launch(dim, std::true_type{}) : launch(dim, std::false_type{}); };
    return a.kv.dim == 64    ? of_type(std::integral_constant<int, 64>{})
           : a.kv.dim == 128 ? of_type(std::integral_constant<int, 128>{})
                             : of_type(std::integral_constant<int, 256>{});
}

}  // namespace twm
