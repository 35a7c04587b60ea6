// Causal attention of packed rows over a paged key-value cache.
//
//   out[row][h] = sum_t w_t v_t / sum_t w_t,   w_t = 2^(8 + c (s_t - r)),   s_t = q . k_t,   c = scale * log2(e) * the head's scale of keys
//
// over the tokens t that the row sees, r a reference for the row's scores: the largest one when it was set, moved (and the sums with
// it) only where a weight would pass 2^15, so that sums are rarely touched again and f16 holds the weights with all of its digits down to 2^-22
// of the largest.
// A weight enters its product, and the sum that divides it, as the one f16 that it is rounded to: errors of 2.2 - 2.8e-4 of a result's norm, 2.0e-4 being the
// f16 result's own rounding.  A second term, as twm_attn_decode has it, would be half of the products again, and these are half of a long prompt's time.
//
// A workgroup takes 128 queries (of 256 values 64) of one key-value head -- tokens times the query heads that share it, so that short prompts fill
// tiles too -- and its four waves 32 each.  Keys and values come through LDS, tile by tile, the next tile on its way while this one is worked on;
// f16 ones directly, 16 bytes a lane, e4m3 ones through registers, where they become f16.  Scores are transposed, S^T = K Q^T: a
// lane then holds the scores of one query, row maxima need one exchange between lanes, and the weights already lie as O^T = V^T P^T wants
// its operand (the product takes tokens in any order that both operands agree on).  V^T comes from LDS through the transposing reads.
// Units of 16 bytes are stored at their place XOR their row's number, so that the rows which one instruction reads lie in different banks.
//
// Where a tile holds tokens that some of the queries do not see, weights alone would not keep an infinity or a NaN away from these (0 times
// either is NaN): there values are looked through first, rows that nobody sees become zeros, and if anything not finite is left, the tile's
// products are made one token at a time, for those who see it.  So they are once more in all tiles where sums came to NaN: an infinite value times a weight
// that f16 rounds to 0 is NaN in a matrix product, where the formula has that infinity.
//
// Bound by no single unit where prompts are long: matrix units are busy half of the time, vector instructions (the exponentials above all) nearly as long, LDS
// a fourth; two workgroups a compute unit cover one another in part.  8192 rows, 28 heads on 4 of 128 f16 values, 505 - 534 us (900 - 950 TFLOP/s of the
// halves that are seen; a large matrix product reaches 1310).  Heads of 64 have half the products for as many exponentials: vector instructions two
// thirds of the time, 300 us (800 TFLOP/s).  Workgroups of eight waves
// that take turns with products and exponentials cost their barriers (580 - 596), blocks of products between blocks of exponentials in one wave the
// registers (579), and 64 queries a wave with the next tile's scores beside this one's exponentials leave one wave a SIMD (heads of 64: 376, with 32 queries
// 309; of 128 they spill).  Short prompts are the way from the sequence by its pages to the keys, and tiles on the diagonal, which cost two whole ones: 37 rows, 14
// heads of 64, 5.3 us; 2048 rows in seven prompts 22.7 us, of which the longest's eleven tiles are half.
#include "twm_kv.h"
#include "twm_slices.h"

#include <algorithm>
#include <cfloat>
#include <cmath>
#include <type_traits>

namespace twm {

namespace {

typedef float float16v __attribute__((ext_vector_type(16)));

constexpr uint32_t kPromptWaves = 4;
template <int D> constexpr uint32_t kPromptRows = D == 256 ? 64 : 128;   // of a workgroup
constexpr int kPromptTile = 64;                                          // tokens of a tile

__device__ __forceinline__ float max_of_halves(float v)
{
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float sum_of_halves(float v)
{
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// What is not finite times 0 is NaN, and stays in the sum
__device__ __forceinline__ half2v times_0(uint4v v, half2v sum)
{
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t pair = v[i];   // (a cast of v[i] itself would take the first one's bits)
        sum = __builtin_elementwise_fma(__builtin_bit_cast(half2v, pair), half2v{(_Float16)0.f, (_Float16)0.f}, sum);
    }
    return sum;
}

struct Prompt {
    AttnArgs a;
    float4v *parts;       // [workgroups][dim / 4][rows of a workgroup], for rows that several workgroups share the tokens of
    float2 *part_sums;    // [workgroups][rows]: reference, sum of weights
    uint32_t tiles, splits, first_tile;   // splits: the most workgroups that share a tile of rows
    float balance;                        // (see parts_of)
    Divisor by_group, by_kv_heads, by_splits;
};

// What a workgroup works on: `rows` rows (tokens times heads of a group) of sequence seq, of which it has those from row0 on
struct Rows {
    uint32_t seq, row0, rows;
    int start, before, first, last;   // the sequence's first row and its position; tokens that any of the workgroup's rows sees: first .. last - 1
};
__device__ __forceinline__ int prompt_begin(const AttnArgs &a, int position) { return a.window ? max(0, max(position, -1) + 1 - (int)a.window) : 0; }

// What a sequence takes of the tiles: those of EACH rows that its rows make begin at tile start * group / EACH + s, which leaves each sequence as
// many as it has, or one more, and needs no sum over those before it.  Tile `back` from the end: its sequence is the last one that begins at or before
// it, found among 64 at once; false: nothing is there.
template <uint32_t EACH> __device__ __forceinline__ bool find_rows(const Prompt &job, uint32_t back, Rows *r)
{
    const AttnArgs &a = job.a;
    const uint32_t lane = threadIdx.x & 63u, at = job.tiles - 1 - back;
    auto rows_before = [&](int start) { return (uint32_t)min(max(start, 0), (int)a.rows) * a.group; };
    uint32_t base = 0, among = a.seqs.seqs;
    int end_of, length_of;
    for (;;) {
        const uint32_t stride = (among + 63u) / 64u, s = base + min(lane * stride, among - 1);
        const int start = a.seqs.starts[s], end = a.seqs.starts[s + 1], length = a.seqs.lengths[s];
        asm volatile("" : : "v"(start), "v"(end), "v"(length));   // (three loads on their way, not one after the other)
        const uint32_t tiles_before = rows_before(start) / EACH + s;
        const uint64_t begun = __ballot(lane * stride < among && tiles_before <= at);
        if (begun == 0) return false;
        const uint32_t found = 63u - (uint32_t)__builtin_clzll(begun);
        base += found * stride;
        among = min(stride, among - found * stride);
        if (stride == 1) {
            r->start = max(__builtin_amdgcn_readlane(start, found), 0);
            r->row0 = (at - (uint32_t)__builtin_amdgcn_readlane(tiles_before, found)) * EACH;
            end_of = __builtin_amdgcn_readlane(end, found);
            length_of = max(__builtin_amdgcn_readlane(length, found), 0);
            break;
        }
    }
    r->seq = base;
    const int tokens = min(end_of, (int)a.rows) - r->start;
    if (tokens <= 0) return false;
    r->rows = (uint32_t)tokens * a.group;
    if (r->row0 >= r->rows) return false;
    r->before = length_of - (end_of - r->start);
    r->first = prompt_begin(a, r->before + (int)job.by_group(r->row0));
    r->last = min(r->before + (int)job.by_group(min(r->row0 + EACH, r->rows) - 1) + 1, a.kv.pages ? (int)(a.seqs.table_stride << a.kv.page_shift) : 0);
    return true;
}
// How many workgroups share these rows' tokens: kLeastPart tiles each at least, and as many as balance the tiles' time with that of the parts on their way
// to the join, which reads 4 D bytes of each row and part: p = sqrt(k tiles / workgroups), k = 80, 40 and 48 for heads of 64, 128 and 256.  Heads of 128:
// 100 rows behind 600 tokens on 8 key-value heads in 2 parts 16.1 us, whole 20.4; 1024 rows of one key-value head in 4 20.2, in 2 23.6, whole 25.0; but of
// four (240 workgroups) whole 28.1, in 2 30.2, and 512 rows of four whole 17.6, in 2 19.9.  300 rows of 256 values behind 2000 tokens, on 2: in 6 parts
// 30.1, in 4 35.7, in 7 36.0.
constexpr int kLeastPart = 4;
__device__ __forceinline__ uint32_t parts_of(const Rows &r, const Prompt &job, int tile, uint32_t *tiles)
{
    const int begin = r.first & ~(tile - 1);
    *tiles = r.last > begin ? (uint32_t)(r.last - begin + tile - 1) / (uint32_t)tile : 0u;
    return max(1u, min(min(job.splits, *tiles / kLeastPart), (uint32_t)sqrtf((float)*tiles * job.balance)));
}

// The place of a unit in its row of keys (of which 16 rows are read at once) and of values (four rows, four units of each)
template <int D> __device__ __forceinline__ uint32_t key_place(uint32_t r, uint32_t unit) { return unit ^ (D == 64 ? (r >> 1) & 7u : r & 15u); }
template <int D> __device__ __forceinline__ uint32_t value_place(uint32_t r, uint32_t unit) { return unit ^ (D == 64 ? (r & 2u) << 1 : (r & 3u) << 2); }

// A tile's pages: a wave's sixteen rows (or eight) are neighbours, which lie in one; bit g: the page of tokens 16 g .. is in the pool
struct Pages {
    int mine;
    uint32_t there;
};
// A lane looks the pages of sixteen tokens up, the wave those of 1024 at once
struct PagesOf {
    const int *table;
    uint32_t pages, page_shift;
    int last, looked_up, page_of;
    uint64_t there;
    __device__ __forceinline__ void look_up(int t0)
    {
        looked_up = t0;
        const int token = t0 + 16 * (int)(threadIdx.x & 63u);
        page_of = token < last ? table[(uint32_t)token >> page_shift] : -1;
        there = __ballot((uint32_t)page_of < pages);
    }
    // of the tile at t0, and of the run of 16 in it that this wave brings in
    __device__ __forceinline__ Pages find(int t0, uint32_t run)
    {
        if (t0 - looked_up >= 1024) look_up(t0);
        const uint32_t group = (uint32_t)(t0 - looked_up) >> 4;
        return Pages{__builtin_amdgcn_readlane(page_of, group + run), (uint32_t)(there >> group) & ((1u << kPromptTile / 16) - 1u)};
    }
};

// N units of row r of a tile's values: zeros where nobody sees the row, looked through otherwise; whether any is not finite
template <int D, uint32_t N> __device__ __forceinline__ bool look_through(char *values, uint32_t r, uint32_t unit, bool dead)
{
    half2v found = {(_Float16)0.f, (_Float16)0.f};
#pragma unroll
    for (uint32_t i = 0; i < N; i++) {
        uint4v *at = (uint4v *)(values + r * D * 2 + (value_place<D>(r, unit + i) << 4));
        if (dead)
            *at = uint4v{0u, 0u, 0u, 0u};
        else
            found = times_0(*at, found);
    }
    return (__builtin_bit_cast(uint32_t, found) & 0x7FFF7FFFu) != 0;   // (a zero of either sign otherwise)
}
// Row r of a tile's values, from a unit on, to the sums of a lane's query, if that sees it
template <int D, int N> __device__ __forceinline__ void add_one(float16v (&o)[N], const char *values, uint32_t r, uint32_t unit, _Float16 weight, bool seen)
{
    const uint32_t half = threadIdx.x >> 5 & 1u;
    const float w = fmaxf((float)weight, FLT_MIN);   // (an infinite value times 0 would be NaN)
#pragma unroll
    for (int i = 0; i < N; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const half4 x = *(const half4 *)(values + r * D * 2 + (value_place<D>(r, unit + 4u * i + j) << 4) + 8u * half);
#pragma unroll
            for (int e = 0; e < 4; e++) o[i][4 * j + e] = seen ? fmaf(w, (float)x[e], o[i][4 * j + e]) : o[i][4 * j + e];
        }
}
// whether any sum is NaN, or one is infinity and another -infinity (one question for all of a lane's)
template <int N> __device__ __forceinline__ bool any_nan(const float16v (&o)[N])
{
    float one = 0.f;
#pragma unroll
    for (int i = 0; i < N; i++)
#pragma unroll
        for (int j = 0; j < 16; j++) one += o[i][j];
    return one != one;
}

// LDS of a workgroup
template <int D> constexpr uint32_t kPromptLds = 4 * kPromptTile * D * 2 + (D == 64 ? kPromptWaves * 64 * 32 * 2 + 16 : 16);
template <int D> constexpr uint32_t kPairsLds = 2 * kPromptTile * D * 2 + kPromptWaves * 2048 + kPromptWaves * 32 * 4 + 16;

}  // namespace

// Two workgroups a compute unit; of heads of 64 f16 values three, whose registers just suffice (8192 rows of 28 heads on 4 297 us, with two 308)
template <int D, bool E4M3> __global__ __launch_bounds__(256, (D == 64 && !E4M3 ? 3 : 2)) void k_attn_prompt(const Prompt job)
{
    constexpr int KT = kPromptTile, kGroups = KT / 16;   // tokens of a tile; runs of 16, each within a page
    constexpr uint32_t kUnits = D / 8, kRow = D * 2;        // of 16 bytes, bytes of a row in LDS
    constexpr uint32_t kTile = KT * kRow, kWaveRows = KT / kPromptWaves;   // bytes of a tile's keys; rows that a wave brings in
    constexpr uint32_t kRows = kPromptRows<D>;
    // two buffers of keys, then two of values; behind them room for the waves' weights, where a tile of keys is too small for them, and a flag
    // for each
    extern __shared__ __align__(16) char lds[];
    const AttnArgs &a = job.a;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63u, half = lane >> 5, col = lane & 31u;

    // the last tiles first: they have the most tokens to look at
    const uint32_t pair = job.by_splits(blockIdx.x), split = blockIdx.x - pair * job.splits, local = job.by_kv_heads(pair), kv_head = pair - local * a.kv.kv_heads;
    Rows mine;
    if (!find_rows<kRows>(job, job.first_tile + local, &mine)) return;
    const uint32_t seq = mine.seq, row0 = mine.row0, rows = mine.rows;
    const int start = mine.start, before = mine.before;
    const int capacity = a.kv.pages ? (int)(a.seqs.table_stride << a.kv.page_shift) : 0;
    uint32_t key_tiles;
    const uint32_t parts = __builtin_amdgcn_readfirstlane(parts_of(mine, job, KT, &key_tiles));
    if (split >= parts) return;

    auto begin_of = [&](int position) { return prompt_begin(a, position); };
    // this lane's query: a row behind the last one repeats it and is not stored
    const uint32_t wave_row = row0 + wave * 32u;
    const uint32_t row = wave_row + col, my_row = min(row, rows - 1);
    const uint32_t my_token = job.by_group(my_row), my_head = kv_head * a.group + (my_row - my_token * a.group);
    const int my_position = before + (int)my_token, my_begin = begin_of(my_position), my_end = min(my_position + 1, capacity);
    // the workgroup's and the wave's first and last ones
    const int low = before + (int)job.by_group(row0), high = before + (int)job.by_group(min(row0 + kRows, rows) - 1);
    const int wave_low = __builtin_amdgcn_readfirstlane(my_position), wave_high = __builtin_amdgcn_readlane(my_position, 31);
    // the tokens that anyone sees, or this part of them
    const uint32_t each_part = key_tiles / parts, one_more = key_tiles - each_part * parts;
    const int all_begin = mine.first & ~(KT - 1), first = max(mine.first, all_begin + (int)(split * each_part + min(split, one_more)) * KT);
    const int last = min(mine.last, all_begin + (int)((split + 1) * each_part + min(split + 1, one_more)) * KT);

    half8 q[D / 16];
    {
        const _Float16 *from = a.q + (size_t)(start + (int)my_token) * a.q_stride + my_head * D + 8u * half;
#pragma unroll
        for (int i = 0; i < D / 16; i++) q[i] = *(const half8_any *)(from + 16 * i);
    }
    const float c = exponent_factor(a.kv, a.scale, kv_head);
    float reference, sum;
    float16v o[D / 32];

    const uint32_t page_mask = (1u << a.kv.page_shift) - 1u;
    const int t_begin = first & ~(KT - 1);
    PagesOf pages_of{a.seqs.tables + (size_t)seq * a.seqs.table_stride, a.kv.pages, a.kv.page_shift, last, t_begin, -1, 0};
    constexpr int kLoads = (int)(kWaveRows * D * (E4M3 ? 1 : 2) / 1024);   // 1 KB each
    constexpr uint32_t kLoadUnits = D * (E4M3 ? 1 : 2) / 16, kRowsPerLoad = 64 / kLoadUnits;
    uint4v k_held[kLoads], v_held[kLoads];   // e4m3 only
    auto bring = [&](int t0, const Pages &pages, uint32_t buf) {
        const uint32_t r0 = wave * kWaveRows;
        // rows of a page outside the pool are read from its first one
        const uint32_t page = (uint32_t)pages.mine < a.kv.pages ? (uint32_t)pages.mine : 0u;
        const size_t at = (kv_chunk(a.kv, page, kv_head) + ((uint32_t)(t0 + (int)r0) & page_mask) * D) * (E4M3 ? 1 : 2);
        const char *k_from = (const char *)a.kv.k + at, *v_from = (const char *)a.kv.v + at;
#pragma unroll
        for (int i = 0; i < kLoads; i++) {
            if constexpr (E4M3) {
                k_held[i] = *(const uint4v *)(k_from + i * 1024 + lane * 16u);
                v_held[i] = *(const uint4v *)(v_from + i * 1024 + lane * 16u);
            } else {
                const uint32_t r = r0 + i * kRowsPerLoad + lane / kUnits;   // the row in the tile, and the unit that this lane's place holds
                const uint32_t row_off = i * 1024u + lane / kUnits * kRow, k_off = row_off + (key_place<D>(r, lane % kUnits) << 4),
                               v_off = row_off + (value_place<D>(r, lane % kUnits) << 4);
                char *to = lds + buf * kTile + (r0 + i * kRowsPerLoad) * kRow;
                __builtin_amdgcn_global_load_lds((const TWM_GLOBAL void *)(k_from + k_off), (TWM_LDS(void) *)to, 16, 0, 0);
                __builtin_amdgcn_global_load_lds((const TWM_GLOBAL void *)(v_from + v_off), (TWM_LDS(void) *)(to + 2 * kTile), 16, 0, 0);
            }
        }
    };
    // e4m3: what has arrived in registers becomes f16 in LDS
    auto keep = [&](uint32_t buf) {
        if constexpr (E4M3) {
#pragma unroll
            for (int i = 0; i < kLoads; i++) {
                const uint32_t r = wave * kWaveRows + i * kRowsPerLoad + lane / kLoadUnits, unit = lane % kLoadUnits * 2;
                char *to = lds + buf * kTile + r * kRow;
                *(half8 *)(to + (key_place<D>(r, unit) << 4)) = to_f16(k_held[i][0], k_held[i][1]);
                *(half8 *)(to + (key_place<D>(r, unit + 1) << 4)) = to_f16(k_held[i][2], k_held[i][3]);
                *(half8 *)(to + 2 * kTile + (value_place<D>(r, unit) << 4)) = to_f16(v_held[i][0], v_held[i][1]);
                *(half8 *)(to + 2 * kTile + (value_place<D>(r, unit + 1) << 4)) = to_f16(v_held[i][2], v_held[i][3]);
            }
        }
    };
    // whether it holds for any lane of any wave; not again before another meeting of the waves
    uint32_t *const flags = (uint32_t *)(lds + kPromptLds<D> - 16);
    auto any_wave = [&](bool mine) {
        const bool any = __any(mine);
        if (lane == 0) flags[wave] = any;
        __syncthreads();
        return (flags[0] | flags[1] | flags[2] | flags[3]) != 0;
    };
    // everything that this wave has brought in and kept has arrived, and that of the other waves
    auto arrived = [&]() {
        __builtin_amdgcn_s_waitcnt(0x0F70);   // vmcnt(0)
        __syncthreads();
    };

    const int high_begin = begin_of(high);
    uint32_t there, buf;
    Pages next;
    // Where a lane reads keys and values in the first buffers: the number of a unit enters by XOR, rows of whole blocks by addition
    const uint32_t k_at = col * kRow + (key_place<D>(col, half) << 4), v_row = 4u * half + (lane >> 2 & 3u);
    const uint32_t v_at = 2 * kTile + v_row * kRow + (value_place<D>(v_row, (lane >> 4 & 1u) * 2u + (lane >> 1 & 1u)) << 4) + (lane & 1u) * 8u;
    // S^T of the tile in buffer `tile`; element j of block b: token 32 b + 8 (j / 4) + 4 half + j % 4
    auto scores = [&](const char *tile, float16v (&s)[KT / 32]) {
#pragma unroll
        for (int b = 0; b < KT / 32; b++)
#pragma unroll
            for (int j = 0; j < 16; j++) s[b][j] = 0.f;
#pragma unroll
        for (int i = 0; i < D / 16; i++)
#pragma unroll
            for (int b = 0; b < KT / 32; b++)
                s[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(*(const half8 *)(tile + (k_at ^ i << 5) + b * 32 * kRow), q[i], s[b], 0, 0, 0);
        // keys of two steps ahead of the products, where the compiler would read those of one and wait (8192 rows 522 -> 518 us, 2048 in seven
        // prompts 25.1 -> 24.1)
        constexpr int kReads = D / 16 * (KT / 32), kAhead = 4;
        __builtin_amdgcn_sched_group_barrier(0x100, kAhead, 0);
#pragma unroll
        for (int i = 0; i < kReads - kAhead; i += 2) {
            __builtin_amdgcn_sched_group_barrier(0x8, 2, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
        }
        __builtin_amdgcn_sched_group_barrier(0x8, kAhead, 0);
    };
    // the largest score; it sets the reference where there is none yet, and nothing is summed
    auto largest = [&](const float16v (&s)[KT / 32]) {
        float most = s[0][0];
#pragma unroll
        for (int b = 0; b < KT / 32; b++)
#pragma unroll
            for (int j = 0; j < 16; j++) most = fmaxf(most, s[b][j]);
        most = max_of_halves(most);
        reference = reference == -INFINITY ? most : reference;
        return most;
    };
    // a weight would pass 2^15: the reference moves, and what is summed with it
    auto raise = [&](float most) {
        const float raised = fmaxf(reference, most), by = shrink(reference, raised, c);
        sum *= by;
#pragma unroll
        for (int i = 0; i < D / 32; i++) o[i] *= by;
        reference = raised;
    };
    // 2^(8 + c (s - reference)).  The difference comes first: a product of the reference by itself would be rounded, and where it is large its rounding would
    // be a power of two in the weight.  NEAR (up to 2^10: 2^-15 of an exponent, a 30th of what f16 takes off a weight): the product after all, one
    // instruction a score instead of two (8192 rows 529 -> 518 us, heads of 64 313 -> 304).
    auto weigh = [&](auto near, const float16v (&s)[KT / 32], half8 (&p)[KT / 16]) {
        constexpr bool NEAR = decltype(near)::value;
        const float from = reference == -INFINITY ? 0.f : reference, base = fmaf(-from, c, 8.0f);
        auto exponent = [&](float x) { return NEAR ? fmaf(x, c, base) : fmaf(x - from, c, 8.0f); };
#pragma unroll
        for (int b = 0; b < KT / 32; b++)
#pragma unroll
            for (int j = 0; j < 16; j += 2) {
                const half2v w = {(_Float16)__builtin_amdgcn_exp2f(exponent(s[b][j])), (_Float16)__builtin_amdgcn_exp2f(exponent(s[b][j + 1]))};
                sum = __builtin_amdgcn_fdot2(w, half2v{(_Float16)1.0f, (_Float16)1.0f}, sum, false);
                p[2 * b + j / 8][j % 8] = w[0];
                p[2 * b + j / 8][j % 8 + 1] = w[1];
            }
    };
    auto add_values = [&](const char *tile, const half8 (&p)[KT / 16]) {
#pragma unroll
        for (int b = 0; b < KT / 16; b++)
#pragma unroll
            for (int i = 0; i < D / 32; i++) {
                // tokens 16 b + 4 half .. + 3 and 8 further, of which a lane is given one value each
                const half4 x = __builtin_bit_cast(half4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((TWM_LDS(short4v) *)(tile + (v_at ^ i << 6) + b * 16 * kRow)));
                const half4 y = __builtin_bit_cast(half4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((TWM_LDS(short4v) *)(tile + (v_at ^ i << 6) + (b * 16 + 8) * kRow)));
                o[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(half8{x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]}, p[b], o[i], 0, 0, 0);
            }
    };
    int whole_end = min(low + 1, last);   // the last tile that everyone sees whole ends here
    int t0;
    bool advanced;
    uint32_t there_now;
    auto advance = [&]() {   // once a tile: the one behind it begins its way, and the pages of the one after that are known
        if (advanced) return;
        if (t0 + KT < last) bring(t0 + KT, next, buf ^ 1u);
        there = next.there;
        next = pages_of.find(t0 + 2 * KT, wave * kWaveRows / 16u);
        advanced = true;
    };
    auto turn = [&]() {
        if (t0 + KT < last) keep(buf ^ 1u);
        buf ^= 1u;
        t0 += KT;
        there_now = there;
        advanced = false;
        arrived();
    };
    for (;;) {
        reference = -INFINITY;
        sum = 0.f;
#pragma unroll
        for (int i = 0; i < D / 32; i++)
#pragma unroll
            for (int j = 0; j < 16; j++) o[i][j] = 0.f;
        there = buf = 0;
        next = Pages{-1, 0};
        if (t_begin < last) {
            pages_of.look_up(t_begin);
            const Pages pages = pages_of.find(t_begin, wave * kWaveRows / 16u);
            there = pages.there;
            bring(t_begin, pages, 0);
            keep(0);
            next = pages_of.find(t_begin + KT, wave * kWaveRows / 16u);
        }
        arrived();
        t0 = t_begin;
        advanced = false;
        there_now = there;
        while (t0 < last) {
            // tiles that every row of the workgroup sees whole
            float raise_to = -INFINITY;
            bool far = false;
            while (t0 >= high_begin && t0 + KT <= whole_end && there_now == (1u << kGroups) - 1u) {
                const char *const tile = lds + buf * kTile;
                advance();
                float16v s[KT / 32];
                half8 p[KT / 16];
                scores(tile, s);
                const float most = largest(s);
                if (__any((most - reference) * c > 7.0f || fabsf(reference) * c > 1024.0f)) {
                    raise_to = most;   // (rare; outside of this loop, so that the sums never move within it)
                    far = true;
                    break;
                }
                weigh(std::true_type{}, s, p);
                add_values(tile, p);
                turn();
            }
            if (__any((raise_to - reference) * c > 7.0f)) {
                raise(raise_to);
                continue;
            }
            if (t0 >= last) break;
            // one that some do not, or that lacks pages: for all waves alike, which meet in its midst; or (far) a whole one of too large scores for the short
            // form of weights, which is this wave's affair: the others may take it as above, and it meets nobody
            const char *const tile = lds + buf * kTile;
            const uint32_t present = there_now;
            advance();
            const bool idle = t0 > wave_high || t0 + KT <= begin_of(wave_low);   // nothing for this wave
            half8 p[KT / 16];
            if (!idle) {
                float16v s[KT / 32];
                scores(tile, s);
                if (t0 >= high_begin && present == (1u << kGroups) - 1u) {   // (everyone sees its beginning)
                    const int seen = my_end - t0 - 4 * (int)half;
#pragma unroll
                    for (int b = 0; b < KT / 32; b++)
#pragma unroll
                        for (int j = 0; j < 16; j++) s[b][j] = 32 * b + 8 * (j / 4) + j % 4 < seen ? s[b][j] : -INFINITY;
                } else {
#pragma unroll
                    for (int b = 0; b < KT / 32; b++)
#pragma unroll
                        for (int j = 0; j < 16; j++) {
                            // (tokens from the first seen one on, as unsigned numbers, against their number: none where the page is absent)
                            const uint32_t seen = present >> (2 * b + j / 8) & 1u ? (uint32_t)max(0, my_end - my_begin) : 0u;
                            s[b][j] = (uint32_t)(t0 + 32 * b + 8 * (j / 4) + 4 * (int)half + j % 4 - my_begin) < seen ? s[b][j] : -INFINITY;
                        }
                }
                const float most = largest(s);
                if (__any((most - reference) * c > 7.0f)) raise(most);
                weigh(std::false_type{}, s, p);
            }
            bool single = false;
            if (!far) {
                // values: rows that nobody sees become zeros, the others are looked through
                constexpr uint32_t kEach = KT * kUnits / 256, kPerRow = kUnits / kEach;
                const uint32_t looked = threadIdx.x / kPerRow, unit = threadIdx.x % kPerRow * kEach;
                const int token = t0 + (int)looked;
                const bool dead = token < first || token >= last || !(present >> (looked / 16) & 1u);
                single = any_wave(look_through<D, kEach>(lds + buf * kTile + 2 * kTile, looked, unit, dead));
                if (single) __syncthreads();   // (flags are read)
            }
            if (!idle && !single) {
                add_values(tile, p);
            } else if (!idle) {
                // the wave's weights to LDS (every wave is done with the tile's keys), then one token after the other
                _Float16 *weights = (_Float16 *)(lds + (D == 64 ? 4 * kTile : buf * kTile)) + wave * (KT * 32);
#pragma unroll
                for (int b = 0; b < KT / 16; b++)
#pragma unroll
                    for (int j = 0; j < 8; j++) weights[(16 * b + 8 * (j / 4) + 4 * (int)half + j % 4) * 32 + (int)col] = p[b][j];
                for (int r = 0; r < KT; r++) {
                    const int at = t0 + r;
                    if (at < first || at >= last || !(present >> (r / 16) & 1u)) continue;
                    const bool seen = at >= my_begin && at < my_end;
                    add_one<D>(o, tile + 2 * kTile, (uint32_t)r, 0, weights[r * 32 + (int)col], seen);
                }
            }
            turn();
        }
        if (E4M3 || max(t_begin, high_begin) + KT > whole_end) break;   // (no tile was taken as whole; e4m3 has no infinity)
        // Sums that are NaN may be an infinite value times a weight that f16 holds as 0, which is that infinity: once more, with no tile taken as whole
        if (!any_wave(any_nan(o))) break;
        whole_end = t_begin;
    }

    sum = sum_of_halves(sum);
    // (where results go is made anew: held all along it would take the registers that a third workgroup of heads of 64 needs)
    uint32_t me = lane;
    asm volatile("" : "+v"(me));
    const uint32_t out_row = wave_row + (me & 31u), out_half = me >> 5;
    if (parts > 1) {
        // to scratch, rows beside each other
        float4v *to = job.parts + (size_t)blockIdx.x * (D / 4 * kRows) + out_row - row0;
#pragma unroll
        for (int i = 0; i < D / 32; i++)
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (out_row < rows)
                    to[(8u * i + 2u * j + out_half) * kRows] = float4v{o[i][4 * j], o[i][4 * j + 1], o[i][4 * j + 2], o[i][4 * j + 3]};
        if (out_row < rows && out_half == 0) job.part_sums[(size_t)blockIdx.x * kRows + out_row - row0] = float2{reference, sum};
    } else if (out_row < rows) {
        if (sum == 0.f) {   // (nothing was seen, or all scores are -infinity, whatever the values)
#pragma unroll
            for (int i = 0; i < D / 32; i++)
#pragma unroll
                for (int j = 0; j < 16; j++) o[i][j] = 0.f;
        }
        const float v_scale = E4M3 && a.kv.v_scales ? a.kv.v_scales[kv_head] : 1.0f, to = sum == 0.f ? 0.f : v_scale / sum;
        const uint32_t token = job.by_group(out_row), head = kv_head * a.group + (out_row - token * a.group);
        _Float16 *out = a.out + (size_t)(start + (int)token) * a.out_stride + head * D + 4u * out_half;
#pragma unroll
        for (int i = 0; i < D / 32; i++)
#pragma unroll
            for (int j = 0; j < 4; j++)
                *(half4_any *)(out + 32 * i + 8 * j) = half4{(_Float16)(o[i][4 * j] * to), (_Float16)(o[i][4 * j + 1] * to), (_Float16)(o[i][4 * j + 2] * to),
                                                             (_Float16)(o[i][4 * j + 3] * to)};
    }
}

// Heads of 256 values, and short sequences: two waves share 32 queries.  Each takes half of a tile's tokens for the scores, with all of a head's values, and half of
// a head's values for the sums, with all of the tile's tokens; weights change hands in LDS, and with them whether a reference must move, which both do
// alike.  One buffer of keys and one of values: the next tile's keys come while values are summed, its values while keys are scored.  Half of a
// head's values a wave for the scores too, whose parts were added through LDS in tiles of 32, took 1.2 - 1.3 times as long (8192 rows, 16 heads on 8: f16
// 866 us, now 734; e4m3 909, now 694; 1500 rows behind 5000, window 1024, e4m3 82, now 69), and every lane's sixteen addresses, if held, spill
// (e4m3 99).  f16 values wait for the next keys, which go to LDS directly; through registers, as e4m3 does, they spill (854).
template <int D, bool E4M3> __global__ __launch_bounds__(256, (D == 256 ? 2 : 3)) void k_attn_prompt_pairs(const Prompt job)
{
    constexpr int KT = kPromptTile, kGroups = KT / 16;
    constexpr uint32_t kUnits = D / 8, kRow = D * 2, kTile = KT * kRow, kWaveRows = KT / kPromptWaves, kRows = 64, kHalf = D / 2;
    extern __shared__ __align__(16) char lds[];
    half8 *const weights = (half8 *)(lds + 2 * kTile);              // [wave][two runs of 16 tokens][lane]
    float *const tops = (float *)(lds + 2 * kTile + 4 * 2048);      // [wave][query]
    uint32_t *const flags = (uint32_t *)(lds + kPairsLds<D> - 16);     // [wave]: 1: a weight would pass 2^15, 2: a value is not finite
    const AttnArgs &a = job.a;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63u, half = lane >> 5, col = lane & 31u;

    const uint32_t pair = job.by_splits(blockIdx.x), split = blockIdx.x - pair * job.splits, local = job.by_kv_heads(pair), kv_head = pair - local * a.kv.kv_heads;
    Rows mine;
    if (!find_rows<64>(job, job.first_tile + local, &mine)) return;
    const uint32_t seq = mine.seq, row0 = mine.row0, rows = mine.rows;
    const int start = mine.start, before = mine.before;
    const int capacity = a.kv.pages ? (int)(a.seqs.table_stride << a.kv.page_shift) : 0;
    uint32_t key_tiles;
    const uint32_t parts = __builtin_amdgcn_readfirstlane(parts_of(mine, job, KT, &key_tiles));
    if (split >= parts) return;

    const uint32_t sharer = wave & 1u, wave_row = row0 + wave / 2u * 32u;
    const uint32_t row = wave_row + col, my_row = min(row, rows - 1);
    const uint32_t my_token = job.by_group(my_row), my_head = kv_head * a.group + (my_row - my_token * a.group);
    const int my_position = before + (int)my_token, my_begin = prompt_begin(a, my_position), my_end = min(my_position + 1, capacity);
    const int low = before + (int)job.by_group(row0), high = before + (int)job.by_group(min(row0 + kRows, rows) - 1);
    const uint32_t each_part = key_tiles / parts, one_more = key_tiles - each_part * parts;
    const int all_begin = mine.first & ~(KT - 1), first = max(mine.first, all_begin + (int)(split * each_part + min(split, one_more)) * KT);
    const int last = min(mine.last, all_begin + (int)((split + 1) * each_part + min(split + 1, one_more)) * KT);

    half8 q[D / 16];
    {
        const _Float16 *from = a.q + (size_t)(start + (int)my_token) * a.q_stride + my_head * D + 8u * half;
#pragma unroll
        for (int i = 0; i < D / 16; i++) q[i] = *(const half8_any *)(from + 16 * i);
    }
    const float c = exponent_factor(a.kv, a.scale, kv_head);
    float reference, sum;
    float16v o[kHalf / 32];

    const uint32_t page_mask = (1u << a.kv.page_shift) - 1u;
    const int t_begin = first & ~(KT - 1);
    PagesOf pages_of{a.seqs.tables + (size_t)seq * a.seqs.table_stride, a.kv.pages, a.kv.page_shift, last, t_begin, -1, 0};
    constexpr int kLoads = (int)(kWaveRows * D * (E4M3 ? 1 : 2) / 1024);   // 1 KB each
    constexpr uint32_t kLoadUnits = D * (E4M3 ? 1 : 2) / 16, kRowsPerLoad = 64 / kLoadUnits;
    uint4v held[kLoads];   // e4m3 only: keys or values on their way
    const uint32_t r0 = wave * kWaveRows;
    auto bring = [&](int t0, int of, bool value) {
        // rows of a page outside the pool are read from its first one
        const uint32_t page = (uint32_t)of < a.kv.pages ? (uint32_t)of : 0u;
        const size_t at = (kv_chunk(a.kv, page, kv_head) + ((uint32_t)(t0 + (int)r0) & page_mask) * D) * (E4M3 ? 1 : 2);
        const char *from = (const char *)(value ? a.kv.v : a.kv.k) + at;
        uint32_t me = lane;
        asm volatile("" : "+v"(me));
#pragma unroll
        for (int i = 0; i < kLoads; i++) {
            if constexpr (E4M3) {
                held[i] = *(const uint4v *)(from + i * 1024 + me * 16u);
            } else {
                const uint32_t r = r0 + i * kRowsPerLoad + me / kUnits;
                const uint32_t off = i * 1024u + me / kUnits * kRow + ((value ? value_place<D>(r, me % kUnits) : key_place<D>(r, me % kUnits)) << 4);
                char *to = lds + (value ? kTile : 0u) + (r0 + i * kRowsPerLoad) * kRow;
                __builtin_amdgcn_global_load_lds((const TWM_GLOBAL void *)(from + off), (TWM_LDS(void) *)to, 16, 0, 0);
            }
        }
    };
    auto keep = [&](bool value) {
        if constexpr (E4M3) {
            uint32_t me = lane;
            asm volatile("" : "+v"(me));
#pragma unroll
            for (int i = 0; i < kLoads; i++) {
                const uint32_t r = r0 + i * kRowsPerLoad + me / kLoadUnits, unit = me % kLoadUnits * 2;
                char *to = lds + (value ? kTile : 0u) + r * kRow;
                *(half8 *)(to + ((value ? value_place<D>(r, unit) : key_place<D>(r, unit)) << 4)) = to_f16(held[i][0], held[i][1]);
                *(half8 *)(to + ((value ? value_place<D>(r, unit + 1) : key_place<D>(r, unit + 1)) << 4)) = to_f16(held[i][2], held[i][3]);
            }
        }
    };
    auto arrived = [&]() {
        if constexpr (!E4M3) __builtin_amdgcn_s_waitcnt(0x0F70);   // vmcnt(0)
        __syncthreads();
    };

    const int high_begin = prompt_begin(a, high);
    int whole_end = min(low + 1, last);
    const uint32_t k_at = (32u * sharer + col) * kRow + (key_place<D>(col, half) << 4), v_row = 4u * half + (lane >> 2 & 3u);
    const uint32_t v_at = (kTile + v_row * kRow + (value_place<D>(v_row, (lane >> 4 & 1u) * 2u + (lane >> 1 & 1u)) << 4) + (lane & 1u) * 8u) ^ sharer * kHalf * 2u;
    const half8 *const pair_weights = weights + (wave & ~1u) * 128u + lane;
    float16v s;
    float added;
    auto weigh = [&]() {
        const float from = reference == -INFINITY ? 0.f : reference;
        half8 p[2];
        added = 0.f;
#pragma unroll
        for (int j = 0; j < 16; j += 2) {
            const half2v w = {(_Float16)__builtin_amdgcn_exp2f(fmaf(s[j] - from, c, 8.0f)), (_Float16)__builtin_amdgcn_exp2f(fmaf(s[j + 1] - from, c, 8.0f))};
            added = __builtin_amdgcn_fdot2(w, half2v{(_Float16)1.0f, (_Float16)1.0f}, added, false);
            p[j / 8][j % 8] = w[0];
            p[j / 8][j % 8 + 1] = w[1];
        }
        weights[wave * 128u + lane] = p[0];
        weights[wave * 128u + 64u + lane] = p[1];
    };

    for (;;) {
        reference = -INFINITY;
        sum = 0.f;
#pragma unroll
        for (int i = 0; i < (int)kHalf / 32; i++)
#pragma unroll
            for (int j = 0; j < 16; j++) o[i][j] = 0.f;
        int t0 = t_begin;
        uint32_t there = 0;
        Pages next{-1, 0};
        if (t0 < last) {
            pages_of.look_up(t0);
            const Pages now = pages_of.find(t0, wave);
            there = now.there;
            bring(t0, now.mine, false);
            keep(false);
            bring(t0, now.mine, true);
            next = pages_of.find(t0 + KT, wave);
            arrived();
        }
        while (t0 < last) {
            const bool more = t0 + KT < last;
            if constexpr (E4M3) {
                // values of this tile to LDS; the next one begins its way
                keep(true);
                if (more) bring(t0 + KT, next.mine, false);
            }
            uint32_t keys_at = k_at;
            asm volatile("" : "+v"(keys_at));   // (sixteen addresses that are made anew, not held)
#pragma unroll
            for (int j = 0; j < 16; j++) s[j] = 0.f;
#pragma unroll
            for (int i = 0; i < D / 16; i++) s = __builtin_amdgcn_mfma_f32_32x32x16_f16(*(const half8 *)(lds + (keys_at ^ i << 5)), q[i], s, 0, 0, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
#pragma unroll
            for (int i = 0; i < D / 16 - 4; i++) {
                __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
            }
            __builtin_amdgcn_sched_group_barrier(0x8, 4, 0);
            const bool whole = t0 >= high_begin && t0 + KT <= whole_end && there == (1u << kGroups) - 1u;
            bool bad = false;
            if (!whole) {
#pragma unroll
                for (int j = 0; j < 16; j++) {
                    const uint32_t seen = there >> (2 * sharer + j / 8) & 1u ? (uint32_t)max(0, my_end - my_begin) : 0u;
                    s[j] = (uint32_t)(t0 + 32 * (int)sharer + 8 * (j / 4) + 4 * (int)half + j % 4 - my_begin) < seen ? s[j] : -INFINITY;
                }
                // values that this wave has brought: rows that nobody sees become zeros, the others are looked through
                if constexpr (!E4M3) __builtin_amdgcn_s_waitcnt(0x0F70);
                uint32_t me = lane;
                asm volatile("" : "+v"(me));
                const uint32_t looked = r0 + me / 4, unit = me % 4 * (kUnits / 4);
                const int token = t0 + (int)looked;
                const bool dead = token < first || token >= last || !(there >> (looked / 16) & 1u);
                bad = __any(look_through<D, kUnits / 4>(lds + kTile, looked, unit, dead));
            }
            float most = s[0];
#pragma unroll
            for (int j = 0; j < 16; j++) most = fmaxf(most, s[j]);
            most = max_of_halves(most);
            weigh();
            if (half == 0) tops[wave * 32u + col] = most;
            const bool over = __any((most - reference) * c > 7.0f);
            if (lane == 0) flags[wave] = (over ? 1u : 0u) | (bad ? 2u : 0u);
            arrived();
            const uint32_t flag = flags[0] | flags[1] | flags[2] | flags[3];
            if (flag & 1u) {
                // the reference moves, for both waves of a pair alike, and what is summed with it
                most = fmaxf(most, tops[(wave ^ 1u) * 32u + col]);
                const float raised = (most - reference) * c > 7.0f ? most : reference;
                const float by = shrink(reference, raised, c);
                sum *= by;
#pragma unroll
                for (int i = 0; i < (int)kHalf / 32; i++) o[i] *= by;
                reference = raised;
                weigh();
                __syncthreads();
            }
            sum += added;
            // every wave is done with the tile's keys
            if (more) {
                if constexpr (E4M3) keep(false);
                bring(t0 + KT, next.mine, E4M3);
            }
            if (!(flag & 2u)) {
#pragma unroll
                for (int b = 0; b < KT / 16; b++) {
                    const half8 p = pair_weights[b * 64];
#pragma unroll
                    for (int i = 0; i < (int)kHalf / 32; i++) {
                        const half4 x = __builtin_bit_cast(half4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((TWM_LDS(short4v) *)(lds + (v_at ^ i << 6) + b * 16 * kRow)));
                        const half4 y = __builtin_bit_cast(half4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((TWM_LDS(short4v) *)(lds + (v_at ^ i << 6) + (b * 16 + 8) * kRow)));
                        o[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(half8{x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]}, p, o[i], 0, 0, 0);
                    }
                }
            } else {
                // one token after the other
                for (int r = 0; r < KT; r++) {
                    const int at = t0 + r;
                    if (at < first || at >= last || !(there >> (r / 16) & 1u)) continue;
                    const bool seen = at >= my_begin && at < my_end;
                    const _Float16 *of = (const _Float16 *)(weights + ((wave & ~1u) + r / 32u) * 128u + r % 32 / 16 * 64 + r / 4 % 2 * 32 + col);
                    add_one<D>(o, lds + kTile, (uint32_t)r, sharer * kHalf / 8u, of[r / 8 % 2 * 4 + r % 4], seen);
                }
            }
            arrived();
            if constexpr (!E4M3) {
                if (more) bring(t0 + KT, next.mine, true);
            }
            t0 += KT;
            there = next.there;
            next = pages_of.find(t0 + KT, wave);
        }
        if (E4M3 || max(t_begin, high_begin) + KT > whole_end) break;
        // (as above: an infinite value times a weight that f16 holds as 0)
        const bool odd = __any(any_nan(o));
        if (lane == 0) flags[wave] = odd;
        __syncthreads();
        if ((flags[0] | flags[1] | flags[2] | flags[3]) == 0) break;
        whole_end = t_begin;
    }

    sum = sum_of_halves(sum);
    if (half == 0) tops[wave * 32u + col] = sum;
    __syncthreads();
    sum += tops[(wave ^ 1u) * 32u + col];
    uint32_t me = lane;   // (as above)
    asm volatile("" : "+v"(me));
    const uint32_t out_row = wave_row + (me & 31u), out_half = me >> 5;
    if (parts > 1) {
        // to scratch, rows beside each other
        float4v *to = job.parts + (size_t)blockIdx.x * (D / 4 * kRows) + out_row - row0;
#pragma unroll
        for (int i = 0; i < (int)kHalf / 32; i++)
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (out_row < rows)
                    to[(sharer * (kHalf / 4) + 8u * i + 2u * j + out_half) * kRows] = float4v{o[i][4 * j], o[i][4 * j + 1], o[i][4 * j + 2], o[i][4 * j + 3]};
        if (out_row < rows && sharer == 0 && out_half == 0) job.part_sums[(size_t)blockIdx.x * kRows + out_row - row0] = float2{reference, sum};
    } else if (out_row < rows) {
        if (sum == 0.f) {   // (nothing was seen, or all scores are -infinity, whatever the values)
#pragma unroll
            for (int i = 0; i < (int)kHalf / 32; i++)
#pragma unroll
                for (int j = 0; j < 16; j++) o[i][j] = 0.f;
        }
        const float v_scale = E4M3 && a.kv.v_scales ? a.kv.v_scales[kv_head] : 1.0f, to = sum == 0.f ? 0.f : v_scale / sum;
        const uint32_t token = job.by_group(out_row), head = kv_head * a.group + (out_row - token * a.group);
        _Float16 *out = a.out + (size_t)(start + (int)token) * a.out_stride + head * D + sharer * kHalf + 4u * out_half;
#pragma unroll
        for (int i = 0; i < (int)kHalf / 32; i++)
#pragma unroll
            for (int j = 0; j < 4; j++)
                *(half4_any *)(out + 32 * i + 8 * j) = half4{(_Float16)(o[i][4 * j] * to), (_Float16)(o[i][4 * j + 1] * to), (_Float16)(o[i][4 * j + 2] * to),
                                                             (_Float16)(o[i][4 * j + 3] * to)};
    }
}

// Joins what several workgroups hold of rows: 256 / (D / 4) rows of a tile and key-value head a workgroup, or a fourth of that where parts
// are many and each wave takes every fourth.
template <int D, int SLICES> __global__ __launch_bounds__(256) void k_attn_prompt_join(const Prompt job)
{
    constexpr uint32_t kRows = kPromptRows<D>, kEach = 256 / SLICES, kHere = kEach / (D / 4);   // threads of a slice, rows of a workgroup
    __shared__ float4v sums_of[SLICES][kEach];
    __shared__ float2 tops_of[SLICES][kEach];
    const AttnArgs &a = job.a;
    const uint32_t local = job.by_kv_heads(blockIdx.x), kv_head = blockIdx.x - local * a.kv.kv_heads;
    Rows mine;
    if (!find_rows<kRows>(job, job.first_tile + local, &mine)) return;
    uint32_t key_tiles;
    const uint32_t parts = parts_of(mine, job, kPromptTile, &key_tiles);
    const uint32_t first_row = blockIdx.y * kHere;
    if (parts == 1 || mine.row0 + first_row >= mine.rows) return;
    const uint32_t slice = threadIdx.x / kEach, x = threadIdx.x % kEach, r = first_row + x % kHere, quad = x / kHere;   // (rows lie beside each other)
    const float2 *sums = job.part_sums + (size_t)blockIdx.x * job.splits * kRows + r;
    const float4v *from = job.parts + (size_t)blockIdx.x * job.splits * (D / 4 * kRows) + quad * kRows + r;
    const float c = exponent_factor(a.kv, a.scale, kv_head);
    float top = -INFINITY, sum = 0.f;
    float4v o = {0.f, 0.f, 0.f, 0.f};
    auto add = [&](const float2 &s, const float4v &part) {
        const float raised = fmaxf(top, s.x), keep = shrink(top, raised, c), by = shrink(s.x, raised, c);
        sum = sum * keep + s.y * by;
        o = o * keep + part * by;
        top = raised;
    };
    if (mine.row0 + r < mine.rows) {
        constexpr uint32_t kAhead = 4;
        for (uint32_t p = slice; p < parts; p += SLICES * kAhead) {
            float2 s[kAhead];
            float4v part[kAhead];
#pragma unroll
            for (uint32_t i = 0; i < kAhead; i++) {
                const uint32_t q = min(p + SLICES * i, parts - 1);
                s[i] = sums[q * kRows];
                part[i] = from[(size_t)q * (D / 4 * kRows)];
            }
#pragma unroll
            for (uint32_t i = 0; i < kAhead; i++)
                if (p + SLICES * i < parts) add(s[i], part[i]);
        }
    }
    if constexpr (SLICES > 1) {
        sums_of[slice][x] = o;
        tops_of[slice][x] = float2{top, sum};
        __syncthreads();
        if (slice != 0) return;
#pragma unroll
        for (uint32_t i = 1; i < SLICES; i++) add(tops_of[i][x], sums_of[i][x]);
    }
    const uint32_t row = mine.row0 + r;
    if (row >= mine.rows) return;
    if (sum == 0.f) o = float4v{0.f, 0.f, 0.f, 0.f};
    const float v_scale = a.kv.v_scales ? a.kv.v_scales[kv_head] : 1.0f, to = sum == 0.f ? 0.f : v_scale / sum;
    const uint32_t token = job.by_group(row), head = kv_head * a.group + (row - token * a.group);
    *(half4_any *)(a.out + (size_t)(mine.start + (int)token) * a.out_stride + head * D + 4u * quad) =
        half4{(_Float16)(o[0] * to), (_Float16)(o[1] * to), (_Float16)(o[2] * to), (_Float16)(o[3] * to)};
}

hipError_t init_attn_prompt()
{
    hipError_t e = hipSuccess;
    auto ask = [&](auto kernel, uint32_t bytes) {
        if (e == hipSuccess) e = hipFuncSetAttribute((const void *)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    };
    ask(k_attn_prompt<64, false>, kPromptLds<64>);
    ask(k_attn_prompt<64, true>, kPromptLds<64>);
    ask(k_attn_prompt<128, false>, kPromptLds<128>);
    ask(k_attn_prompt<128, true>, kPromptLds<128>);
    ask(k_attn_prompt_pairs<256, false>, kPairsLds<256>);
    ask(k_attn_prompt_pairs<256, true>, kPairsLds<256>);
    ask(k_attn_prompt_pairs<128, false>, kPairsLds<128>);
    ask(k_attn_prompt_pairs<128, true>, kPairsLds<128>);
    ask(k_attn_prompt_pairs<64, false>, kPairsLds<64>);
    ask(k_attn_prompt_pairs<64, true>, kPairsLds<64>);
    return e;
}

hipError_t launch_attn_prompt(hipStream_t s, const AttnArgs &a, void *scratch, size_t scratch_bytes)
{
    auto launch = [&](auto dim) {
        constexpr int D = decltype(dim)::value;
        const uint64_t capacity = (uint64_t)a.seqs.table_stride << a.kv.page_shift;
        // Waves in pairs for heads of 256 values, and where no sequence can be longer than eight tiles by the table's width and the chip is not full of
        // them: tiles of 64 rows and half of a tile's tokens a wave take less time each, if more together.  28 heads on 4 of 128: 128 rows 8.2 us, 9.8 in
        // the other form, 512 19.1 and 21.3, 1000 in twenty prompts 11.8 and 12.4; 200 rows of 32 heads on 32 in e4m3 10.1 and 14.7; 37 rows of 14 heads
        // of 64 5.3 and 8.1; but 1000 rows in five prompts 17.8 and 16.1, 4000 in twenty 40 and 34, 8192 in one 670 and 500.
        const uint64_t pairs_tiles = (uint64_t)a.rows * a.group / 64 + a.seqs.seqs;
        const bool pairs = D == 256 || (capacity <= 512 && pairs_tiles * a.kv.kv_heads * capacity <= 2048 * kPromptTile);
        const uint32_t each = pairs ? 64 : 128;
        // every sequence begins a tile of its own
        const uint64_t tiles = (uint64_t)a.rows * a.group / each + a.seqs.seqs, workgroups = tiles * a.kv.kv_heads;
        // Tokens are shared out where rows alone leave most of the chip without work (two workgroups a compute unit), as far as there may be some
        const uint64_t seen = std::min(capacity, a.window ? (uint64_t)a.window + each : capacity);
        Prompt job;
        job.a = a;
        job.tiles = (uint32_t)tiles;
        job.by_group = Divisor(a.group);
        job.by_kv_heads = Divisor(a.kv.kv_heads);
        job.balance = (D == 64 ? 80.0f : D == 128 ? 40.0f : 48.0f) / (float)workgroups;
        const float balanced = std::sqrt((float)(seen / kPromptTile + 1) * job.balance);   // of the most tiles that there may be
        job.splits = each != kPromptRows<D> ? 1u
                                            : (uint32_t)std::max<uint64_t>(1, std::min<uint64_t>(std::min<uint64_t>(512 / workgroups, seen / (kPromptTile * kLeastPart)),
                                                                                                 (uint64_t)balanced));
        job.by_splits = Divisor(job.splits);
        job.parts = (float4v *)scratch;
        job.part_sums = (float2 *)((char *)scratch + (size_t)workgroups * job.splits * each * D * 4);
        if (job.splits > 1 && (size_t)workgroups * job.splits * each * (D * 4 + 8) > scratch_bytes) return hipErrorOutOfMemory;   // (at most 34 MB of 256)
        const hipError_t error = in_slices((uint32_t)tiles, most_workgroups(256) / (a.kv.kv_heads * job.splits), [&](uint32_t tile, uint32_t here) {
            job.first_tile = tile;
            const dim3 grid(here * a.kv.kv_heads * job.splits);
            if (pairs)
                hipLaunchKernelGGL((a.kv.e4m3 ? k_attn_prompt_pairs<D, true> : k_attn_prompt_pairs<D, false>), grid, dim3(256), kPairsLds<D>, s, job);
            else if constexpr (D != 256)
                hipLaunchKernelGGL((a.kv.e4m3 ? k_attn_prompt<D, true> : k_attn_prompt<D, false>), grid, dim3(256), kPromptLds<D>, s, job);
            return hipGetLastError();
        });
        if (error != hipSuccess || job.splits == 1) return error;
        // (one slice: at most 512 workgroups)
        if (job.splits >= 8)
            hipLaunchKernelGGL((k_attn_prompt_join<D, 4>), dim3((uint32_t)workgroups, each / (64 / (D / 4))), dim3(256), 0, s, job);
        else
            hipLaunchKernelGGL((k_attn_prompt_join<D, 1>), dim3((uint32_t)workgroups, each / (256 / (D / 4))), dim3(256), 0, s, job);
        return hipGetLastError();
    };
    return a.kv.dim == 64    ? launch(std::integral_constant<int, 64>{})
           : a.kv.dim == 128 ? launch(std::integral_constant<int, 128>{})
                             : launch(std::integral_constant<int, 256>{});
}

}  // namespace twm
