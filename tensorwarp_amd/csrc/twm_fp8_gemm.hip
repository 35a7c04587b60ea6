// C[M,N] = A[M,K] x W[N,K]^T in 8-bit floating point (e4m3) with f32 scales, one per row and 128 features of A and one per
// 128 x 128 block of W:
//
//   C[m][n] = sum over blocks b of a_scales[m][b] * w_scales[n / 128][b] * (sum over the block's k of A[m][k] * W[n][k])
//
// Two ways to a block's sum.  The matrix unit's 8-bit instructions cut every product of eight neighbouring features off below 2^-13 of
// the largest one's power of two before they add (measured: 2^14 + 2^0 is 2^14 within a group of eight and exact across two; against the
// exact sum results were off by 1.2e-5 of their norm on bell-shaped values and 5e-5 on evenly drawn codes).  That is below the rounding
// of an f16 result (2^-11), so f16 results of more than 16 rows use them in tiles.  f32 results, which are to hold 32-bit sums, do not, and
// those of up to 16 rows, which wait for the weights, have no need to: the codes become f16 there, which holds each exactly, as do the
// f32 products of the f16 instructions.  A block's sum is scaled by one f32 factor per lane (the rows of A are the lanes' columns of the
// result, those of W lie in its registers) and added to the f32 sum.  Both arrays are read as the caller holds them, row by
// row: a lane's operand is 32 consecutive bytes of a row, and which of the 128 features a lane holds does not matter as long as
// both operands agree.
//
// Measured, and what bounds it: one row of 3584 -> 37888 24.8 us, 5.5 TB/s: the weights' way from memory; 13 rows of 11008 -> 4096 11.7,
// 3.9 TB/s: the ramp and the tail of a launch of 256 workgroups and the two ranges' sums; 333 rows of 18944 -> 3584 40: tiles 33 (the operands' way to LDS) and the six
// ranges' sums 6; 2048 rows of 4096 -> 22016 179, 2.06 PFLOP/s in f16: products with the factors' multiplications take 104 to 116 by
// themselves, the operands' way to LDS 149 (9.4 TB/s over the chip), and the two do not overlap wholly.  A ring of five buffers with two
// blocks' loads in flight took 187 to 190 where this took 172, tiles of 256 x 192 were behind but for a few row counts.
#include "twm_device.h"

#include <cstdio>
#include <type_traits>

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

// Rows of results begin where the ones before them end, on any element's boundary; the memory takes vectors there too
typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef half4 half4_any __attribute__((aligned(2)));
typedef float4v float4v_any __attribute__((aligned(4)));
typedef uint4v uint4v_any __attribute__((aligned(2)));

// columns n .. n + 3 of row m
__device__ __forceinline__ void store_quad(const Fp8Gemm &g, uint32_t m, uint32_t n, const float4v &v)
{
    if (m >= g.m || n >= g.n) return;
    const size_t at = (size_t)m * g.n + n;
    const bool whole = n + 4u <= g.n;
    if (g.c_f16) {
        _Float16 *c = (_Float16 *)g.c + at;
        if (whole) {
            *(half4_any *)c = half4{(_Float16)v[0], (_Float16)v[1], (_Float16)v[2], (_Float16)v[3]};
        } else {
#pragma unroll
            for (uint32_t j = 0; j < 3; j++)
                if (n + j < g.n) c[j] = (_Float16)v[j];
        }
    } else {
        float *c = (float *)g.c + at;
        if (whole) {
            *(float4v_any *)c = v;
        } else {
#pragma unroll
            for (uint32_t j = 0; j < 3; j++)
                if (n + j < g.n) c[j] = v[j];
        }
    }
}

}  // namespace

// ---- few rows: every wave its own blocks ---------------------------------------------------------------------------------
//
// 16 * NT columns x 16 * MT rows per workgroup; wave w takes the blocks w, w + WAVES, ... of the workgroup's range of K, U of them
// in flight, and the waves' sums are added in LDS in wave order.  Operands go from memory to registers.  TAIL: K ends inside a
// block.  Bound: the weights' way through memory.
template <int MT, int NT, int U, int WAVES, bool TAIL>
__global__ __launch_bounds__(WAVES * 64) void k_fp8_rows_few(const Fp8Gemm g, uint32_t kb_per_split, float *__restrict__ partials, uint32_t n_ld)
{
    __shared__ float4v sums[WAVES][NT * MT][64];
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63u;
    const uint32_t n0 = blockIdx.x * (16u * NT), m0 = blockIdx.y * (16u * MT), part = (lane >> 4) * 32u;
    const uint32_t b0 = blockIdx.z * kb_per_split, b1 = min(b0 + kb_per_split, g.kb);
    // rows behind the end replay the last one and are not stored
    const uint8_t *w_row[NT], *a_row[MT];
    const float *as_row[MT];
    const TWM_CONSTANT float *ws_row[NT];
#pragma unroll
    for (int t = 0; t < NT; t++) {
        w_row[t] = g.w + (size_t)min(n0 + 16u * t + (lane & 15u), g.n - 1u) * g.k;
        ws_row[t] = (const TWM_CONSTANT float *)(g.w_scales + (size_t)(min(n0 + 16u * t, g.n - 1u) >> 7) * g.kb);
    }
#pragma unroll
    for (int t = 0; t < MT; t++) {
        const uint32_t m_row = min(m0 + 16u * t + (lane & 15u), g.m - 1u);
        a_row[t] = g.a + (size_t)m_row * g.k;
        as_row[t] = g.a_scales + (size_t)m_row * g.kb;
    }
    float4v acc[NT][MT] = {};
    for (uint32_t b = b0 + wave; b < b1; b += WAVES * U) {
        int8v w[U][NT], a[U][MT];
        float as[U][MT], ws[U][NT];
#pragma unroll
        for (uint32_t u = 0; u < U; u++) {
            const uint32_t at = min(b + u * WAVES, b1 - 1u), k0 = at * 128u + part;   // (past the end the last block, which is not added)
#pragma unroll
            for (int t = 0; t < NT; t++) {
                w[u][t] = load_32<TAIL>(w_row[t], k0, g.k);
                ws[u][t] = ws_row[t][at];
            }
#pragma unroll
            for (int t = 0; t < MT; t++) {
                a[u][t] = load_32<TAIL>(a_row[t], k0, g.k);
                as[u][t] = as_row[t][at];
            }
        }
#pragma unroll
        for (uint32_t u = 0; u < U; u++) {
            if (u && b + u * WAVES >= b1) break;
#pragma unroll
            for (int t = 0; t < NT; t++)
#pragma unroll
                for (int j = 0; j < MT; j++) acc[t][j] += block_sum(w[u][t], a[u][j]) * (as[u][j] * ws[u][t]);
        }
    }
#pragma unroll
    for (int t = 0; t < NT; t++)
#pragma unroll
        for (int j = 0; j < MT; j++) sums[wave][t * MT + j][lane] = acc[t][j];
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < NT * MT * 64u; i += WAVES * 64u) {
        const uint32_t t = i >> 6, l = i & 63u, m = m0 + 16u * (t % MT) + (l & 15u), n = n0 + 16u * (t / MT) + (l >> 4) * 4u;
        float4v s = sums[0][t][l];
#pragma unroll
        for (int w = 1; w < WAVES; w++) s += sums[w][t][l];
        if (partials) {
            if (m < g.m && n < n_ld) *(float4v *)(partials + ((size_t)blockIdx.z * g.m + m) * n_ld + n) = s;
        } else {
            store_quad(g, m, n, s);
        }
    }
}

// ---- many rows: tiles staged in LDS --------------------------------------------------------------------------------------
//
// A workgroup computes BM rows x BN columns in blocks of 128 features.  Both operands' blocks (128 bytes a row) go from memory
// to LDS directly, two buffers; eight rows per load instruction, lane l = (row l / 8, 16-byte slot l % 8).  Slot s of row r
// holds the row's piece s ^ (r / 2 % 8): two rows span the 64 banks, so that sixteen neighbouring rows' reads of one piece fall
// on all of them (the 16-byte reads of a wave take eight cycles each so; with s ^ (r % 8) they took as many).  Waves own S * TN
// columns x S * TM rows each (columns within one 128-column block of W's scales).  The rows' scales come to LDS four blocks at a time,
// 16 bytes a row: read from memory by the lanes that need them, each was a cache line of its own, half as many again as the operands'
// (2048 x 22016 x 4096 254 us, with none of them read 197).
//
// S = 16: v_mfma_f32_16x16x128_f8f6f4 takes a tile's whole block at once.  Results in f16 only: within each eight neighbouring
// features the unit cuts products off at 2^-13 of the largest one's power of two.
// S = 32: the codes become f16 between LDS and eight v_mfma_f32_32x32x16_f16; every product and sum in f32.

typedef float float16v __attribute__((ext_vector_type(16)));

namespace {

typedef __attribute__((address_space(3))) void *LdsPtr;
// `bytes` from p on: reads behind them give zeros
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer_of(const void *p, uint32_t bytes)
{
    return __builtin_amdgcn_make_buffer_rsrc((void *)p, 0, (int)bytes, 0x00020000);
}

// (a wave's results, 64 columns in f32 or twice as many in f16, take the operands' place at the end)
template <int BM, int BN> struct Fp8Tile {
    uint8_t w[2][BN * 128];
    uint8_t a[2][BM * 128];
    float scales[2][BM * 4];   // of four blocks of A
};

// a lane's part of one operand tile of S rows x 128 features, and of the tile's result
template <int S> struct Fp8Mfma;
template <> struct Fp8Mfma<16> {
    typedef float4v Sum;
    int8v part;
    // bytes 32 (lane / 16) .. + 31 of row lane % 16; base: the tile in LDS
    __device__ __forceinline__ void read(const uint8_t *base, const uint32_t (&at)[4])
    {
        const uint4v lo = *(const uint4v *)(base + at[0]), hi = *(const uint4v *)(base + at[1]);
        part = int8v{(int)lo[0], (int)lo[1], (int)lo[2], (int)lo[3], (int)hi[0], (int)hi[1], (int)hi[2], (int)hi[3]};
    }
    static __device__ __forceinline__ void places(uint32_t lane, uint32_t (&at)[4])
    {
        for (uint32_t p = 0; p < 2; p++) at[p] = (lane & 15u) * 128u + (((2u * (lane >> 4) + p) ^ (lane >> 1 & 7u)) * 16u);
        at[2] = at[3] = 0;
    }
    static __device__ __forceinline__ Sum product(const Fp8Mfma &w, const Fp8Mfma &a)
    {
        return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w.part, a.part, Sum{}, 0, 0, 0, 0, 0, 0);
    }
};
template <> struct Fp8Mfma<32> {
    typedef float16v Sum;
    uint4v part[4];
    // bytes 64 h + 32 (lane / 32) .. + 31 of row lane % 32, h = 0, 1
    __device__ __forceinline__ void read(const uint8_t *base, const uint32_t (&at)[4])
    {
#pragma unroll
        for (int p = 0; p < 4; p++) part[p] = *(const uint4v *)(base + at[p]);
    }
    static __device__ __forceinline__ void places(uint32_t lane, uint32_t (&at)[4])
    {
        for (uint32_t p = 0; p < 4; p++) at[p] = (lane & 31u) * 128u + (((4u * (p >> 1) + 2u * (lane >> 5) + (p & 1u)) ^ (lane >> 1 & 7u)) * 16u);
    }
    static __device__ __forceinline__ Sum product(const Fp8Mfma &w, const Fp8Mfma &a)
    {
        Sum d = {};
#pragma unroll
        for (int p = 0; p < 4; p++)
#pragma unroll
            for (int e = 0; e < 4; e += 2)
                d = __builtin_amdgcn_mfma_f32_32x32x16_f16(to_f16((int)w.part[p][e], (int)w.part[p][e + 1]), to_f16((int)a.part[p][e], (int)a.part[p][e + 1]), d, 0, 0, 0);
        return d;
    }
};

// Which tile: workgroups go to the eight XCDs in turn; XCD x takes the x-th eighth of a list of the tiles that runs in bands of
// eight row blocks, so that what an XCD works on at a time shares its operands in that XCD's L2.
__device__ __forceinline__ void tile_of(uint32_t blocks_n, uint32_t blocks_m, uint32_t &bn, uint32_t &bm)
{
    constexpr uint32_t kBand = 8;
    const uint32_t tiles = blocks_n * blocks_m, share = tiles >> 3, rest = tiles & 7u, x8 = blockIdx.x & 7u;
    const uint32_t t = x8 * share + (x8 < rest ? x8 : rest) + (blockIdx.x >> 3);
    const uint32_t band = t / (kBand * blocks_n), u = t - band * kBand * blocks_n;
    const uint32_t high = blocks_m - band * kBand < kBand ? blocks_m - band * kBand : kBand;
    bn = u / high;
    bm = band * kBand + u % high;
}

// The results of a wave, TM x TN tiles from row m0 and column n0 on.  Every wave of the workgroup comes here, its reads of LDS done.
template <int S, int TN, int TM>
__device__ __forceinline__ void store_tile(const Fp8Gemm &g, const typename Fp8Mfma<S>::Sum (&acc)[TN][TM], uint8_t *lds, uint32_t wave, uint32_t lane,
                                           uint32_t m0, uint32_t n0, float *partials, uint32_t n_ld)
{
    const uint32_t row = lane % S;
    // Registers 4 e .. 4 e + 3 of a lane: columns (256 / S) e + 4 (lane / S) .. + 3 of the tile, row lane % S.  They leave by way of LDS,
    // so that a row leaves in whole lines: up to 128 columns at a time in f16, 64 in f32, 256 bytes a row; piece p of row r stands at
    // p ^ (r % PIECES).  (Stored from the registers, 32 or 64 bytes a row: 2048 x 22016 x 4096 198 us, by way of LDS 184; 2048 x 8192 x
    // 1024 33.8 and 24.1; where rows begin on any element's boundary, 711 x 34978 x 384, 53.1 element by element and 22.8 so.)
    __builtin_amdgcn_s_waitcnt(0);
    __builtin_amdgcn_s_barrier();
    const bool f16 = g.c_f16 && !partials;
    const uint32_t ld = partials ? n_ld : g.n;
    auto rows = [&](auto which) {
        constexpr bool F16 = decltype(which)::value;
        constexpr uint32_t COLS = F16 ? S * TN : 64, ROW = COLS * (F16 ? 2 : 4), PIECES = ROW / 16, TILES = COLS / S;
        uint8_t *mine = lds + wave * (S * TM * ROW);
#pragma unroll
        for (uint32_t i0 = 0; i0 < TN; i0 += TILES) {
#pragma unroll
            for (uint32_t i = 0; i < TILES; i++)
#pragma unroll
                for (int j = 0; j < TM; j++)
#pragma unroll
                    for (uint32_t e = 0; e < S * S / 256; e++) {
                        const uint32_t r = j * S + row, quad = i * (S / 4) + e * (64 / S) + lane / S;   // columns 4 quad .. + 3
                        const auto &v = acc[i0 + i][j];
                        if constexpr (F16) {
                            *(half4 *)(mine + r * ROW + ((quad >> 1) ^ (r % PIECES)) * 16u + (quad & 1u) * 8u) =
                                half4{(_Float16)v[4 * e], (_Float16)v[4 * e + 1], (_Float16)v[4 * e + 2], (_Float16)v[4 * e + 3]};
                        } else {
                            *(float4v *)(mine + r * ROW + (quad ^ (r % PIECES)) * 16u) = float4v{v[4 * e], v[4 * e + 1], v[4 * e + 2], v[4 * e + 3]};
                        }
                    }
            // (a wave reads what it has written itself)
#pragma unroll
            for (uint32_t at = 0; at < S * TM * PIECES; at += 64u) {
                const uint32_t r = (at + lane) / PIECES, p = (at + lane) % PIECES, m = m0 + r;
                const uint32_t n = n0 + i0 * S + p * (F16 ? 8u : 4u);
                typedef std::conditional_t<F16, _Float16, float> Result;
                constexpr uint32_t EACH = 16u / sizeof(Result);
                const Result *from = (const Result *)(mine + r * ROW + (p ^ (r % PIECES)) * 16u);
                const uint4v v = *(const uint4v *)from;
                if (m >= g.m || n >= ld) continue;
                Result *to = (!F16 && partials ? (Result *)partials + (size_t)blockIdx.y * g.m * ld : (Result *)g.c) + (size_t)m * ld + n;
                if (n + EACH <= ld) {
                    *(uint4v_any *)to = v;
                } else {
#pragma unroll
                    for (uint32_t e = 0; e < EACH - 1u; e++)
                        if (n + e < ld) to[e] = from[e];
                }
            }
        }
    };
    if (S == 16 && f16) rows(std::integral_constant<bool, true>{});
    else rows(std::integral_constant<bool, false>{});
}

}  // namespace

template <int S, int TN, int TM, int WN, int WM>
__global__ __launch_bounds__(WN * WM * 64) void k_fp8_tile(const Fp8Gemm g, uint32_t blocks_n, uint32_t blocks_m, uint32_t kb_per_split,
                                                           float *__restrict__ partials, uint32_t n_ld)
{
    typedef Fp8Mfma<S> Mfma;
    constexpr int BN = S * TN * WN, BM = S * TM * WM, WAVES = WN * WM;
    constexpr int LW = BN / 8 / WAVES, LA = BM / 8 / WAVES;   // load instructions of eight rows per wave
    constexpr int DEPTH = S == 16 ? 3 : 2;                    // results of the matrix unit in flight
    // A block's loads, from the last row of products of the block two before on.  Eight waves issue theirs one by one, with every
    // second product (issued together they held every wave of the CU up until the last had been taken: 2048 x 22016 x 4096 204 us,
    // one by one 196); of four waves' workgroups two share a CU and take turns.
    constexpr int PARTS = LW + LA, EVERY = WAVES == 8 && TN * TM >= 32 ? 2 : 1, PER = WAVES == 8 && S == 16 ? 1 : WAVES == 8 ? (PARTS + TM - 1) / TM : PARTS;
    constexpr int EARLY = TM / EVERY * PER < PARTS ? TM / EVERY * PER : PARTS;   // those of the last row
    static_assert(LW % 2 == 0 && LA % 2 == 0 && (PARTS - EARLY + PER - 1) / PER * EVERY <= (TN - 1) * TM);
    static_assert(BN % (8 * WAVES) == 0 && BM % (8 * WAVES) == 0 && 128 % (S * TN) == 0 && TN % 2 == 0);
    static_assert(S * TN % 64 == 0 && WAVES * S * TM * 256u <= sizeof(Fp8Tile<BM, BN>));
    extern __shared__ uint8_t lds[];
    Fp8Tile<BM, BN> &tile = *(Fp8Tile<BM, BN> *)lds;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63u;
    const uint32_t wn = wave % WN, wm = wave / WN;

    uint32_t n0, m0;
    tile_of(blocks_n, blocks_m, n0, m0);
    n0 *= BN;
    m0 *= BM;
    const uint32_t kb0 = blockIdx.y * kb_per_split, kb1 = min(kb0 + kb_per_split, g.kb);

    // Loads: instruction j of a wave fills eight rows; this lane's row and piece of instructions 0 and 1, the others 16 rows further
    // each.  The buffers' limits are checked on the lane's offset: a row behind the end, or a piece behind the end of K, reads as
    // zeros.  (The block's offset k0 stands outside of the check: a lane in a row and in K stays in that row.)
    const uint32_t l_row = lane >> 3, piece[2] = {((lane & 7u) ^ (l_row >> 1)) * 16u, ((lane & 7u) ^ (l_row >> 1) ^ 4u) * 16u};
    const __amdgpu_buffer_rsrc_t w_buf = buffer_of(g.w + (size_t)n0 * g.k, min((uint32_t)BN, g.n - n0) * g.k);
    const __amdgpu_buffer_rsrc_t a_buf = buffer_of(g.a + (size_t)m0 * g.k, min((uint32_t)BM, g.m - m0) * g.k);
    const uint32_t w_row = (wave * LW * 8u + l_row) * g.k, a_row = (wave * LA * 8u + l_row) * g.k;
    auto load = [&](uint32_t buf, uint32_t b, int part) {
        const int j = part < LW ? part : part - LW;
        const uint32_t k0 = b * 128u, in_k = piece[j & 1] < g.k - k0, from = (part < LW ? w_row : a_row) + piece[j & 1] + j * 8u * g.k;
        uint8_t *to = part < LW ? &tile.w[buf][(wave * LW + j) * 1024u] : &tile.a[buf][(wave * LA + j) * 1024u];
        __builtin_amdgcn_raw_ptr_buffer_load_lds(part < LW ? w_buf : a_buf, (LdsPtr)to, 16, in_k ? from : 0xFFFFFFFFu, k0, 0, 0);
    };
    // Scales of blocks kb0 + 4 c .. + 3 of a row per lane, 64 rows a wave; where a row has no four blocks left, one by one
    const float *as = g.a_scales + (size_t)m0 * g.kb;
    const __amdgpu_buffer_rsrc_t as_buf = buffer_of(as, min((uint32_t)BM, g.m - m0) * g.kb * 4u);
    auto load_scales = [&](uint32_t c) {
        if (wave >= BM / 64) return;
        const uint32_t r = wave * 64u + lane, b = kb0 + 4u * c;
        float *to = &tile.scales[c & 1u][wave * 256u];
        if (b + 4u <= g.kb) {
            __builtin_amdgcn_raw_ptr_buffer_load_lds(as_buf, (LdsPtr)to, 16, r * g.kb * 4u, b * 4u, 0, 0);
        } else {
            const float *from = as + (size_t)min(r, g.m - 1u - m0) * g.kb;
            *(float4v *)(to + lane * 4u) = float4v{from[min(b, g.kb - 1u)], from[min(b + 1u, g.kb - 1u)], from[min(b + 2u, g.kb - 1u)], from[g.kb - 1u]};
        }
    };

    uint32_t at[4];   // this lane's pieces of an operand tile
    Mfma::places(lane, at);
    const uint32_t row = lane % S;   // the lane's row of A in a tile
    // (columns behind the end have no scale: any block's will do)
    const TWM_CONSTANT float *ws_row = (const TWM_CONSTANT float *)(g.w_scales + (size_t)min((n0 + wn * TN * S) >> 7, (g.n - 1u) >> 7) * g.kb);
    // the factor of row tile j in the block `done` blocks from kb0
    auto scale = [&](int j, uint32_t done) { return tile.scales[done >> 2 & 1u][((wm * TM + j) * S + row) * 4u + (done & 3u)]; };

    typename Mfma::Sum acc[TN][TM];
#pragma unroll
    for (int i = 0; i < TN; i++)
#pragma unroll
        for (int j = 0; j < TM; j++) acc[i][j] = typename Mfma::Sum{};

    if (kb0 < kb1) {
        load_scales(0);
#pragma unroll
        for (int part = 0; part < PARTS; part++) load(0, kb0, part);
#pragma unroll
        for (int part = 0; part < EARLY; part++)
            if (kb0 + 1 < kb1) load(1, kb0 + 1, part);
        Mfma w[2], a[TM];
        float s_next[TM], ws_next = ws_row[kb0];
        __builtin_amdgcn_s_waitcnt(0);
        __syncthreads();
#pragma unroll
        for (int j = 0; j < TM; j++) s_next[j] = scale(j, 0);
        w[0].read(&tile.w[0][wn * TN * S * 128u], at);
#pragma unroll
        for (int j = 0; j < TM; j++) a[j].read(&tile.a[0][(wm * TM + j) * S * 128u], at);
        // (the buffer is a constant of each of two copies of the step, so that LDS addresses are a register and an offset)
        auto step = [&](auto which, uint32_t b) {
            constexpr uint32_t buf = decltype(which)::value;
            float s[TM];
#pragma unroll
            for (int j = 0; j < TM; j++) s[j] = s_next[j] * ws_next;
            const uint32_t done_b = b - kb0;
            ws_next = ws_row[b + 1 < kb1 ? b + 1 : b];
            typename Mfma::Sum d[DEPTH];
#pragma unroll
            for (int t = 0; t < TN * TM + DEPTH - 1; t++) {
                const int i = t / TM, j = t % TM;
                if (t < TN * TM) {
                    if (j == 0) {
                        if (i + 1 < TN) {
                            w[(i + 1) & 1].read(&tile.w[buf][(wn * TN + i + 1) * S * 128u], at);
                        } else {
                            // every operand of this block is in registers: once all waves are here the buffer can be filled again,
                            // and the next block is complete
                            __builtin_amdgcn_s_waitcnt(0);
                            __builtin_amdgcn_s_barrier();
                            // (four blocks' scales ahead of their first use, when the half that they replace has been read)
                            if ((done_b & 3u) == 1u && b + 3 < kb1) load_scales((done_b >> 2) + 1u);
#pragma unroll
                            for (int jj = 0; jj < TM; jj++) s_next[jj] = scale(jj, done_b + 1u);
                            w[(i + 1) & 1].read(&tile.w[buf ^ 1u][wn * TN * S * 128u], at);
                        }
                    }
                    d[t % DEPTH] = Mfma::product(w[i & 1], a[j]);
                    const int last_row = t - (TN - 1) * TM;
#pragma unroll
                    for (int part = 0; part < PER && t % EVERY == 0; part++) {
                        const int early = last_row / EVERY * PER + part, late = EARLY + t / EVERY * PER + part;
                        if (last_row >= 0 && early < EARLY && b + 2 < kb1) load(buf, b + 2, early);
                        if (late < PARTS && b + 1 < kb1) load(buf ^ 1u, b + 1, late);
                    }
                    if (i == TN - 1) a[j].read(&tile.a[buf ^ 1u][(wm * TM + j) * S * 128u], at);
                }
                const int done = t - (DEPTH - 1);
                if (done >= 0) {
                    typename Mfma::Sum &sum = acc[done / TM][done % TM];
                    sum += d[done % DEPTH] * s[done % TM];
                    asm volatile("" : "+v"(sum));   // (here: the compiler moved these down past all products, whose results then held a register each)
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        for (uint32_t b = kb0; b < kb1; b += 2) {
            step(std::integral_constant<uint32_t, 0>{}, b);
            if (b + 1 < kb1) step(std::integral_constant<uint32_t, 1>{}, b + 1);
        }
    }
    store_tile<S, TN, TM>(g, acc, lds, wave, lane, m0 + wm * TM * S, n0 + wn * TN * S, partials, n_ld);
}

// The sum of the K-ranges' results, in their order; a thread per four columns.
__global__ __launch_bounds__(256) void k_fp8_splits(const Fp8Gemm g, const float *__restrict__ partials, uint32_t n_ld, uint32_t splits)
{
    const uint64_t i = (uint64_t)blockIdx.x * 256u + threadIdx.x;
    const uint32_t quads = n_ld / 4u;
    const uint64_t m = i / quads;
    if (m >= g.m) return;
    const uint32_t n = (uint32_t)(i - m * quads) * 4u;
    const float *at = partials + m * n_ld + n;
    const size_t step = (size_t)g.m * n_ld;
    float4v s = *(const float4v *)at;
    for (uint32_t z = 1; z < splits; z++) s += *(const float4v *)(at + z * step);
    store_quad(g, (uint32_t)m, n, s);
}

namespace {

// columns x rows of a form, its kernel, and what it was measured to take: us per block of 128 features of a workgroup alone on a
// CU, of one among as many as the CU holds, per workgroup besides, and per block for a part of W that no other row block reads
struct Fp8Form {
    uint32_t bn, bm, threads, lds;
    void (*kernel)(const Fp8Gemm, uint32_t, uint32_t, uint32_t, float *, uint32_t);
    uint32_t per_cu;
    float block_alone, block_among, besides, block_cold;
};
#define TWM_FP8_FORM(S, TN, TM, WN, WM, ...) \
    Fp8Form{S * TN * WN, S * TM * WM, WN * WM * 64, (uint32_t)sizeof(Fp8Tile<S * TM * WM, S * TN * WN>), k_fp8_tile<S, TN, TM, WN, WM>, __VA_ARGS__}
const Fp8Form kFp8Forms[] = {
    TWM_FP8_FORM(16, 8, 4, 2, 4, 1, 1.55f, 0.52f, 4.6f, 0.00f),   // 256 columns x 256 rows, eight waves
    TWM_FP8_FORM(16, 4, 4, 2, 2, 2, 0.68f, 0.49f, 2.6f, 0.05f),   // 128 x 128
    TWM_FP8_FORM(16, 4, 2, 2, 2, 3, 0.57f, 0.37f, 0.9f, 0.04f),   // 128 columns x 64 rows
    TWM_FP8_FORM(32, 2, 2, 2, 2, 2, 0.91f, 0.72f, 3.9f, 0.00f),   // 128 x 128, sums of exact products
    TWM_FP8_FORM(32, 2, 1, 2, 2, 3, 0.64f, 0.48f, 1.7f, 0.13f),   // 128 columns x 64 rows, sums of exact products
};
constexpr uint32_t kFp8Fast = 3, kFp8FormCount = sizeof kFp8Forms / sizeof kFp8Forms[0];   // the first ones: 8-bit instructions

hipError_t launch_fp8_tile(hipStream_t s, const Fp8Gemm &g, uint32_t form, uint32_t splits, float *ws, size_t ws_bytes)
{
    const Fp8Form &f = kFp8Forms[form];
    const uint32_t bn = (g.n + f.bn - 1) / f.bn, bm = (g.m + f.bm - 1) / f.bm, n_ld = (g.n + 3u) & ~3u;
    const uint32_t per = splits > 1 ? (g.kb + splits - 1) / splits : g.kb;
    // (the planner's splits fit, and its forms with 8-bit instructions are for f16 results, the others for f32)
    if ((splits > 1 && (uint64_t)splits * g.m * n_ld * 4 > ws_bytes) || (form < kFp8Fast) != (g.c_f16 != 0)) return hipErrorInvalidValue;
    float *partials = splits > 1 ? ws : nullptr;
    hipLaunchKernelGGL(f.kernel, dim3(bn * bm, splits), dim3(f.threads), f.lds, s, g, bn, bm, per, partials, n_ld);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || splits == 1) return e;
    hipLaunchKernelGGL(k_fp8_splits, dim3((unsigned)(((uint64_t)g.m * (n_ld / 4) + 255) / 256)), dim3(256), 0, s, g, partials, n_ld, splits);
    return hipGetLastError();
}

// columns per workgroup (in 16s), blocks in flight and waves of the kernel for few rows; 16 * MT rows
template <int MT, int NT, int U, int WAVES>
hipError_t launch_fp8_few(hipStream_t s, const Fp8Gemm &g, uint32_t splits, float *ws, size_t ws_bytes)
{
    const uint32_t n_ld = (g.n + 3u) & ~3u, per = splits > 1 ? (g.kb + splits - 1) / splits : g.kb;
    if (splits > 1 && (uint64_t)splits * g.m * n_ld * 4 > ws_bytes) return hipErrorInvalidValue;
    float *partials = splits > 1 ? ws : nullptr;
    auto kernel = g.k % 128 ? k_fp8_rows_few<MT, NT, U, WAVES, true> : k_fp8_rows_few<MT, NT, U, WAVES, false>;
    hipLaunchKernelGGL(kernel, dim3((g.n + 16u * NT - 1) / (16u * NT), (g.m + 16u * MT - 1) / (16u * MT), splits), dim3(WAVES * 64), 0, s, g, per,
                       partials, n_ld);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || splits == 1) return e;
    hipLaunchKernelGGL(k_fp8_splits, dim3((unsigned)(((uint64_t)g.m * (n_ld / 4) + 255) / 256)), dim3(256), 0, s, g, partials, n_ld, splits);
    return hipGetLastError();
}

// Which kernel: few = 1: k_fp8_rows_few in that of kFp8OneForms, 2, 4: with that many times 16 rows and `form` times 16 columns; 0:
// k_fp8_tile in `form`.  splits: ranges of K.
struct Fp8Plan {
    uint32_t few, form, splits;
};

constexpr double kFp8Bandwidth = 8.9e6, kFp8SplitBandwidth = 6.7e6;             // bytes per us: operands from memory; ranges' sums out and in
constexpr double kFp8Launch = 1.93, kFp8SecondLaunch = 1.65, kFp8PerSplit = 0.33;   // us

// Up to 16 rows: columns (in 16s) and waves of the kernel for few rows
struct Fp8OneForm {
    uint32_t nt, waves;
    hipError_t (*launch)(hipStream_t, const Fp8Gemm &, uint32_t, float *, size_t);
};
enum : uint32_t { kOneNarrow, kOneNarrowDeep, kOneTwo, kOneTwoShallow, kOneMany };
const Fp8OneForm kFp8OneForms[] = {{1, 8, launch_fp8_few<1, 1, 2, 8>}, {1, 16, launch_fp8_few<1, 1, 2, 16>}, {2, 16, launch_fp8_few<1, 2, 1, 16>},
                                   {2, 8, launch_fp8_few<1, 2, 1, 8>}, {1, 4, launch_fp8_few<1, 1, 2, 4>}};

// One round of workgroups where there is one (of 32 columns where 16 would take two; 1 x 3584 x 4608 6.3 us, of 16 6.5, at 8 rows 7.0
// and 8.1; 1 x 37888 x 3584 24.7 and 25.5, at 16 rows 31 and 39).  On narrow matrices two blocks a wave in flight in eight waves
// (1 x 1100 x 4864 4.9 us, one in sixteen 5.1; 16 x 4096 x 2816 5.1 and 5.3), in sixteen where a few rows wait for much from memory
// (1 x 4096 x 18944 15.4, in eight 18.4).  A long K is shared out: among four ranges where the columns fill less than half the CUs
// (1 x 1100 x 18944 9.7 us, in one 13.3; 16 rows 12.0 and 20.3; 16 x 1100 x 8960 8.3 and 10.3), two where the rows are many enough for their
// products to count (16 x 4096 x 18944 20.7 and 23.9, 8 x 3584 x 18944 16.7 and 20.4).
void fp8_one_form(uint32_t m, uint32_t n, uint32_t k, uint32_t &form, uint32_t &splits)
{
    const uint32_t tiles = (n + 15u) / 16u, kb = (k + 127u) / 128u;
    splits = 1;
    if (tiles > 512u) {
        form = tiles <= 1024u ? kOneMany : k < 16u * 128u ? kOneTwoShallow : kOneTwo;
    } else if (tiles > 256u) {
        form = k < 16u * 128u ? kOneTwoShallow : kOneTwo;
    } else if ((tiles <= 128u && kb >= 64u) || (m >= 8u && kb >= 80u)) {
        form = kOneTwoShallow;
        splits = tiles <= 128u ? 4u : 2u;
    } else {
        form = m <= 4u && (uint64_t)n * k > 22000000u ? kOneNarrowDeep : kOneNarrow;
    }
}

// The kernel for few rows above 16 of them, us: a launch, eight blocks of 128 features, a block of a workgroup alone on a CU, one of many,
// and a workgroup besides
struct Fp8FewForm {
    uint32_t mt, nt;
    double launch, eight, block_alone, block_among, besides;
};
const Fp8FewForm kFp8FewForms[] = {{2, 1, 2.32, 0.08, 0.148, 0.193, 0.114}, {4, 1, 2.13, 0.26, 0.316, 0.387, 0.099}, {4, 2, 2.0, 0.50, 0.375, 0.474, 0.213}};

// Up to 16 rows the kernel for few rows (8 x 3584 x 3584 5.4 us, in tiles 8.5; 16 x 3739 x 15200 19.6 and 20.5; only above a hundred MB of
// weights are tiles a tenth ahead).  Above, whichever is expected to take the least time, by the figures above: fitted to the
// times of 370 shapes of 17 .. 2048 rows in every form and split, of which the choice is 0.8 % behind the best in the mean.  (The kernel
// for few rows is ahead where tiles are far fewer than CUs: 200 x 851 x 1024 5.8 us, in tiles 6.9 for f16 results and 8.5 for f32.)
Fp8Plan plan_fp8(uint32_t m, uint32_t n, uint32_t k, bool f16, size_t ws_bytes)
{
    const uint32_t kb = (k + 127u) / 128u;
    const uint64_t n_ld = (n + 3u) & ~3u;
    if (m <= 16) {
        Fp8Plan one = {1, 0, 1};
        fp8_one_form(m, n, k, one.form, one.splits);
        const uint32_t per = (kb + one.splits - 1) / one.splits;
        one.splits = per ? (kb + per - 1) / per : 1;
        if (one.splits * m * n_ld * 4 > ws_bytes) one.splits = 1;
        return one;
    }
    Fp8Plan best = {0, f16 ? kFp8Fast - 1 : kFp8FormCount - 1, 1};
    double least = 1e30;
    static const uint32_t kSplits[] = {1, 2, 3, 4, 6, 8, 12, 16};
    for (uint32_t want : kSplits) {
        if (want > 1 && kb / want < 2) break;
        const uint32_t per = want > 1 ? (kb + want - 1) / want : kb, splits = per ? (kb + per - 1) / per : 1;
        if (splits > 1 && splits * m * n_ld * 4 > ws_bytes) break;
        const double joined = splits > 1 ? kFp8SecondLaunch + kFp8PerSplit * splits + (double)splits * m * n * 8 / kFp8SplitBandwidth : 0.0;
        for (uint32_t i = f16 ? 0 : kFp8Fast; i < (f16 ? kFp8Fast : kFp8FormCount); i++) {
            const Fp8Form &f = kFp8Forms[i];
            const uint32_t blocks_m = (m + f.bm - 1) / f.bm;
            const uint64_t groups = (uint64_t)((n + f.bn - 1) / f.bn) * blocks_m * splits, full = groups / (256u * f.per_cu),
                           rest = (groups % (256u * f.per_cu) + 255u) / 256u;
            if (splits > 1 && groups > 1100) continue;
            const double alone = f.block_alone + f.block_cold / blocks_m;
            auto turn = [&](uint64_t among) { return per * (alone > among * f.block_among ? alone : among * f.block_among) + f.besides; };
            double us = full * turn(f.per_cu) + (rest ? turn(rest) : 0.0);
            const double memory = ((double)n * k + (double)m * k) / kFp8Bandwidth;
            us = (us > memory ? us : memory) + kFp8Launch + joined;
            if (us < least) {
                least = us;
                best = Fp8Plan{0, i, splits};
            }
        }
        for (const Fp8FewForm &f : kFp8FewForms) {
            const uint64_t tiles = (uint64_t)((n + 16 * f.nt - 1) / (16 * f.nt)) * ((m + 16 * f.mt - 1) / (16 * f.mt)), groups = tiles * splits;
            // (32 columns, with less than four blocks: most of the eight waves have none; 38 x 9269 x 256 5.8 us, in tiles 4.2)
            if (m > 400 || (m <= 32) != (f.mt == 2) || (f.nt == 2 && kb < 4) || (splits > 1 && (splits > 4 || tiles > 192 || kb / splits < 4))) continue;
            const double alone = per * f.block_alone, among = groups * (per * f.block_among + f.besides) / 256;
            const double us = f.launch + (per + 7) / 8 * f.eight + (alone > among ? alone : among) + joined;
            if (us < least) {
                least = us;
                best = Fp8Plan{f.mt, f.nt, splits};
            }
        }
    }
    return best;
}

}  // namespace

// Once per device, outside any stream capture: the forms with more LDS than a launch gets unasked.
hipError_t init_fp8_gemm()
{
    for (const Fp8Form &f : kFp8Forms) {
        const hipError_t e = hipFuncSetAttribute((const void *)f.kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)f.lds);
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

hipError_t launch_fp8_gemm(hipStream_t s, const uint8_t *a, const float *a_scales, const uint8_t *w, const float *w_scales, uint32_t m,
                           uint32_t n, uint32_t k, void *c, bool c_f16, float *ws, size_t ws_bytes)
{
    if (m == 0 || n == 0) return hipSuccess;
    const Fp8Gemm g = {a, w, a_scales, w_scales, m, n, k, (k + 127u) / 128u, c, c_f16 ? 1u : 0u};
    const Fp8Plan plan = plan_fp8(m, n, k, c_f16, ws_bytes);
    if (plan.few == 0) return launch_fp8_tile(s, g, plan.form, plan.splits, ws, ws_bytes);
    if (plan.few == 2) return launch_fp8_few<2, 1, 1, 8>(s, g, plan.splits, ws, ws_bytes);
    if (plan.few == 4 && plan.form == 1) return launch_fp8_few<4, 1, 1, 8>(s, g, plan.splits, ws, ws_bytes);
    if (plan.few == 4) return launch_fp8_few<4, 2, 1, 8>(s, g, plan.splits, ws, ws_bytes);
    return kFp8OneForms[plan.form].launch(s, g, plan.splits, ws, ws_bytes);
}

void describe_fp8_gemm(uint32_t m, uint32_t n, uint32_t k, bool c_f16, size_t ws_bytes, char *text, size_t bytes)
{
    const Fp8Plan plan = plan_fp8(m, n, k, c_f16, ws_bytes);
    if (m == 0 || n == 0) {
        snprintf(text, bytes, "nothing to launch");
    } else if (plan.few == 0) {
        const Fp8Form &f = kFp8Forms[plan.form];
        snprintf(text, bytes, "k_fp8_tile: %u columns x %u rows, %u waves, %s instructions, %u K-split%s", f.bn, f.bm, f.threads / 64, plan.form < kFp8Fast ? "8-bit" : "f16",
                 plan.splits, plan.splits == 1 ? "" : "s");
    } else {
        const uint32_t nt = plan.few == 1 ? kFp8OneForms[plan.form].nt : plan.form, waves = plan.few == 1 ? kFp8OneForms[plan.form].waves : 8u;
        snprintf(text, bytes, "k_fp8_rows_few: %u columns x %u rows, %u waves, f16 instructions, %u K-split%s", 16u * nt, 16u * plan.few, waves, plan.splits,
                 plan.splits == 1 ? "" : "s");
    }
}

}  // namespace twm
