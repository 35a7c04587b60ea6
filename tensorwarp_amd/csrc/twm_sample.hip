// One token per row of logits, from a uniform number that the caller gives: temperature, top-k, top-p and min-p.
//
//   w[i] = exp((x[i] - max x) / temperature), in 64 bits, kept as the whole number round(w * 2^S): sums of whole numbers do not
//   depend on their order, so that every way of sharing a row out gives the same token.  S is the largest that keeps the sum of
//   a row of that many columns below 2^63 (44 at 152064 columns); a token whose weight rounds to nothing (below 2^-45 of the
//   largest) is never chosen.
//   In descending order of x, equal ones by index, the first top_k tokens remain; of these the shortest run that holds top_p of
//   their sum (a token stays while the sum before it is below that); of these the tokens with w >= min_p.  Each rule keeps a
//   prefix of the order, so what remains is the tokens whose key -- the bits of x that order as x does, then the inverted
//   index -- is at least one 64-bit number, and with w >= min_p.
//   The token is the first by index at which the running sum of what remains exceeds u times the whole.
//
// How a row is worked through: its largest logit; then, where top-k or top-p ask for it, a histogram of the tokens' numbers and
// weights over 2048 bins of (max - x) / temperature, 1/64 wide or narrower, in LDS; from its running sums the one or two bins in which top-k
// and top-p end; then one more pass that adds the weights of the tokens in the bins before those and lists the tokens in them
// (some hundred), whose exact order is settled by ranges of their keys until a wave's lanes hold them; and at last the running sum
// through the one part of the row that u falls into.  A row whose list would be too long (thousands of nearly equal logits) is
// settled eight bits of the key at a time instead.  Many rows, or short ones: a workgroup each, one launch.  A few long
// rows: parts of a row each have a workgroup, in up to three launches, the last workgroup of a row to arrive doing what concerns the
// whole row.
//
// Measured: 1 row of 152064 logits 14 us without limits, 20 with top-k, 24 with top-k and top-p, 25 with top-p; 32 such rows 43 with
// top-p and 33 with both; 256 rows of 32000 23 without limits, 25, 28 and 40.  Bound: for one row latency (three launches, 2.5 us from
// the end of one to the first load of the next; the passes themselves 1 to 3 us; histogram to cut and list to token 4 and 7); for many
// rows the vector instructions of the weights, 33 a token in each of two passes, eighteen of them in 64 bits: of 40 us for 256 rows of
// 32000 the largest logit takes 6, the histogram 11, the cut 1.5, adding and listing 12, settling the list 3, the token 3.  Rows kept in
// registers over the passes (25.5 us instead of 27.2 with both limits, 24.4 instead of 22.7 without any) and the tokens that are in
// gathered ahead of their weights (40.1 and 40.3) were not worth their code.
#include "twm_device.h"
#include "twm_slices.h"

namespace twm {

namespace {

constexpr uint32_t kSampleBins = 2048, kSampleList = 2048, kSampleSpans = 64;
// A top_k up to which its tokens are listed one and all: a quarter of the list, the rest for those next to the last; on rows of up to
// kSampleShort columns fewer than a wave's lanes
constexpr uint32_t kSampleListAll = 512, kSampleListAllShort = 56, kSampleShort = 12288;
constexpr uint32_t kSampleBatch = 8;          // loads of a thread in flight
constexpr uint32_t kSamplePart = 4096;        // columns of a part, or a multiple: half a batch of 1024 threads
constexpr uint32_t kSampleCounterStep = 32;   // a row's arrival counter has a cache line of its own
constexpr uint32_t kNoBin = 0xFFFFFFFFu;
constexpr uint32_t kSampleGroups = 256;       // workgroups that run at once, one a compute unit

// a number that orders as the float does (-0 as 0); NaN below everything
__device__ __forceinline__ uint32_t sample_order(float v)
{
    const uint32_t u = __float_as_uint(v + 0.0f);
    return v != v ? 0u : u ^ ((uint32_t)((int)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float sample_value(uint32_t order)
{
    return __uint_as_float(order & 0x80000000u ? order ^ 0x80000000u : ~order);
}
// a token's place in the order: larger for a larger logit and, among equal ones, for a smaller index
__device__ __forceinline__ uint64_t sample_key(float v, uint32_t i) { return (uint64_t)sample_order(v) << 32 | (0xFFFFFFFFu - i); }

// a * b + c with c, the same for all lanes, in scalar registers (the compiler would copy c into the result's registers first, as many
// instructions again: 256 rows of 32000 49 us instead of 45)
__device__ __forceinline__ double times_plus(double a, double b, double c)
{
    double r;
    asm("v_fma_f64 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "s"(c));
    return r;
}

// One row's inputs
struct SampleArgs {
    const float *logits, *uniform, *temperature, *top_p, *min_p;
    const int *top_k;
    int *out;
    uint32_t cols, spans, span;   // a row's parts: `spans` of `span` columns, the last one shorter
    uint32_t each;                // parts per workgroup
    int s;                        // S
};

struct SampleRules {
    float largest, finite;             // finite: the largest, or 0 for an infinity
    float per_bin, deepest;            // bins / temperature, in 32 bits; depth (see there) from which on weights are nothing
    double log2_one, top_p, least, uniform;   // log2_one = 64 log2(e) / temperature; least = 2^S min_p
    uint64_t top_k;        // 0: no limit
    uint32_t list_all;
    const double *power;   // 2^(S + j / 64), j = 0 .. 63, in LDS
    bool greedy;

    // round(2^S w) of one logit, and whether w is at least min_p (any answer where the weight is nothing).  2^z = 2^(n / 64) 2^(f / 64),
    // n whole and |f| <= 1/2: the first from a table of 64 numbers and the exponent, the second the exponential's series up to the
    // fifth power, whose rest is below 2^-54.  (Without the table the series needs twelve powers, and the passes that call this are
    // bound by its instructions: 256 rows of 32000 45 us instead of 43.)  n comes from adding 1.5 2^52, which leaves it in the
    // low bits: no conversion but the first, no branch.  Nothing below e^-40 < 2^-57.
    __device__ __forceinline__ uint64_t weight(float v, bool &above) const
    {
        const bool top = v == largest;
        const bool any = depth(v) <= deepest;   // (NaN: a NaN)
        const double d = (double)(top ? finite : v) - (double)finite, at = fma(d, log2_one, 6755399441055744.0);
        const uint32_t n = (uint32_t)__double2loint(at);
        const double f = fma(d, log2_one, 6755399441055744.0 - at), p = power[n % 64u];
        constexpr double c = 0.6931471805599453 / 64.0;
        double e = times_plus(f, c * c * c * c * c / 120.0, c * c * c * c / 24.0);
        e = times_plus(e, f, c * c * c / 6.0);
        e = times_plus(e, f, c * c * 0.5);
        e = times_plus(e, f, c);
        e = fma(p * f, e, p);
        e = __hiloint2double(__double2hiint(e) + (int)((n & ~63u) << 14), __double2loint(e));
        above = e >= least;
        // (2^52 added leaves the nearest whole number in the low bits)
        const uint64_t whole = (uint64_t)__double_as_longlong(e + 4503599627370496.0) & 0xFFFFFFFFFFFFFull;
        return any ? whole : 0;
    }
    // the weight of a token that is above min_p, else 0
    __device__ __forceinline__ uint64_t kept(float v) const
    {
        bool above;
        const uint64_t whole = weight(v, above);
        return above ? whole : 0;
    }
    // bins (largest - v) / temperature: falls as v grows, like its weight's logarithm; every rounding in it keeps the order
    __device__ __forceinline__ float depth(float v) const { return v == largest ? 0.0f : (largest - v) * per_bin; }
    __device__ __forceinline__ uint32_t bin(float v) const
    {
        const float f = depth(v);
        return f < (float)(kSampleBins - 1) ? (uint32_t)f : kSampleBins - 1;
    }
    // the depth at which a bin begins: bin(v) < b is depth(v) < begin(b), for every b up to kNoBin (but for infinite depths, whose weight
    // is nothing)
    static __device__ __forceinline__ float begin(uint32_t b) { return b < kSampleBins ? (float)b : INFINITY; }
    __device__ __forceinline__ bool limited() const { return top_k != 0 || top_p < 1.0; }
    // Whether the tokens of the bins are counted only: top_p does not matter, or it is settled among the listed tokens, which are then
    // all of the first top_k (the weights of the others are not needed: 256 rows of 32000 with both limits 27.2 us instead of 33.3, with
    // top-k alone 24.1 instead of 30.2).  On short rows only if the list then is short enough to be compared at once, since narrowing it
    // takes more than the weights do (100 rows of 1000 with top_k 50 13.4 us
    // instead of 15.0, but with top_k up to 99 16.2 instead of 14.7; 256 of 16000 24.8 and 25.0).
    __device__ __forceinline__ bool counted() const { return top_k != 0 && (top_p >= 1.0 || top_k <= list_all); }
};

// What a pass over the row leaves: the largest key, and the smallest logit above -infinity, as the inverted number that orders as it
// does (0: none)
struct SampleEnds {
    uint64_t key;
    uint32_t low;
};

__device__ __forceinline__ SampleRules sample_rules(const SampleArgs &a, const double *power, uint32_t row, const SampleEnds &ends)
{
    const float largest = sample_value((uint32_t)(ends.key >> 32));
    SampleRules r;
    r.largest = largest;
    r.finite = fabsf(largest) < INFINITY ? largest : 0.0f;
    const float t = a.temperature ? a.temperature[row] : 1.0f, p = a.top_p ? a.top_p[row] : 1.0f, m = a.min_p ? a.min_p[row] : 0.0f;
    const int k = a.top_k ? a.top_k[row] : 0;
    r.greedy = !(t > 0.0f);
    r.log2_one = 64.0 * 1.4426950408889634 / (double)t;
    // 64 bins for a factor of e; more where the row's logits are so close that it needs less than all 2048 bins (thousands of tokens would
    // share one, too many for the list: 152064 logits of a deviation of 0.1, top-p, 363 us with 64, 27 so).  2040: those of a last
    // rounding stay below 2047.
    const float per_one = 1.0f / t, range = (largest - sample_value(~ends.low)) * per_one, more = 2040.0f * __builtin_amdgcn_rcpf(fmaxf(range, 1e-3f));
    const float bins = range < 31.0f && more * per_one < 1e37f ? more : 64.0f;   // (NaN: 64)
    r.per_bin = bins * per_one;
    r.deepest = 40.0f * bins;
    r.top_p = p < 1.0f ? (double)p : 1.0;   // (NaN: no limit)
    r.power = power;
    r.least = ldexp(m < 1.0f ? (double)m : m != m ? 0.0 : 1.0, a.s);   // (NaN: no limit; the largest always remains)
    r.top_k = k > 0 && (uint32_t)k < a.cols ? (uint64_t)k : 0u;
    r.list_all = a.cols > kSampleShort ? kSampleListAll : kSampleListAllShort;
    r.uniform = a.uniform[row];
    return r;
}

// Where the limits end, from the histogram: the tokens of bin k_bin are the last of the first top_k; p_first .. p_last are the
// bins in which top_p can end (which one depends on the tokens of k_bin that are in).  kNoBin: no such limit.
struct SampleCut {
    uint32_t k_bin, p_first, p_last;
    uint32_t above_k;          // tokens in the bins before k_bin
    uint32_t all;              // every token that may remain is listed (p_first 0, masses 0)
    uint64_t mass_k, mass_p;   // weights in the bins before k_bin and before p_first; mass_k: of all bins where there is no k_bin

    // bins before sure() are in, those from behind() on are out (p_last is k_bin at most where both are there)
    __device__ __forceinline__ uint32_t behind() const { return k_bin != kNoBin ? k_bin + 1u : p_last != kNoBin ? p_last + 1u : kNoBin; }
    __device__ __forceinline__ uint32_t sure() const { return p_first != kNoBin ? p_first : k_bin; }
    __device__ __forceinline__ bool listed(uint32_t b) const { return b == k_bin || (b >= p_first && b <= p_last && p_first != kNoBin); }
};

// What a row's workgroups leave for each other between and within launches
struct SampleRow {
    uint64_t key[kSampleSpans], mass[kSampleSpans];
    uint32_t low[kSampleSpans];
    uint64_t bin_mass[kSampleBins];
    uint32_t bin_count[kSampleBins];
    uint64_t list_key[kSampleList], list_mass[kSampleList];
    SampleCut cut;
    uint32_t listed;
};

struct SampleShared {
    struct {
        uint64_t mass[kSampleBins];
        uint32_t count[kSampleBins];
    } bins;
    struct {
        uint64_t key[kSampleList];
        uint64_t mass[kSampleList];   // bit 63: the token is above min_p
    } list;
    double power[64];
    uint64_t few_key[64], few_mass[64], few_before[64];
    uint32_t few_count[64];
    uint64_t spans[kSampleSpans];
    uint64_t wave64[16];
    uint32_t wave32[16];
    SampleCut cut;
    SampleEnds ends;
    uint64_t prefix, taken_mass, least, low, high;
    uint32_t listed, taken_count, stop, base;
};

// the sums up to and with each lane (DPP: shifts within sixteen lanes, then their last lane to the lanes behind); LANES 16: within each
// sixteen
template <uint32_t LANES = 64> __device__ __forceinline__ uint64_t wave_running(uint64_t v)
{
#define TWM_SCAN_STEP(CTRL, ROWS) \
    v += (uint64_t)(uint32_t)__builtin_amdgcn_update_dpp(0, (int)(v >> 32), CTRL, ROWS, 0xf, false) << 32 | \
         (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, false)
    TWM_SCAN_STEP(0x111, 0xf);   // row_shr:1
    TWM_SCAN_STEP(0x112, 0xf);
    TWM_SCAN_STEP(0x114, 0xf);
    TWM_SCAN_STEP(0x118, 0xf);
    if (LANES == 64) {
        TWM_SCAN_STEP(0x142, 0xa);   // row_bcast:15 into the second and fourth sixteen
        TWM_SCAN_STEP(0x143, 0xc);   // row_bcast:31 into the upper half
    }
#undef TWM_SCAN_STEP
    return v;
}
template <uint32_t LANES = 64> __device__ __forceinline__ uint32_t wave_running(uint32_t v)
{
#define TWM_SCAN_STEP(CTRL, ROWS) v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, false)
    TWM_SCAN_STEP(0x111, 0xf);
    TWM_SCAN_STEP(0x112, 0xf);
    TWM_SCAN_STEP(0x114, 0xf);
    TWM_SCAN_STEP(0x118, 0xf);
    if (LANES == 64) {
        TWM_SCAN_STEP(0x142, 0xa);
        TWM_SCAN_STEP(0x143, 0xc);
    }
#undef TWM_SCAN_STEP
    return v;
}
__device__ __forceinline__ uint64_t lane_value(uint64_t v, int lane)
{
    return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), lane) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)v, lane);
}
__device__ __forceinline__ uint64_t wave_sum_u64(uint64_t v) { return lane_value(wave_running(v), 63); }
__device__ __forceinline__ uint32_t wave_most_u32(uint32_t v)
{
#define TWM_MAX_STEP(N) v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x120 + N, 0xf, 0xf, true))   // row_ror:N
    TWM_MAX_STEP(8);
    TWM_MAX_STEP(4);
    TWM_MAX_STEP(2);
    TWM_MAX_STEP(1);
#undef TWM_MAX_STEP
    const uint32_t a = __builtin_amdgcn_readlane(v, 0), b = __builtin_amdgcn_readlane(v, 16);
    const uint32_t c = __builtin_amdgcn_readlane(v, 32), d = __builtin_amdgcn_readlane(v, 48);
    return max(max(a, b), max(c, d));
}
__device__ __forceinline__ uint64_t wave_most_u64(uint64_t v)
{
    const uint32_t high = wave_most_u32((uint32_t)(v >> 32));
    return (uint64_t)high << 32 | wave_most_u32((uint32_t)(v >> 32) == high ? (uint32_t)v : 0u);
}

template <uint32_t THREADS> struct Sampler {
    static_assert(kSampleBatch * THREADS == 2 * kSamplePart);
    static constexpr uint32_t kWaves = THREADS / 64;
    static_assert(kWaves == 16);   // (a value per wave is summed by sixteen lanes)
    const SampleArgs &a;
    SampleShared &sh;
    const float *x;
    uint32_t row, tid, lane, wave;

    __device__ __forceinline__ Sampler(const SampleArgs &args, SampleShared &shared, uint32_t r)
        : a(args), sh(shared), x(args.logits + (size_t)r * args.cols), row(r), tid(threadIdx.x), lane(threadIdx.x & 63u), wave(__builtin_amdgcn_readfirstlane(threadIdx.x >> 6))
    {
    }

    // f(v, i, j) for the columns of parts first .. last of the row, the j-th of a batch of eight loads, and for NaN in place of those
    // behind the last (a NaN is never chosen: what f does with one, it does with these); then(base) after each batch of 8 * THREADS columns
    template <typename F, typename G> __device__ __forceinline__ void each(uint32_t first, uint32_t last, F &&f, G &&then) const
    {
        const uint64_t begin = (uint64_t)first * a.span, end = (uint64_t)(last + 1) * a.span < a.cols ? (uint64_t)(last + 1) * a.span : a.cols;
        for (uint64_t base = begin; base < end; base += kSampleBatch * THREADS) {
            const float *from = x + base;
            float v[kSampleBatch];
            if (end - base >= kSampleBatch * THREADS) {
#pragma unroll
                for (uint32_t j = 0; j < kSampleBatch; j++) v[j] = (from + j * THREADS)[tid];
            } else {
                const uint32_t most = (uint32_t)(end - base);
#pragma unroll
                for (uint32_t j = 0; j < kSampleBatch; j++) v[j] = j * THREADS + tid < most ? (from + j * THREADS)[tid] : NAN;
            }
            // (the last batch of a part or of a short row is half a batch or less: 100 rows of 1000, top-p, 11.5 us instead of 13.5)
            if (base + (kSampleBatch / 2) * THREADS < end) {
#pragma unroll
                for (uint32_t j = 0; j < kSampleBatch; j++) f(v[j], (uint32_t)base + j * THREADS + tid, j);
            } else {
#pragma unroll
                for (uint32_t j = 0; j < kSampleBatch / 2; j++)
                    if (base + j * THREADS < end) f(v[j], (uint32_t)base + j * THREADS + tid, j);
            }
            then(base);
        }
    }
    template <typename F> __device__ __forceinline__ void each(uint32_t first, uint32_t last, F &&f) const
    {
        each(first, last, [&](float v, uint32_t i, uint32_t) { f(v, i); }, [](uint64_t) {});
    }

    __device__ __forceinline__ uint64_t block_sum(uint64_t v)
    {
        v = wave_sum_u64(v);
        __syncthreads();
        if (lane == 0) sh.wave64[wave] = v;
        __syncthreads();
        return lane_value(wave_running<16>(sh.wave64[lane % 16u]), 15);
    }

    // of parts first .. last, in thread 0
    __device__ __forceinline__ SampleEnds ends(uint32_t first, uint32_t last)
    {
        SampleEnds e = {0, 0};
        each(first, last, [&](float v, uint32_t i) {
            const uint64_t key = sample_key(v, i);
            e.key = key > e.key ? key : e.key;
            e.low = v > -INFINITY ? max(e.low, ~(uint32_t)(key >> 32)) : e.low;
        });
        e.key = wave_most_u64(e.key);
        e.low = wave_most_u32(e.low);
        if (lane == 0) {
            sh.wave64[wave] = e.key;
            sh.wave32[wave] = e.low;
        }
        __syncthreads();
        if (wave == 0) e = SampleEnds{wave_most_u64(sh.wave64[lane % 16u]), wave_most_u32(sh.wave32[lane % 16u])};
        return e;
    }

    // SampleRules::power: the exponential's series up to the twelfth power, |x| <= ln 2 / 2 (seen after the workgroup's next barrier)
    __device__ __forceinline__ void fill_power()
    {
        if (tid >= 64u) return;
        const bool upper = tid >= 32u;
        const double x = (upper ? (double)(int)tid - 64.0 : (double)tid) * (0.6931471805599453 / 64.0);
        double e = 1.0;
#pragma unroll
        for (int i = 12; i > 0; i--) e = fma(e, x * (1.0 / (double)i), 1.0);
        sh.power[tid] = ldexp(e, a.s + upper);
    }

    __device__ __forceinline__ void clear_bins()
    {
        for (uint32_t b = tid; b < kSampleBins; b += THREADS) {
            sh.bins.mass[b] = 0;
            sh.bins.count[b] = 0;
        }
        __syncthreads();
    }

    // Tokens per bin for top-k, weights per bin for top-p
    __device__ __forceinline__ void histogram(const SampleRules &r, uint32_t first, uint32_t last)
    {
        if (r.counted()) {
            // (of those that may have no weight, at the end of the order, too: that they take no place among top_k makes no difference)
            each(first, last, [&](float v, uint32_t) {
                if (r.depth(v) <= r.deepest) atomicAdd(&sh.bins.count[r.bin(v)], 1u);
            });
            return;
        }
        each(first, last, [&](float v, uint32_t) {
            bool above;
            const uint64_t whole = r.weight(v, above);
            if (whole) {
                const uint32_t b = r.bin(v);
                if (r.top_k) atomicAdd(&sh.bins.count[b], 1u);
                if (r.top_p < 1.0) atomicAdd((unsigned long long *)&sh.bins.mass[b], (unsigned long long)whole);
            }
        });
    }

    // f(bin, tokens before it, in it, weights before it, in it) for the bins with tokens, and the sums over all
    struct Running {
        uint32_t count, all_count;
        uint64_t mass, all_mass;   // count, mass: before this thread's bins
    };
    static constexpr uint32_t kEach = kSampleBins / THREADS;
    __device__ __forceinline__ Running running()
    {
        uint32_t count = 0;
        uint64_t mass = 0;
#pragma unroll
        for (uint32_t j = 0; j < kEach; j++) {
            count += sh.bins.count[tid * kEach + j];
            mass += sh.bins.mass[tid * kEach + j];
        }
        const uint32_t run_count = wave_running(count);
        const uint64_t run_mass = wave_running(mass);
        if (lane == 63u) {
            sh.wave32[wave] = run_count;
            sh.wave64[wave] = run_mass;
        }
        __syncthreads();
        const uint32_t in_wave = sh.wave32[lane % 16u], waves = wave_running<16>(in_wave);
        const uint64_t mass_in_wave = sh.wave64[lane % 16u], mass_waves = wave_running<16>(mass_in_wave);
        return {run_count - count + (uint32_t)__builtin_amdgcn_readlane(waves - in_wave, wave), (uint32_t)__builtin_amdgcn_readlane(waves, 15),
                run_mass - mass + lane_value(mass_waves - mass_in_wave, (int)wave), lane_value(mass_waves, 15)};
    }
    template <typename F> __device__ __forceinline__ void each_bin(const Running &all, F &&f)
    {
        uint32_t c0 = all.count;
        uint64_t m0 = all.mass;
#pragma unroll
        for (uint32_t j = 0; j < kEach; j++) {
            const uint32_t b = tid * kEach + j, c = sh.bins.count[b];
            const uint64_t m = sh.bins.mass[b];
            if (c || m) f(b, c0, c, m0, m);
            c0 += c;
            m0 += m;
        }
    }

    // sh.cut from the whole row's histogram in sh.bins
    __device__ __forceinline__ void find_cut(const SampleRules &r)
    {
        if (tid == 0) sh.cut = SampleCut{kNoBin, kNoBin, kNoBin, 0, 0, 0, 0};
        const Running all = running();
        const bool by_k = r.top_k != 0 && r.top_k < all.all_count;
        if (!by_k && tid == 0) sh.cut.mass_k = all.all_mass;
        if (by_k)
            each_bin(all, [&](uint32_t b, uint32_t c0, uint32_t c, uint64_t m0, uint64_t m) {
                if (c0 < r.top_k && c0 + c >= r.top_k) {
                    sh.cut.k_bin = b;
                    sh.cut.above_k = c0;
                    sh.cut.mass_k = m0;
                    sh.taken_mass = m0 + m;
                }
            });
        __syncthreads();
        if (r.top_p < 1.0 && r.counted()) {
            if (tid == 0) {
                sh.cut.all = 1;
                sh.cut.p_first = 0;
                sh.cut.p_last = by_k ? sh.cut.k_bin : kSampleBins - 1u;
            }
        } else if (r.top_p < 1.0) {
            const double low = goal(r.top_p, sh.cut.mass_k), high = goal(r.top_p, by_k ? sh.taken_mass : all.all_mass);
            each_bin(all, [&](uint32_t b, uint32_t, uint32_t, uint64_t m0, uint64_t m) {
                if ((double)m0 < low && (double)(m0 + m) >= low) {
                    sh.cut.p_first = b;
                    sh.cut.mass_p = m0;
                }
                if ((double)m0 < high && (double)(m0 + m) >= high) sh.cut.p_last = b;
            });
        }
        __syncthreads();
    }

    // the sum before which a token has to begin to remain (the first one always does)
    static __device__ __forceinline__ double goal(double top_p, uint64_t mass)
    {
        const double g = top_p * (double)mass;
        return g > 0.5 ? g : 0.5;
    }

    // Adds the weights of parts first .. last that are in for certain to sh.spans, and lists the tokens of the bins that are not
    // settled; sh.listed counts on past the end of a full list.  (Both are clear and the workgroup has seen that.)
    __device__ __forceinline__ void gather(const SampleRules &r, const SampleCut &cut, uint32_t first, uint32_t last)
    {
        // (a token that is neither in for certain nor out is looked at again below, where its bin is settled)
        const float sure = SampleRules::begin(cut.sure()), end = fminf(SampleRules::begin(cut.behind()), r.deepest + 1.0f);
        // (a part is half a batch long or whole batches)
        uint64_t sum[2] = {0, 0};
        uint32_t pending = 0;   // those of a thread's batch that are to be listed: seldom more than one, and not worth eight tries a wave
        each(
            first, last,
            [&](float v, uint32_t i, uint32_t j) {
                const float depth = r.depth(v);
                pending |= depth >= sure && depth < end ? 1u << j : 0u;
                if (depth < sure) sum[j * 2 / kSampleBatch] += r.kept(v);
            },
            [&](uint64_t base) {
                while (pending) {
                    const uint32_t i = (uint32_t)base + (uint32_t)__builtin_ctz(pending) * THREADS + tid;
                    pending &= pending - 1u;
                    const float v = x[i];
                    bool above;
                    const uint64_t whole = r.weight(v, above);
                    if (whole == 0 || !cut.listed(r.bin(v))) continue;
                    const uint32_t at = atomicAdd(&sh.listed, 1u);
                    if (at < kSampleList) {
                        sh.list.key[at] = sample_key(v, i);
                        sh.list.mass[at] = whole | (above ? 1ull << 63 : 0ull);
                    }
                }
#pragma unroll
                for (uint32_t h = 0; h < 2; h++) {
                    const uint64_t half = wave_sum_u64(sum[h]);
                    if (lane == 0 && half) atomicAdd((unsigned long long *)&sh.spans[(uint32_t)(base + h * (kSampleBatch / 2 * THREADS)) / a.span], (unsigned long long)half);
                    sum[h] = 0;
                }
            });
    }

    // Of the listed tokens with keys of at least `least` in bins first .. last, the lowest key that remains: of the first `want` in the
    // row (by_mass false) or of those before which less than `end` lies, `count` tokens and `mass` weights being before them all.
    // The range of their keys is cut into 2048 parts, and the part in which the end falls again, until it holds no more tokens than a
    // wave has lanes (once, but for equal logits); those are compared with each other.
    __device__ __forceinline__ uint64_t narrow(const SampleRules &r, uint32_t n, uint32_t first, uint32_t last, uint64_t least, bool by_mass, uint64_t want,
                                               double end, uint64_t count, uint64_t mass)
    {
        auto bin_of = [&](uint64_t key) { return r.bin(sample_value((uint32_t)(key >> 32))); };
        if (tid == 0) {
            sh.low = ~0ull;
            sh.high = 0;
        }
        __syncthreads();
        uint64_t low = ~0ull, high = 0;
        for (uint32_t i = tid; i < n; i += THREADS) {
            const uint64_t key = sh.list.key[i];
            const uint32_t b = bin_of(key);
            if (key < least || b < first || b > last) continue;
            low = key < low ? key : low;
            high = key > high ? key : high;
        }
        low = ~wave_most_u64(~low);
        high = wave_most_u64(high);
        if (lane == 0 && high) {
            atomicMin((unsigned long long *)&sh.low, (unsigned long long)low);
            atomicMax((unsigned long long *)&sh.high, (unsigned long long)high);
        }
        __syncthreads();
        low = sh.low;
        high = sh.high;
        uint32_t held = n;
        while (low < high && held > 64u) {
            const int bits = 64 - __clzll((long long)(high - low)), shift = bits > 11 ? bits - 11 : 0;
            clear_bins();
            for (uint32_t i = tid; i < n; i += THREADS) {
                const uint64_t key = sh.list.key[i];
                if (key < low || key > high) continue;   // (between them every listed key is one of the bins first .. last)
                const uint32_t b = (uint32_t)((high - key) >> shift);
                atomicAdd(&sh.bins.count[b], 1u);
                atomicAdd((unsigned long long *)&sh.bins.mass[b], (unsigned long long)(sh.list.mass[i] & ~(1ull << 63)));
            }
            if (tid == 0) sh.stop = 0;   // (nothing ends here: every one of them remains)
            __syncthreads();
            each_bin(running(), [&](uint32_t b, uint32_t c0, uint32_t c, uint64_t m0, uint64_t m) {
                const bool here = by_mass ? (double)(mass + m0) < end && (double)(mass + m0 + m) >= end : count + c0 < want && count + c0 + c >= want;
                if (!here) return;
                const uint64_t top = high - ((uint64_t)b << shift), part = (1ull << shift) - 1u;
                sh.high = top;
                sh.low = top - low > part ? top - part : low;
                sh.taken_count = (uint32_t)(count + c0);
                sh.taken_mass = mass + m0;
                sh.stop = c;
            });
            __syncthreads();
            held = sh.stop;
            if (held) {
                low = sh.low;
                high = sh.high;
                count = sh.taken_count;
                mass = sh.taken_mass;
            }
            __syncthreads();
        }
        if (low >= high || held == 0) return low;
        if (tid < 64u) {
            sh.few_count[tid] = 0;
            sh.few_before[tid] = 0;
        }
        if (tid == 0) sh.taken_count = 0;
        __syncthreads();
        for (uint32_t i = tid; i < n; i += THREADS) {
            const uint64_t key = sh.list.key[i];
            if (key < low || key > high) continue;
            const uint32_t at = atomicAdd(&sh.taken_count, 1u);
            sh.few_key[at] = key;
            sh.few_mass[at] = sh.list.mass[i] & ~(1ull << 63);
        }
        __syncthreads();
        const uint64_t key = lane < held ? sh.few_key[lane] : 0ull;
        held = sh.taken_count;   // (at most the 64 there is room for)
        // a lane each, compared with a sixteenth of them by each wave
        uint32_t ahead = 0;
        uint64_t mass_ahead = 0;
        for (uint32_t j = wave; j < held; j += kWaves) {
            const bool before = sh.few_key[j] > key;
            ahead += before;
            mass_ahead += before ? sh.few_mass[j] : 0ull;
        }
        if (lane < held && ahead) {
            atomicAdd(&sh.few_count[lane], ahead);
            atomicAdd((unsigned long long *)&sh.few_before[lane], (unsigned long long)mass_ahead);
        }
        __syncthreads();
        count += sh.few_count[lane];
        mass += sh.few_before[lane];
        const bool in = lane < held && (by_mass ? (double)mass < end : count < want);
        return ~wave_most_u64(in ? ~key : 0ull);
    }

    // Settles the listed tokens: adds the weights of those that remain to sh.spans, returns their lowest key (none: all ones)
    __device__ __forceinline__ uint64_t settle(const SampleRules &r, const SampleCut &cut, uint32_t n)
    {
        uint64_t least = 0;
        if (n == 0) return ~0ull;
        if (cut.k_bin != kNoBin) least = narrow(r, n, cut.k_bin, cut.k_bin, 0, false, r.top_k, 0.0, cut.above_k, cut.mass_k);
        // (where the first top_k end among tokens that were counted but have no weight, the listed ones are all within them)
        if (cut.all && least == ~0ull) least = 0;
        if (cut.p_first != kNoBin) {
            uint64_t in_k = 0;
            if (cut.k_bin != kNoBin || cut.all)
                for (uint32_t i = tid; i < n; i += THREADS) {
                    const uint64_t key = sh.list.key[i];
                    if (key >= least && (cut.all || r.bin(sample_value((uint32_t)(key >> 32))) == cut.k_bin)) in_k += sh.list.mass[i] & ~(1ull << 63);
                }
            in_k = block_sum(in_k);
            const uint64_t by_p = narrow(r, n, cut.p_first, cut.p_last, least, true, 0, goal(r.top_p, cut.mass_k + in_k), 0, cut.mass_p);
            least = by_p > least ? by_p : least;
        }
        for (uint32_t i = tid; i < n; i += THREADS) {
            const uint64_t key = sh.list.key[i], mass = sh.list.mass[i];
            if (key >= least && mass >> 63) atomicAdd((unsigned long long *)&sh.spans[(0xFFFFFFFFu - (uint32_t)key) / a.span], (unsigned long long)(mass & ~(1ull << 63)));
        }
        __syncthreads();
        return least;
    }

    // The lowest key that remains, eight bits at a time over the whole row: of the first `want` keys (by_mass false) or of those
    // before which less than `end` lies; keys below `least` do not take part.
    __device__ uint64_t select(const SampleRules &r, bool by_mass, uint64_t want, double end, uint64_t least)
    {
        __syncthreads();
        if (tid == 0) {
            sh.prefix = 0;
            sh.taken_count = 0;
            sh.taken_mass = 0;
        }
        for (int shift = 56; shift >= 0; shift -= 8) {
            for (uint32_t b = tid; b < 256; b += THREADS) {
                sh.bins.mass[b] = 0;
                sh.bins.count[b] = 0;
            }
            __syncthreads();
            const uint64_t prefix = sh.prefix;
            each(0, a.spans - 1u, [&](float v, uint32_t i) {
                    const uint64_t key = sample_key(v, i);
                    if (key < least || (shift < 56 && (key >> (shift + 8)) != prefix)) return;
                    bool above;
                    const uint64_t whole = r.weight(v, above);
                    if (whole == 0) return;
                    atomicAdd(&sh.bins.count[(key >> shift) & 255u], 1u);
                    atomicAdd((unsigned long long *)&sh.bins.mass[(key >> shift) & 255u], (unsigned long long)whole);
                });
            __syncthreads();
            if (tid == 0) {
                uint32_t last = 256;
                for (int b = 255; b >= 0; b--) {
                    if (sh.bins.count[b] == 0) continue;
                    if (last < 256) {
                        // whether the order goes on into this bin
                        const bool on = by_mass ? (double)(sh.taken_mass + sh.bins.mass[last]) < end : sh.taken_count + sh.bins.count[last] < want;
                        if (!on) break;
                        sh.taken_count += sh.bins.count[last];
                        sh.taken_mass += sh.bins.mass[last];
                    }
                    last = (uint32_t)b;
                }
                sh.prefix = prefix << 8 | last;
                // all of a bin's tokens are in, or it holds one: any key down to the bin's lowest will do
                sh.stop = by_mass ? sh.bins.count[last] == 1 : sh.taken_count + sh.bins.count[last] <= want;
            }
            __syncthreads();
            if (sh.stop) {
                const uint64_t found = sh.prefix << shift;
                __syncthreads();
                return found;
            }
        }
        const uint64_t found = sh.prefix;
        __syncthreads();
        return found;
    }

    // the weights that remain of the whole row, with the lowest key by select
    __device__ void settle_long(const SampleRules &r)
    {
        uint64_t least = 0;
        if (r.top_k) least = select(r, false, r.top_k, 0.0, 0);
        if (r.top_p < 1.0) {
            uint64_t sum = 0;
            each(0, a.spans - 1u, [&](float v, uint32_t i) {
                    bool above;
                    if (sample_key(v, i) >= least) sum += r.weight(v, above);
                });
            sum = block_sum(sum);
            const uint64_t by_p = select(r, true, 0, goal(r.top_p, sum), least);
            least = by_p > least ? by_p : least;
        }
        for (uint32_t span = 0; span < a.spans; span++) {
            uint64_t sum = 0;
            each(span, span, [&](float v, uint32_t i) {
                if (sample_key(v, i) >= least) sum += r.kept(v);
            });
            sum = block_sum(sum);
            if (tid == 0) sh.spans[span] = sum;
        }
        if (tid == 0) sh.least = least;
        __syncthreads();
    }

    // The token, from the parts' sums in sh.spans; in(v, i): whether the limits leave a token
    template <typename F> __device__ __forceinline__ void choose(const SampleRules &r, F &&in)
    {
        // (a lane per part)
        const uint64_t part = lane < a.spans ? sh.spans[lane] : 0, parts = wave_running(part), total = lane_value(parts, 63);
        const double u = r.uniform;
        // the first index at which the running sum is above u times the whole, below the whole for any u
        const double g = u > 0.0 ? u * (double)total : 0.0;
        const uint64_t end = g >= (double)total ? total - 1u : (uint64_t)g;
        const uint32_t span = (uint32_t)__builtin_ctzll(__ballot(parts > end));
        uint64_t before = lane_value(parts - part, (int)span);
        const uint64_t last = (uint64_t)(span + 1) * a.span < a.cols ? (uint64_t)(span + 1) * a.span : a.cols;
        // four neighbouring columns a thread
        for (uint64_t at = (uint64_t)span * a.span; at < last; at += 4u * THREADS) {
            uint64_t mine[4], sum = 0;
#pragma unroll
            for (uint32_t j = 0; j < 4; j++) {
                const uint64_t i = at + tid * 4u + j;
                mine[j] = 0;
                if (i < last) {
                    const float v = x[i];
                    if (in(v, (uint32_t)i)) {
                        mine[j] = r.kept(v);
                    }
                }
                sum += mine[j];
            }
            uint64_t run = wave_running(sum);
            __syncthreads();
            if (lane == 63u) sh.wave64[wave] = run;
            __syncthreads();
            const uint64_t in_wave = sh.wave64[lane % 16u], waves = wave_running<16>(in_wave);
            run += before + lane_value(waves - in_wave, (int)wave) - sum;
#pragma unroll
            for (uint32_t j = 0; j < 4; j++) {
                if (mine[j] && run <= end && run + mine[j] > end) a.out[row] = (int)(at + tid * 4u + j);
                run += mine[j];
            }
            before += lane_value(waves, 15);
            if (before > end) break;
        }
    }

    // from sh.list (n tokens found) and sh.spans to the token
    __device__ __forceinline__ void finish(const SampleRules &r, const SampleCut &cut, uint32_t n)
    {
        if (n > kSampleList) {
            settle_long(r);
            const uint64_t least = sh.least;
            choose(r, [=](float v, uint32_t i) { return sample_key(v, i) >= least; });
            return;
        }
        const uint64_t least = settle(r, cut, n);
        const uint32_t sure = cut.sure();
        choose(r, [=](float v, uint32_t i) { return r.bin(v) < sure || sample_key(v, i) >= least; });
    }
};

// whether a row's largest key is of a token that can be chosen
__device__ __forceinline__ bool sample_any(uint64_t key) { return (uint32_t)(key >> 32) > sample_order(-INFINITY); }
__device__ __forceinline__ int sample_index(uint64_t key) { return (int)(0xFFFFFFFFu - (uint32_t)key); }

}  // namespace

// A workgroup per row.  WAVES 8: so few registers (64; eight values of a lane are spilled, 20 bytes at a time) that a compute unit holds
// two workgroups
template <int WAVES> __global__ __launch_bounds__(1024, WAVES) void k_sample(const SampleArgs a)
{
    __shared__ SampleShared sh;
    Sampler<1024> s(a, sh, blockIdx.x);
    s.fill_power();
    if (s.tid < kSampleSpans) sh.spans[s.tid] = 0;
    const SampleEnds ends = s.ends(0, a.spans - 1u);
    if (s.tid == 0) {
        sh.ends = ends;
        sh.listed = 0;
    }
    __syncthreads();
    const uint64_t key = sh.ends.key;
    const SampleRules r = sample_rules(a, sh.power, s.row, sh.ends);
    if (!sample_any(key) || r.greedy) {
        if (s.tid == 0) a.out[s.row] = sample_any(key) ? sample_index(key) : 0;
        return;
    }
    SampleCut cut = {kNoBin, kNoBin, kNoBin, 0, 0, 0, 0};
    if (r.limited()) {
        s.clear_bins();
        s.histogram(r, 0, a.spans - 1u);
        __syncthreads();
        s.find_cut(r);
        cut = sh.cut;
    }
    s.gather(r, cut, 0, a.spans - 1u);
    __syncthreads();
    s.finish(r, cut, sh.listed);
}

// ---- few rows: a workgroup per part of a row ------------------------------------------------------------------------------

namespace {

template <typename V> __device__ __forceinline__ void leave(V *to, V v) { __hip_atomic_store(to, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
template <typename V> __device__ __forceinline__ V left(const V *from) { return __hip_atomic_load(from, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

// The parts that workgroup x of a row takes
__device__ __forceinline__ uint32_t first_part(const SampleArgs &a) { return blockIdx.x * a.each; }
__device__ __forceinline__ uint32_t last_part(const SampleArgs &a) { return min(blockIdx.x * a.each + a.each, a.spans) - 1u; }

// Whether this workgroup is the row's last to arrive, what all of them left being in memory then; the counter is zero again after
__device__ __forceinline__ bool last_to_arrive(SampleShared &sh, unsigned *counter)
{
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (threadIdx.x == 0) {
        const bool last = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == gridDim.x - 1u;
        if (last) leave(counter, 0u);
        sh.stop = last;
    }
    __syncthreads();
    return sh.stop != 0;
}

// the row's ends, from its workgroups' (of the launch before)
__device__ __forceinline__ SampleEnds row_ends(const SampleRow &state, uint32_t groups)
{
    const uint32_t lane = threadIdx.x & 63u;
    return SampleEnds{wave_most_u64(lane < groups ? state.key[lane] : 0), wave_most_u32(lane < groups ? state.low[lane] : 0u)};
}

}  // namespace

__global__ __launch_bounds__(1024) void k_sample_largest(const SampleArgs a, SampleRow *__restrict__ rows)
{
    __shared__ SampleShared sh;
    Sampler<1024> s(a, sh, blockIdx.y);
    SampleRow &state = rows[blockIdx.y];
    for (uint32_t b = blockIdx.x * 1024u + s.tid; b < kSampleBins; b += gridDim.x * 1024u) {
        state.bin_mass[b] = 0;
        state.bin_count[b] = 0;
    }
    const SampleEnds ends = s.ends(first_part(a), last_part(a));
    if (s.tid == 0) {
        state.key[blockIdx.x] = ends.key;
        state.low[blockIdx.x] = ends.low;
        if (blockIdx.x == 0) state.listed = 0;
    }
}

__global__ __launch_bounds__(1024) void k_sample_limits(const SampleArgs a, SampleRow *__restrict__ rows, unsigned *__restrict__ counters)
{
    __shared__ SampleShared sh;
    Sampler<1024> s(a, sh, blockIdx.y);
    SampleRow &state = rows[blockIdx.y];
    const SampleEnds ends = row_ends(state, gridDim.x);
    const uint64_t key = ends.key;
    const SampleRules r = sample_rules(a, sh.power, s.row, ends);
    if (!sample_any(key) || r.greedy || !r.limited()) return;
    s.fill_power();
    s.clear_bins();
    s.histogram(r, first_part(a), last_part(a));
    __syncthreads();
    for (uint32_t b = s.tid; b < kSampleBins; b += 1024u) {
        if (sh.bins.count[b]) __hip_atomic_fetch_add(&state.bin_count[b], sh.bins.count[b], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        if (sh.bins.mass[b]) __hip_atomic_fetch_add(&state.bin_mass[b], sh.bins.mass[b], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    if (!last_to_arrive(sh, &counters[s.row * kSampleCounterStep])) return;
    for (uint32_t b = s.tid; b < kSampleBins; b += 1024u) {
        sh.bins.count[b] = left(&state.bin_count[b]);
        sh.bins.mass[b] = left(&state.bin_mass[b]);
    }
    __syncthreads();
    s.find_cut(r);
    if (s.tid == 0) state.cut = sh.cut;
}

__global__ __launch_bounds__(1024) void k_sample_token(const SampleArgs a, SampleRow *__restrict__ rows, unsigned *__restrict__ counters)
{
    __shared__ SampleShared sh;
    Sampler<1024> s(a, sh, blockIdx.y);
    SampleRow &state = rows[blockIdx.y];
    const SampleEnds ends = row_ends(state, gridDim.x);
    const uint64_t key = ends.key;
    const SampleRules r = sample_rules(a, sh.power, s.row, ends);
    if (!sample_any(key) || r.greedy) {
        if (blockIdx.x == 0 && s.tid == 0) a.out[s.row] = sample_any(key) ? sample_index(key) : 0;
        return;
    }
    SampleCut cut = {kNoBin, kNoBin, kNoBin, 0, 0, 0, 0};
    if (r.limited()) cut = state.cut;
    s.fill_power();
    if (s.tid < kSampleSpans) sh.spans[s.tid] = 0;
    if (s.tid == 0) sh.listed = 0;
    __syncthreads();
    s.gather(r, cut, first_part(a), last_part(a));
    __syncthreads();
    const uint32_t mine = sh.listed, there = mine < kSampleList ? mine : kSampleList;
    if (s.tid >= first_part(a) && s.tid <= last_part(a)) leave(&state.mass[s.tid], sh.spans[s.tid]);
    if (s.tid == 0) {
        sh.base = mine ? __hip_atomic_fetch_add(&state.listed, mine, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : 0u;
    }
    __syncthreads();
    for (uint32_t i = s.tid; i < there; i += 1024u) {
        const uint32_t at = sh.base + i;
        if (at < kSampleList) {
            leave(&state.list_key[at], sh.list.key[i]);
            leave(&state.list_mass[at], sh.list.mass[i]);
        }
    }
    if (!last_to_arrive(sh, &counters[s.row * kSampleCounterStep])) return;
    const uint32_t n = left(&state.listed);
    for (uint32_t i = s.tid; i < n && i < kSampleList; i += 1024u) {
        sh.list.key[i] = left(&state.list_key[i]);
        sh.list.mass[i] = left(&state.list_mass[i]);
    }
    if (s.tid < a.spans) sh.spans[s.tid] = left(&state.mass[s.tid]);
    __syncthreads();
    s.finish(r, cut, n);
}

// S: the largest for which 2^S times `cols` stays below 2^63 (51 at most: see weight)
static int sample_bits(uint32_t cols)
{
    int bits = 0;
    while (bits < 32 && (1ull << bits) < cols) bits++;
    return 62 - bits < 51 ? 62 - bits : 51;
}

hipError_t launch_sample(hipStream_t s, const float *logits, uint32_t rows, uint32_t cols, const float *uniform, const float *temperature,
                         const int *top_k, const float *top_p, const float *min_p, int *out, void *scratch, size_t scratch_bytes,
                         unsigned *counters, uint32_t n_counters)
{
    if (rows == 0) return hipSuccess;
    // parts of 4096 columns, longer ones where there would be too many
    uint32_t span = (uint32_t)(((uint64_t)cols + kSampleSpans - 1) / kSampleSpans);
    span = span <= kSamplePart ? kSamplePart : (span + 2 * kSamplePart - 1) / (2 * kSamplePart) * (2 * kSamplePart);
    const uint32_t spans = cols ? (cols + span - 1) / span : 1u;
    SampleArgs a = {logits, uniform, temperature, top_p, min_p, top_k, out, cols, spans, span, spans, sample_bits(cols)};
    // A workgroup per row takes 15 us and 0.72 for each 1000 columns, several of them 22 us and 0.85 for each 1000 columns that one of
    // them works through (measured at 1 to 250 rows of 8000 to 152064 columns, top-p: 128 rows of 60000 59 us and 50, 66 of 20000 28
    // either way, 20 of 10000 20 and 24).
    const uint32_t most_groups = rows < kSampleGroups ? kSampleGroups / rows : 1u, each = (spans + most_groups - 1) / most_groups;
    if (5ull * cols > 50000ull + 6ull * each * span && scratch && counters && (uint64_t)rows * kSampleCounterStep <= n_counters &&
        (uint64_t)rows * sizeof(SampleRow) <= scratch_bytes) {
        a.each = each;
        const uint32_t groups = (spans + a.each - 1) / a.each;
        SampleRow *state = (SampleRow *)scratch;
        hipLaunchKernelGGL(k_sample_largest, dim3(groups, rows), dim3(1024), 0, s, a, state);
        hipError_t e = hipGetLastError();
        if (e == hipSuccess && (top_k || top_p)) {
            hipLaunchKernelGGL(k_sample_limits, dim3(groups, rows), dim3(1024), 0, s, a, state, counters);
            e = hipGetLastError();
        }
        if (e != hipSuccess) return e;
        hipLaunchKernelGGL(k_sample_token, dim3(groups, rows), dim3(1024), 0, s, a, state, counters);
        return hipGetLastError();
    }
    // two workgroups a compute unit where there are more rows than those: 4096 rows of 1000 119 us instead of 177, 512 of 32000 65 instead
    // of 74; up to as many rows the registers count, 256 of 32000 39.9 instead of 41.1
    return in_slices(rows, most_workgroups(1024), [&](uint32_t row, uint32_t here) {
        SampleArgs part = a;
        part.logits = logits + (size_t)row * cols;
        part.uniform = uniform + row;
        part.temperature = temperature ? temperature + row : nullptr;
        part.top_k = top_k ? top_k + row : nullptr;
        part.top_p = top_p ? top_p + row : nullptr;
        part.min_p = min_p ? min_p + row : nullptr;
        part.out = out + row;
        hipLaunchKernelGGL(rows <= kSampleGroups ? k_sample<4> : k_sample<8>, dim3(here), dim3(1024), 0, s, part);
        return hipGetLastError();
    });
}

}  // namespace twm
