// One token per row of logits, from a uniform number that the caller gives: temperature, top-k, top-p and min-p.
//
//   w[i] = exp((x[i] - max x) / temperature), in 64 bits, kept as the whole number round(w * 2^S): sums of whole numbers do not
//   depend on their order, so that every way of sharing a row out gives the same token.  S is the largest that keeps the sum of
//   a row of that many columns below 2^63 (45 at 152064 columns); a token whose weight rounds to nothing (below 2^-46 of the
//   largest) is never chosen.
//   In descending order of x, equal ones by index, the first top_k tokens remain; of these the shortest run that holds top_p of
//   their sum (a token stays while the sum before it is below that); of these the tokens with w >= min_p.  Each rule keeps a
//   prefix of the order, so what remains is the tokens whose key -- the bits of x that order as x does, then the inverted
//   index -- is at least one 64-bit number, and with w >= min_p.
//   The token is the first by index at which the running sum of what remains exceeds u times the whole.
#include "twm_device.h"

namespace twm {

namespace {

constexpr uint32_t kSampleThreads = 1024;

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

struct RowRules {
    double largest, temperature, top_p, min_p, scale;
    uint64_t top_k;
    bool greedy;
};

// 2^S w of one logit
__device__ __forceinline__ uint64_t sample_weight(const RowRules &r, float x, double &w)
{
    const double v = x;
    w = v == r.largest ? 1.0 : v < r.largest && x > -INFINITY ? exp((v - r.largest) / r.temperature) : 0.0;
    return (uint64_t)rint(w * r.scale);
}

struct SampleShared {
    uint64_t mass[256];
    uint32_t count[256];
    uint64_t wave64[kSampleThreads / 64];
    uint64_t prefix, taken_count, taken_mass;
    uint32_t largest, stop;
};

__device__ __forceinline__ uint64_t wave_sum_u64(uint64_t v)
{
#pragma unroll
    for (int step = 32; step; step >>= 1) v += __shfl_xor(v, step);
    return v;
}

// the sum over the workgroup, in every thread
__device__ uint64_t block_sum_u64(SampleShared &sh, uint64_t v)
{
    v = wave_sum_u64(v);
    __syncthreads();
    if ((threadIdx.x & 63u) == 0) sh.wave64[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0;
    for (uint32_t w = 0; w < kSampleThreads / 64; w++) v += sh.wave64[w];
    return v;
}

}  // namespace

__global__ __launch_bounds__(1024) void k_sample(const float *__restrict__ logits, uint32_t cols, const float *__restrict__ uniform,
                                                 const float *__restrict__ temperature, const int *__restrict__ top_k,
                                                 const float *__restrict__ top_p, const float *__restrict__ min_p, double scale, int *__restrict__ out)
{
    __shared__ SampleShared sh;
    const uint32_t row = blockIdx.x, tid = threadIdx.x;
    const float *x = logits + (size_t)row * cols;
    if (tid == 0) sh.largest = 0;
    __syncthreads();
    uint32_t most = 0;
    for (uint64_t i = tid; i < cols; i += kSampleThreads) most = max(most, sample_order(x[i]));
    atomicMax(&sh.largest, most);
    __syncthreads();
    most = sh.largest;
    if (most <= sample_order(-INFINITY)) {   // nothing but -infinity and NaN
        if (tid == 0) out[row] = 0;
        return;
    }
    RowRules r;
    r.largest = sample_value(most);
    const float t = temperature ? temperature[row] : 1.0f;
    r.greedy = !(t > 0.0f);
    r.temperature = t;
    r.scale = scale;
    const int k = top_k ? top_k[row] : 0;
    r.top_k = r.greedy ? 1u : k > 0 ? (uint64_t)k : ~0ull;
    const float p = top_p ? top_p[row] : 1.0f;
    r.top_p = p != p ? 1.0 : p;
    const float mp = min_p ? min_p[row] : 0.0f;
    r.min_p = mp != mp ? 0.0 : mp > 1.0f ? 1.0 : mp;
    if (r.greedy) r.temperature = 1.0;

    auto key_of = [&](uint64_t i, float v) { return (uint64_t)sample_order(v) << 32 | (0xFFFFFFFFu - (uint32_t)i); };

    // the smallest key among the first `want` of the order (by_mass false) or among those before which less than `goal` lies;
    // keys below `least` do not take part
    auto select = [&](bool by_mass, uint64_t want, double goal, uint64_t least) -> uint64_t {
        if (tid == 0) {
            sh.prefix = 0;
            sh.taken_count = 0;
            sh.taken_mass = 0;
        }
        for (int shift = 56; shift >= 0; shift -= 8) {
            if (tid < 256) {
                sh.mass[tid] = 0;
                sh.count[tid] = 0;
            }
            __syncthreads();
            const uint64_t prefix = sh.prefix;
            for (uint64_t i = tid; i < cols; i += kSampleThreads) {
                const float v = x[i];
                const uint64_t key = key_of(i, v);
                if (key < least || (shift < 56 && (key >> (shift + 8)) != prefix)) continue;
                double w;
                const uint64_t whole = sample_weight(r, v, w);
                if (whole == 0) continue;
                atomicAdd(&sh.count[(key >> shift) & 255u], 1u);
                atomicAdd((unsigned long long *)&sh.mass[(key >> shift) & 255u], (unsigned long long)whole);
            }
            __syncthreads();
            if (tid == 0) {
                uint32_t last = 256;
                for (int b = 255; b >= 0; b--) {
                    if (sh.count[b] == 0) continue;
                    if (last < 256) {
                        // whether the order goes on into this bin
                        const bool on = by_mass ? (double)(sh.taken_mass + sh.mass[last]) < goal : sh.taken_count + sh.count[last] < want;
                        if (!on) break;
                        sh.taken_count += sh.count[last];
                        sh.taken_mass += sh.mass[last];
                    }
                    last = (uint32_t)b;
                }
                sh.prefix = prefix << 8 | last;
                // all of a bin's tokens are in, or it holds one: any key down to the bin's lowest will do
                const bool whole_bin = by_mass ? sh.count[last] == 1 : sh.taken_count + sh.count[last] <= want;
                sh.stop = whole_bin;
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
    };

    uint64_t least = 0;
    if (r.top_k < cols) least = select(false, r.top_k, 0.0, 0);
    if (r.top_p < 1.0 && !r.greedy) {
        uint64_t sum = 0;
        for (uint64_t i = tid; i < cols; i += kSampleThreads) {
            const float v = x[i];
            double w;
            if (key_of(i, v) >= least) sum += sample_weight(r, v, w);
        }
        sum = block_sum_u64(sh, sum);
        const uint64_t by_p = select(true, 0, r.top_p * (double)sum, least);
        least = by_p > least ? by_p : least;
    }

    // what remains of one logit
    auto left = [&](uint64_t i) -> uint64_t {
        if (i >= cols) return 0;
        const float v = x[i];
        if (key_of(i, v) < least) return 0;
        double w;
        const uint64_t whole = sample_weight(r, v, w);
        return w >= r.min_p ? whole : 0;
    };
    uint64_t total = 0;
    for (uint64_t i = tid; i < cols; i += kSampleThreads) total += left(i);
    total = block_sum_u64(sh, total);
    const double u = uniform[row];
    // the first index at which the running sum is above `goal`: u times the whole, below the whole for any u
    double goal_f = u > 0.0 ? u * (double)total : 0.0;
    const uint64_t goal = goal_f >= (double)total ? total - 1u : (uint64_t)goal_f;
    uint64_t before = 0;
    for (uint64_t at = 0; at < cols; at += kSampleThreads) {
        const uint64_t mine = left(at + tid);
        uint64_t run = mine;   // sum up to and with this lane
#pragma unroll
        for (int step = 1; step < 64; step <<= 1) {
            const uint64_t other = __shfl_up(run, step);
            if ((tid & 63u) >= (uint32_t)step) run += other;
        }
        __syncthreads();
        if ((tid & 63u) == 63u) sh.wave64[tid >> 6] = run;
        __syncthreads();
        uint64_t tile = 0;
        for (uint32_t w = 0; w < kSampleThreads / 64; w++) {
            if (w == (tid >> 6)) run += before + tile;
            tile += sh.wave64[w];
        }
        if (mine && run > goal && run - mine <= goal) out[row] = (int)(at + tid);
        before += tile;
        if (before > goal) break;
    }
}

// 2^S: the largest power of two whose product with `cols` stays below 2^63 (and is a double's 52 bits at most)
static double sample_scale(uint32_t cols)
{
    int bits = 0;
    while (bits < 32 && (1ull << bits) < cols) bits++;
    const int s = 62 - bits < 52 ? 62 - bits : 52;
    return (double)(1ull << s);
}

hipError_t launch_sample(hipStream_t s, const float *logits, uint32_t rows, uint32_t cols, const float *uniform, const float *temperature,
                         const int *top_k, const float *top_p, const float *min_p, int *out)
{
    if (rows == 0) return hipSuccess;
    hipLaunchKernelGGL(k_sample, dim3(rows), dim3(kSampleThreads), 0, s, logits, cols, uniform, temperature, top_k, top_p, min_p, sample_scale(cols), out);
    return hipGetLastError();
}

}  // namespace twm
