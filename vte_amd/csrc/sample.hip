// Drawing the next tokens on the device: temperature, top-k, top-p, min-p and
// the draw from given uniforms, per row of fp32 logits, gfx950.
//
// Semantics (the host sampler's of vte/core/sampler.py:54-129, with min-p
// behind top-p): weights w_i = exp((x_i - max) / T); order by (value
// descending, index ascending); top-k keeps the first k, top-p those with at
// most top_p * (mass of the top-k) before them, min-p those with w_i >= min_p;
// the token is the first of the kept whose mass up to and with it exceeds u *
// (kept mass).  T <= 0: the first of all.  Every filter keeps a prefix of the
// order.
//
// Weights are whole numbers, round(w * 2^44) in 64 bits (a row of 2^18 stays
// below 2^63): sums are exact in any order, so the token does not depend on
// how the row is cut or on the order of atomics.  An entry below 2^-45 of the
// largest has no weight.
#include "vte_common.h"

#define SMP_THREADS 1024
#define SMP_IDX_BITS 18
#define SMP_DIGIT 10
#define SMP_LEVELS 5  // 32 + 18 bits of (key, index) in digits of 10

struct SmpRow {
    const float* x;
    int n;
    float max;
    double inv_t, min_w;
    uint64_t floor_c;  // entries ordered behind this one are out
};

// Order-preserving key: larger value, larger key; NaN below everything.
__device__ __forceinline__ uint32_t smp_key(float x) {
    if (x != x) return 0u;
    const uint32_t u = __float_as_uint(x == 0.f ? 0.f : x);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
// Place of an entry in the order, as one number: larger comes first.
__device__ __forceinline__ uint64_t smp_place(uint32_t key, int i) {
    return ((uint64_t)key << SMP_IDX_BITS) | (uint64_t)(((1 << SMP_IDX_BITS) - 1) - i);
}
__device__ __forceinline__ double smp_weight(const SmpRow& r, float x) {
    if (x == r.max) return 1.0;
    return x > -INFINITY ? exp(((double)x - (double)r.max) * r.inv_t) : 0.0;  // NaN: 0
}
__device__ __forceinline__ uint64_t smp_mass(double w) { return (uint64_t)rint(w * 17592186044416.0); }

// First entry in the order at which the running sum (of 1 per entry, or of
// masses) exceeds `target`, among the entries still in; its place, and the sum
// of masses up to and with it.  Returns 0 if the sum never exceeds it (then
// `mass` is the sum of all).  Digit by digit over the places, all threads.
__device__ uint64_t smp_select(const SmpRow& r, bool count, uint64_t target, uint64_t& mass, uint64_t* sums,
                               uint64_t* masses, uint64_t* sh) {
    uint64_t prefix = 0, above_sum = 0, above_mass = 0;
    for (int level = 0; level < SMP_LEVELS; ++level) {
        const int shift = (SMP_LEVELS - 1 - level) * SMP_DIGIT;
        __syncthreads();
        sums[threadIdx.x] = 0;
        masses[threadIdx.x] = 0;
        __syncthreads();
        for (int i = threadIdx.x; i < r.n; i += SMP_THREADS) {
            const float x = r.x[i];
            const uint64_t c = smp_place(smp_key(x), i);
            if (c < r.floor_c || (level > 0 && (c >> (shift + SMP_DIGIT)) != prefix)) continue;
            const double w = smp_weight(r, x);
            if (w < r.min_w) continue;
            const uint64_t m = smp_mass(w);
            const int d = (int)(c >> shift) & ((1 << SMP_DIGIT) - 1);
            atomicAdd((unsigned long long*)&masses[d], (unsigned long long)m);
            if (count) atomicAdd((unsigned long long*)&sums[d], 1ull);
        }
        __syncthreads();
        if (threadIdx.x == 0) {
            const uint64_t* by = count ? sums : masses;
            int d = (1 << SMP_DIGIT) - 1;
            for (; d >= 0; --d) {
                if (above_sum + by[d] > target) break;
                above_sum += by[d];
                above_mass += masses[d];
            }
            sh[0] = (uint64_t)(int64_t)d;
            sh[1] = above_sum;
            sh[2] = above_mass;
            sh[3] = d >= 0 ? masses[d] : 0;
        }
        __syncthreads();
        above_sum = sh[1];
        above_mass = sh[2];
        mass = above_mass + sh[3];
        if ((int64_t)sh[0] < 0) return 0;
        prefix = (prefix << SMP_DIGIT) | sh[0];
    }
    return prefix;
}

__global__ __launch_bounds__(SMP_THREADS) void sample_kernel(const float* __restrict__ logits, int vocab,
                                                             const float* __restrict__ temperature,
                                                             const int* __restrict__ top_k,
                                                             const float* __restrict__ top_p,
                                                             const float* __restrict__ min_p,
                                                             const double* __restrict__ u, int* __restrict__ tokens) {
    __shared__ uint64_t sums[SMP_THREADS], masses[SMP_THREADS], sh[4];
    const int row = blockIdx.x, tid = threadIdx.x;
    SmpRow r;
    r.x = logits + (size_t)row * vocab;
    r.n = vocab;
    uint64_t best = 0;
    for (int i = tid; i < vocab; i += SMP_THREADS) best = max(best, smp_place(smp_key(r.x[i]), i));
    sums[tid] = best;
    __syncthreads();
    for (int s = SMP_THREADS / 2; s > 0; s >>= 1) {
        if (tid < s) sums[tid] = max(sums[tid], sums[tid + s]);
        __syncthreads();
    }
    best = sums[0];
    const int first = ((1 << SMP_IDX_BITS) - 1) - (int)(best & ((1 << SMP_IDX_BITS) - 1));
    r.max = r.x[first];
    const float T = temperature ? temperature[row] : 1.f;
    if (!(r.max > -INFINITY) || !(T > 0.f)) {  // nothing to draw from; greedy
        if (tid == 0) tokens[row] = r.max > -INFINITY ? first : -1;
        return;
    }
    r.inv_t = 1.0 / (double)T;
    r.min_w = 0.0;
    r.floor_c = 0;
    uint64_t mass = 0;
    const int k = top_k ? top_k[row] : 0;
    r.floor_c = smp_select(r, true, k > 0 ? (uint64_t)(k - 1) : ~0ull, mass, sums, masses, sh);
    const double p = top_p ? (double)top_p[row] : 1.0;
    if (p > 0.0 && p < 1.0) {
        const uint64_t c = smp_select(r, false, (uint64_t)(p * (double)mass), mass, sums, masses, sh);
        r.floor_c = max(r.floor_c, c);
    }
    const double mp = min_p ? (double)min_p[row] : 0.0;
    if (mp > 0.0) {
        r.min_w = fmin(mp, 1.0);
        smp_select(r, false, ~0ull, mass, sums, masses, sh);
    }
    const double t = u[row] * (double)mass;
    const uint64_t target = t > 0.0 ? min((uint64_t)fmin(t, 9.2e18), mass - 1) : 0;
    const uint64_t c = smp_select(r, false, target, mass, sums, masses, sh);
    if (tid == 0) tokens[row] = ((1 << SMP_IDX_BITS) - 1) - (int)(c & ((1 << SMP_IDX_BITS) - 1));
}

namespace vte {
long long sample_scratch_bytes(int) { return 256; }
hipError_t sample(const float* logits, int rows, int vocab, const float* temperature, const int* top_k,
                  const float* top_p, const float* min_p, const double* u, int* tokens, void*, hipStream_t st) {
    hipLaunchKernelGGL(sample_kernel, dim3(rows), dim3(SMP_THREADS), 0, st, logits, vocab, temperature, top_k, top_p,
                       min_p, u, tokens);
    return hipGetLastError();
}
}  // namespace vte
