// Drawing the next tokens on the device: temperature, top-k, top-p, min-p and
// the draw from given uniforms, per row of fp32 logits, gfx950.
//
// Semantics (the host sampler's of vte/core/sampler.py:54-129, with min-p
// behind top-p): weights w_i = exp(x_i / T); order by (value descending, index
// ascending); top-k keeps the first k, top-p those with at most top_p * (mass of
// the top-k) before them, min-p those with w_i >= min_p * (largest weight); the
// token is the first of the kept whose mass up to and with it exceeds u * (kept
// mass).  T <= 0: the first of all.  Every filter keeps a prefix of the order, so
// all that matters is at which mass each ends.
//
// The row is not sorted.  With y = 64 x / T, entries fall into bins floor(y); the
// bin g below the largest entry's has weight e^(-g/64) times the sum of its
// entries' e^(-(floor(y) + 1 - y) / 64), which are whole numbers of 2^-44 summed in
// 64 bits: exact in any order and however the row is cut.  Sums over bins say in
// which bin each filter and the draw end, and only the entries of these few bins
// are ordered.  2048 bins reach down to e^-32 of the largest weight; an entry
// below has none.
//   1. sample_bins_kernel: blocks of a row each sum their part into bins.
//   2. sample_draw_kernel: one block a row merges them, collects the entries of
//      the bins in question and ends the filters and the draw in them.
#include <algorithm>
#include "vte_common.h"

#define SMP_THREADS 1024
#define SMP_WAVES (SMP_THREADS / 64)
#define SMP_SUB 256         // entries whose largest one is kept (one wave's 16-byte load)
#define SMP_BINS 2048
#define SMP_PER_UNIT 64.0   // bins per unit of x / T
#define SMP_ONE 17592186044416.0  // 2^44
#define SMP_IDX_BITS 18
#define SMP_DIGIT 10
#define SMP_LEVELS 5        // 32 + 18 bits of (key, index) in digits of 10
#define SMP_LIST 6144       // entries that are collected at most; more: the row is read again
#define SMP_SMALL 1024      // entries of a bin that are ordered by counting
#define SMP_SPLIT 16        // blocks of a row at most

// Scratch of a row.
struct SmpScratch {
    uint64_t* mass;  // [blocks][SMP_BINS]
    uint32_t* count; // [blocks][SMP_BINS], rows with a top-k only
    float* sub;      // [entries / SMP_SUB] largest entry of each
    float* max;      // [blocks]
};
__host__ __device__ inline size_t smp_row_bytes(int blocks, int subs) {
    return (size_t)blocks * SMP_BINS * 12 + ((size_t)subs * 4 + SMP_SPLIT * 4 + 15) / 16 * 16;
}
__device__ __forceinline__ SmpScratch smp_scratch(uint8_t* base, int row, int blocks, int subs) {
    uint8_t* p = base + (size_t)row * smp_row_bytes(blocks, subs);
    SmpScratch s;
    s.mass = reinterpret_cast<uint64_t*>(p);
    s.count = reinterpret_cast<uint32_t*>(p + (size_t)blocks * SMP_BINS * 8);
    s.max = reinterpret_cast<float*>(p + (size_t)blocks * SMP_BINS * 12);
    s.sub = s.max + SMP_SPLIT;
    return s;
}

// Order-preserving key: larger value, larger key (NaN does not come here).
__device__ __forceinline__ uint32_t smp_key(float x) {
    const uint32_t u = __float_as_uint(x == 0.f ? 0.f : x);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
// Place of an entry in the order, as one number: larger comes first.
__device__ __forceinline__ uint64_t smp_place(float x, int i) {
    return ((uint64_t)smp_key(x) << SMP_IDX_BITS) | (uint64_t)(((1 << SMP_IDX_BITS) - 1) - i);
}
__device__ __forceinline__ int smp_index(uint64_t place) {
    return ((1 << SMP_IDX_BITS) - 1) - (int)(place & ((1 << SMP_IDX_BITS) - 1));
}

// Where a row's bins lie: the largest value (of the row or of a part), 64 / T and floor(64 max / T).
struct SmpScale {
    float max;
    double s, top;
};
__device__ __forceinline__ SmpScale smp_scale(float max, float T) {
    SmpScale c;
    c.max = max;
    c.s = SMP_PER_UNIT / (double)T;
    c.top = floor((double)max * c.s);
    return c;
}
// Bin of x (false: no weight, NaN among them) and its weight in the bin, in units of 2^-44.
__device__ __forceinline__ bool smp_bin(const SmpScale& c, float x, int& g, uint64_t& m) {
    const double y = (double)x * c.s, a = floor(y);
    double d = c.top - a, f = (a + 1.0 - y) * (1.0 / SMP_PER_UNIT);
    if (x == c.max && !(fabs(d) < 1.0)) d = 0.0, f = 0.0;  // infinite or beyond whole numbers: itself alone
    if (!(d < (double)SMP_BINS)) return false;
    g = (int)d;
    double p = fma(f, 1.0 / 720.0, -1.0 / 120.0);  // e^-f, f <= 1/64: the next term is below 2^-54
    p = fma(f, p, 1.0 / 24.0);
    p = fma(f, p, -1.0 / 6.0);
    p = fma(f, p, 0.5);
    p = fma(f, p, -1.0);
    p = fma(f, p, 1.0);
    // 2^52 + p 2^44 holds the whole number in its low bits
    m = (uint64_t)__double_as_longlong(fma(p, SMP_ONE, 4503599627370496.0)) & 0xFFFFFFFFFFFFFull;
    return true;
}

// Four entries of subset `sub` that lane holds: 16-byte loads where the row allows them.
struct SmpFour {
    float x[4];
    int i[4];
};
__device__ __forceinline__ SmpFour smp_load(const float* row, int vocab, int sub, int lane, bool wide) {
    SmpFour r;
    const int base = sub * SMP_SUB;
    if (wide && base + SMP_SUB <= vocab) {
        const float4 v = *reinterpret_cast<const float4*>(row + base + 4 * lane);
        r.x[0] = v.x; r.x[1] = v.y; r.x[2] = v.z; r.x[3] = v.w;
#pragma unroll
        for (int e = 0; e < 4; ++e) r.i[e] = base + 4 * lane + e;
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            r.i[e] = base + 64 * e + lane;
            r.x[e] = r.i[e] < vocab ? row[r.i[e]] : -INFINITY;
        }
    }
    return r;
}
__device__ __forceinline__ float smp_max4(const SmpFour& r) {  // NaN counts as nothing
    return fmaxf(fmaxf(fmaxf(r.x[0], -INFINITY), r.x[1]), fmaxf(r.x[2], r.x[3]));
}

// grid (blocks of a row, rows).  The block's first KEEP subsets a wave stay in registers between the two passes.
#define SMP_KEEP 4
__global__ __launch_bounds__(SMP_THREADS) void sample_bins_kernel(const float* __restrict__ logits, int vocab,
                                                                  const float* __restrict__ temperature,
                                                                  const int* __restrict__ top_k, uint8_t* scratch,
                                                                  int subs) {
    __shared__ unsigned long long mass[SMP_BINS];
    __shared__ unsigned count[SMP_BINS];
    __shared__ float wmax[SMP_WAVES];
    const int row = blockIdx.y, blocks = gridDim.x, tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    const float* x = logits + (size_t)row * vocab;
    const bool wide = (reinterpret_cast<uintptr_t>(x) & 15) == 0;
    const SmpScratch sc = smp_scratch(scratch, row, blocks, subs);
    const int lo = (int)((long long)subs * blockIdx.x / blocks), hi = (int)((long long)subs * (blockIdx.x + 1) / blocks);
    const float T = temperature ? temperature[row] : 1.f;
    const bool counts = top_k != nullptr && top_k[row] > 0;
    SmpFour keep[SMP_KEEP];
    float best = -INFINITY;
    auto first = [&](const SmpFour& f, int sub) {
        const float m = wave_max(smp_max4(f));
        if (lane == 0) sc.sub[sub] = m;
        best = fmaxf(best, m);
    };
#pragma unroll
    for (int j = 0; j < SMP_KEEP; ++j)
        if (lo + wv + SMP_WAVES * j < hi) keep[j] = smp_load(x, vocab, lo + wv + SMP_WAVES * j, lane, wide);
    for (int i = tid; i < SMP_BINS; i += SMP_THREADS) {
        mass[i] = 0;
        count[i] = 0;
    }
#pragma unroll
    for (int j = 0; j < SMP_KEEP; ++j)
        if (lo + wv + SMP_WAVES * j < hi) first(keep[j], lo + wv + SMP_WAVES * j);
    for (int sub = lo + wv + SMP_WAVES * SMP_KEEP; sub < hi; sub += SMP_WAVES) first(smp_load(x, vocab, sub, lane, wide), sub);
    if (lane == 0) wmax[wv] = best;
    __syncthreads();
    best = wmax[0];
#pragma unroll
    for (int w = 1; w < SMP_WAVES; ++w) best = fmaxf(best, wmax[w]);
    if (tid == 0) sc.max[blockIdx.x] = best;
    if (!(best > -INFINITY) || !(T > 0.f)) return;  // nothing in it; greedy rows need the maxima only
    const SmpScale c = smp_scale(best, T);
    auto second = [&](const SmpFour& f) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            int g;
            uint64_t m;
            if (!smp_bin(c, f.x[e], g, m)) continue;
            atomicAdd(&mass[g], (unsigned long long)m);
            if (counts) atomicAdd(&count[g], 1u);
        }
    };
#pragma unroll
    for (int j = 0; j < SMP_KEEP; ++j)
        if (lo + wv + SMP_WAVES * j < hi) second(keep[j]);
#pragma unroll 2
    for (int sub = lo + wv + SMP_WAVES * SMP_KEEP; sub < hi; sub += SMP_WAVES) second(smp_load(x, vocab, sub, lane, wide));
    __syncthreads();
    for (int i = tid; i < SMP_BINS; i += SMP_THREADS) {
        sc.mass[(size_t)blockIdx.x * SMP_BINS + i] = mass[i];
        if (counts) sc.count[(size_t)blockIdx.x * SMP_BINS + i] = count[i];
    }
}

// Sum over the threads up to and with this one; `sh` holds one value a wave.
template <typename V>
__device__ __forceinline__ V smp_scan(V v, V* sh) {
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const V up = __shfl_up(v, d, 64);
        if (lane >= d) v += up;
    }
    __syncthreads();
    if (lane == 63) sh[wv] = v;
    __syncthreads();
    V before = 0;
    for (int w = 0; w < wv; ++w) before += sh[w];
    return before + v;
}

struct SmpRow {
    const float* x;
    int vocab, subs;
    bool wide;
    SmpScale c;
};
struct SmpShared {
    uint64_t mass[SMP_BINS];    // weight of all bins up to and with this one, in 2^-44 of the largest possible
    uint32_t count[SMP_BINS];
    uint64_t list[SMP_LIST];    // places of the collected entries
    uint64_t place[SMP_SMALL];  // of one bin; digits' sums of a large one
    uint64_t m[SMP_SMALL];
    uint32_t digit_n[SMP_SMALL];
    uint16_t need[1024];        // subsets that may hold wanted entries
    uint32_t wanted[SMP_BINS / 32];
    uint64_t wave[SMP_WAVES];
    uint64_t found, found_m;
    int n, n_need, n_match, overflow;
};

__device__ __forceinline__ double smp_edge(int g) { return exp(-(double)g / SMP_PER_UNIT); }  // weight at the bin's upper end
// First bin whose running weight exceeds t (the last one with weight if none does): a bin with weight, whatever t is.
__device__ __forceinline__ int smp_find(const SmpShared& S, double t) {
    const double all = (double)S.mass[SMP_BINS - 1];
    const bool none = !(all > t);
    int lo = 0, hi = SMP_BINS - 1;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        const double m = (double)S.mass[mid];
        if (none ? m >= all : m > t) hi = mid;
        else lo = mid + 1;
    }
    return lo;
}
__device__ __forceinline__ double smp_before(const SmpShared& S, int g) { return g ? (double)S.mass[g - 1] : 0.0; }

// f(place, bin, weight) for the entries in question: the collected ones, or where there were too many all of the row's.
template <typename F>
__device__ __forceinline__ void smp_each(const SmpShared& S, const SmpRow& r, F f) {
    int g;
    uint64_t m;
    if (!S.overflow) {
        for (int i = threadIdx.x; i < S.n; i += SMP_THREADS) {
            const uint64_t c = S.list[i];
            const uint32_t k = (uint32_t)(c >> SMP_IDX_BITS);
            if (smp_bin(r.c, __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k), g, m)) f(c, g, m);
        }
        return;
    }
    for (int i = threadIdx.x; i < r.vocab; i += SMP_THREADS) {
        const float x = r.x[i];
        if (smp_bin(r.c, x, g, m)) f(smp_place(x, i), g, m);
    }
}

// In bin b (one with entries): the first entry in the order at which the running weight exceeds t (COUNT: the t-th
// entry, from 1), the bin's last one if none does.  Its place, and the bin's weight up to and with it.  All threads.
template <bool COUNT>
__device__ uint64_t smp_end(SmpShared& S, const SmpRow& r, int b, double t, uint64_t& upto) {
    const int tid = threadIdx.x;
    t = fmax(t, COUNT ? 1.0 : 0.0);
    __syncthreads();
    if (tid == 0) S.n_match = 0;
    __syncthreads();
    smp_each(S, r, [&](uint64_t c, int g, uint64_t m) {
        if (g != b) return;
        const int at = atomicAdd(&S.n_match, 1);
        if (at < SMP_SMALL) {
            S.place[at] = c;
            S.m[at] = m;
        }
    });
    __syncthreads();
    const int n = S.n_match;
    if (n <= SMP_SMALL) {  // every entry sums those before it
        if (tid < n) {
            const uint64_t mine = S.place[tid];
            uint64_t sum = 0, rank = 0;
            for (int i = 0; i < n; ++i) {
                const bool before = S.place[i] >= mine;
                sum += before ? S.m[i] : 0;
                rank += before;
            }
            const bool passes = COUNT ? (double)rank >= t : (double)sum > t;
            const bool passed = COUNT ? (double)(rank - 1) >= t : (double)(sum - S.m[tid]) > t;
            if ((passes && !passed) || (!passes && rank == (uint64_t)n)) {
                S.found = mine;
                S.found_m = sum;
            }
        }
        __syncthreads();
        upto = S.found_m;
        return S.found;
    }
    // many entries in one bin (a flat row, ties): digit by digit over the places
    uint64_t prefix = 0, before = 0, before_n = 0;
    for (int level = 0; level < SMP_LEVELS; ++level) {
        const int shift = (SMP_LEVELS - 1 - level) * SMP_DIGIT;
        __syncthreads();
        S.m[tid] = 0;
        S.digit_n[tid] = 0;
        __syncthreads();
        smp_each(S, r, [&](uint64_t c, int g, uint64_t m) {
            if (g != b || (level > 0 && (c >> (shift + SMP_DIGIT)) != prefix)) return;
            const int d = SMP_THREADS - 1 - ((int)(c >> shift) & (SMP_THREADS - 1));  // largest first
            atomicAdd((unsigned long long*)&S.m[d], (unsigned long long)m);
            atomicAdd(&S.digit_n[d], 1u);
        });
        __syncthreads();
        const uint64_t m = S.m[tid], c = S.digit_n[tid];
        const uint64_t sum = before + smp_scan<unsigned long long>(m, (unsigned long long*)S.wave);
        __syncthreads();
        const uint64_t num = before_n + smp_scan<unsigned long long>(c, (unsigned long long*)S.wave);
        const bool passes = COUNT ? (double)num >= t : (double)sum > t;
        const bool passed = COUNT ? (double)(num - c) >= t : (double)(sum - m) > t;
        __syncthreads();
        if (tid == 0) S.n_match = -1;
        __syncthreads();
        if (c && !passed) atomicMax(&S.n_match, passes ? SMP_THREADS : tid);  // the last digit, if none passes
        __syncthreads();
        const int last = S.n_match;
        __syncthreads();
        if (c && !passed && (last == SMP_THREADS ? passes : tid == last)) {
            S.found = (uint64_t)(SMP_THREADS - 1 - tid);
            S.place[0] = sum - m;
            S.place[1] = num - c;
            S.found_m = sum;
        }
        __syncthreads();
        prefix = (prefix << SMP_DIGIT) | S.found;
        before = S.place[0];
        before_n = S.place[1];
    }
    upto = S.found_m;
    return prefix;
}

__global__ __launch_bounds__(SMP_THREADS) void sample_draw_kernel(const float* __restrict__ logits, int vocab,
                                                                  const float* __restrict__ temperature,
                                                                  const int* __restrict__ top_k,
                                                                  const float* __restrict__ top_p,
                                                                  const float* __restrict__ min_p,
                                                                  const double* __restrict__ u, int* __restrict__ tokens,
                                                                  uint8_t* scratch, int blocks, int subs) {
    __shared__ SmpShared S;
    const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    const SmpScratch sc = smp_scratch(scratch, row, blocks, subs);
    const float T = temperature ? temperature[row] : 1.f;
    float top = sc.max[0];
    for (int i = 1; i < blocks; ++i) top = fmaxf(top, sc.max[i]);
    SmpRow r;
    r.x = logits + (size_t)row * vocab;
    r.vocab = vocab;
    r.subs = subs;
    r.wide = (reinterpret_cast<uintptr_t>(r.x) & 15) == 0;
    if (!(top > -INFINITY)) {  // nothing to draw from
        if (tid == 0) tokens[row] = -1;
        return;
    }
    if (!(T > 0.f)) {  // greedy: the first subset with the maximum, its first entry
        if (tid == 0) S.n = subs;
        __syncthreads();
        for (int s = tid; s < subs; s += SMP_THREADS)
            if (sc.sub[s] == top) atomicMin(&S.n, s);
        __syncthreads();
        if (wv == 0) {
            const SmpFour f = smp_load(r.x, vocab, S.n, lane, r.wide);
            int at = vocab;
#pragma unroll
            for (int e = 3; e >= 0; --e) at = f.x[e] == top ? min(at, f.i[e]) : at;
            for (int d = 1; d < 64; d *= 2) at = min(at, __shfl_xor(at, d, 64));
            if (lane == 0) tokens[row] = at;
        }
        return;
    }
    r.c = smp_scale(top, T);
    const int k = top_k ? top_k[row] : 0;
    const double p = top_p ? (double)top_p[row] : 1.0, mp = min_p ? (double)min_p[row] : 0.0;
    const bool has_k = k > 0, has_p = p > 0.0 && p < 1.0, has_m = mp > 0.0;

    // ---- the row's bins: thread t sums bins 2 t and 2 t + 1 over the parts ----
    uint64_t m[2] = {0, 0};
    uint32_t n[2] = {0, 0};
    for (int i = 0; i < blocks; ++i) {
        const float part = sc.max[i];
        if (!(part > -INFINITY)) continue;
        const double d = part == top ? 0.0 : r.c.top - floor((double)part * r.c.s);  // bins between their first ones
        if (!(d < (double)SMP_BINS)) continue;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int g = 2 * tid + e - (int)d;
            if (g < 0) continue;
            m[e] += sc.mass[(size_t)i * SMP_BINS + g];
            if (has_k) n[e] += sc.count[(size_t)i * SMP_BINS + g];
        }
    }
    {
        // whole numbers again, so that running sums do not fall and an empty bin adds nothing
        const unsigned long long a = (unsigned long long)rint((double)m[0] * smp_edge(2 * tid));
        const unsigned long long b = (unsigned long long)rint((double)m[1] * smp_edge(2 * tid + 1));
        const unsigned long long s = smp_scan<unsigned long long>(a + b, (unsigned long long*)S.wave);
        S.mass[2 * tid] = s - b;
        S.mass[2 * tid + 1] = s;
        if (has_k) {
            __syncthreads();
            const uint32_t c = smp_scan<uint32_t>(n[0] + n[1], (uint32_t*)S.wave);
            S.count[2 * tid] = c - n[1];
            S.count[2 * tid + 1] = c;
        }
    }
    for (int i = tid; i < SMP_BINS / 32; i += SMP_THREADS) S.wanted[i] = 0;
    if (tid == 0) {
        S.n = 0;
        S.n_need = 0;
        S.overflow = 0;
    }
    __syncthreads();

    // ---- in which bins the filters and the draw may end ----
    const double all = (double)S.mass[SMP_BINS - 1];
    double z_lo = all, z_hi = all;  // mass of the top-k
    int kb = -1;
    if (has_k && (uint32_t)k < S.count[SMP_BINS - 1]) {
        int lo = 0, hi = SMP_BINS - 1;  // first bin whose running count reaches k
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (S.count[mid] >= (uint32_t)k) hi = mid;
            else lo = mid + 1;
        }
        z_hi = (double)S.mass[lo];
        z_lo = z_hi;
        if (S.count[lo] != (uint32_t)k) {
            kb = lo;
            z_lo = smp_before(S, lo);
        }
    }
    int last = kb, p0 = 0, p1 = -1, m0 = 0, m1 = -1;
    double k_lo = z_lo, k_hi = z_hi;  // kept mass
    if (has_p) {
        p0 = smp_find(S, p * z_lo);
        p1 = z_lo == z_hi ? p0 : smp_find(S, p * z_hi);
        k_lo = fmin(k_lo, smp_before(S, p0));
        k_hi = fmin(k_hi, (double)S.mass[p1]);
        last = max(last, p1);
    }
    double floor_w = 0.0;
    if (has_m) {  // bins around the least weight's
        int g = 0;
        uint64_t w = 0;
        smp_bin(r.c, top, g, w);
        floor_w = fmin(mp, 1.0) * (double)w;  // in units of 2^-44 of bin 0's upper end
        const double y = (log(SMP_ONE) - log(floor_w)) * SMP_PER_UNIT;
        m0 = (int)fmin(fmax(floor(y - 1e-6), 0.0), (double)(SMP_BINS - 1));
        m1 = (int)fmin(fmax(floor(y + 1e-6), 0.0), (double)(SMP_BINS - 1));
        k_lo = fmin(k_lo, smp_before(S, m0));
        k_hi = fmin(k_hi, (double)S.mass[m1]);
        last = max(last, m1);
    }
    const double uu = fmin(fmax(u[row], 0.0), 1.0);  // NaN: 0
    // the draw lies before the end of the kept mass even where u is 1
    auto drawn = [&](double mass) { return fmin(uu * mass, mass * (1.0 - 1e-15)); };
    const int u0 = smp_find(S, drawn(k_lo)), u1 = k_lo == k_hi ? u0 : smp_find(S, drawn(k_hi));
    last = max(last, u1);
    auto want = [&](int a, int b) {
        for (int g = a + tid; g <= b; g += SMP_THREADS) atomicOr(&S.wanted[g >> 5], 1u << (g & 31));
    };
    if (kb >= 0) want(kb, kb);
    want(p0, p1);
    want(m0, m1);
    want(u0, u1);
    // ---- collect their entries, from the subsets whose largest one is not behind the last of these bins ----
    for (int s = tid; s < subs; s += SMP_THREADS) {
        int g;
        uint64_t w;
        if (smp_bin(r.c, sc.sub[s], g, w) && g <= last) S.need[atomicAdd(&S.n_need, 1)] = (uint16_t)s;
    }
    __syncthreads();
    auto take = [&](const SmpFour& f) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            int g = 0;
            uint64_t w;
            const bool in = smp_bin(r.c, f.x[e], g, w) && (S.wanted[g >> 5] >> (g & 31) & 1);
            const uint64_t ask = __ballot(in);
            if (ask == 0) continue;
            int at = 0;
            if (lane == 0) at = atomicAdd(&S.n, __popcll(ask));
            at = __shfl(at, 0, 64) + __popcll(ask & ((1ull << lane) - 1));
            if (in && at < SMP_LIST) S.list[at] = smp_place(f.x[e], f.i[e]);
        }
    };
    for (int i = wv; i < S.n_need; i += 4 * SMP_WAVES) {
        SmpFour f[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (i + j * SMP_WAVES < S.n_need) f[j] = smp_load(r.x, vocab, S.need[i + j * SMP_WAVES], lane, r.wide);
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (i + j * SMP_WAVES < S.n_need) take(f[j]);
    }
    __syncthreads();
    if (tid == 0 && S.n > SMP_LIST) S.overflow = 1;
    __syncthreads();

    // ---- end the filters, then the draw ----
    uint64_t upto;
    double z = z_hi;
    if (kb >= 0) {
        smp_end<true>(S, r, kb, (double)((uint32_t)k - (kb ? S.count[kb - 1] : 0)), upto);
        z = fmin(fmax(smp_before(S, kb) + (double)upto * smp_edge(kb), z_lo), z_hi);  // roundings apart it lies there
    }
    double kept = z;
    if (has_p) {
        const int b = smp_find(S, p * z);
        smp_end<false>(S, r, b, (p * z - smp_before(S, b)) / smp_edge(b), upto);
        kept = fmin(kept, smp_before(S, b) + (double)upto * smp_edge(b));
    }
    if (has_m) {  // the weights in bins m0 and m1 that reach the least one
        __syncthreads();
        if (tid < 2) S.m[tid] = 0;
        __syncthreads();
        const double e0 = smp_edge(m0), e1 = smp_edge(m1);
        smp_each(S, r, [&](uint64_t, int g, uint64_t w) {
            if ((g == m0 && (double)w * e0 >= floor_w) || (g == m1 && (double)w * e1 >= floor_w))
                atomicAdd((unsigned long long*)&S.m[g == m0 ? 0 : 1], (unsigned long long)w);
        });
        __syncthreads();
        kept = fmin(kept, smp_before(S, m0) + (double)S.m[0] * e0 + (double)S.m[1] * e1);
    }
    const double t = drawn(fmin(fmax(kept, k_lo), k_hi));
    const int b = smp_find(S, t);
    const uint64_t place = smp_end<false>(S, r, b, (t - smp_before(S, b)) / smp_edge(b), upto);
    if (tid == 0) tokens[row] = smp_index(place);
}

namespace vte {
// Blocks of a row: enough that two of 1024 threads lie on every CU.
static int sample_blocks(int rows) { return std::max(1, std::min(SMP_SPLIT, 2 * device_cus() / rows)); }

long long sample_scratch_bytes(int rows) {
    return (long long)rows * (long long)smp_row_bytes(sample_blocks(rows), (1 << SMP_IDX_BITS) / SMP_SUB);
}
hipError_t sample(const float* logits, int rows, int vocab, const float* temperature, const int* top_k,
                  const float* top_p, const float* min_p, const double* u, int* tokens, void* scratch,
                  hipStream_t st) {
    const int subs = (vocab + SMP_SUB - 1) / SMP_SUB, blocks = std::min(sample_blocks(rows), subs);
    hipLaunchKernelGGL(sample_bins_kernel, dim3(blocks, rows), dim3(SMP_THREADS), 0, st, logits, vocab, temperature,
                       top_k, (uint8_t*)scratch, subs);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(sample_draw_kernel, dim3(rows), dim3(SMP_THREADS), 0, st, logits, vocab, temperature, top_k,
                       top_p, min_p, u, tokens, (uint8_t*)scratch, blocks, subs);
    return hipGetLastError();
}
}  // namespace vte
