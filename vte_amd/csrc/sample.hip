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
// The row is not sorted.  With y = 32 x / T, entries fall into bins round(y); the
// bin g below the largest entry's has weight e^(-g/32) times the sum of its
// entries' e^((y - round(y)) / 32), which are whole numbers of 2^-44 summed in 64
// bits: the same in any order and however the row is cut.  Sums over bins say in
// which bin each filter and the draw end, and only the entries of these few bins
// are ordered.  1024 bins reach down to e^-32 of the largest weight; an entry
// below has none, nor has a bin whose sum is below 2^-45 of it.  An entry's weight
// and a bin's sum are rounded once each, by 2^-45 of the largest weight at most, so
// masses are off by vocab * 2^-44 of it at most; borders are compared in fp64.
//   1. sample_bins_kernel: blocks of a row each sum their part into bins.
//   2. sample_draw_kernel: merges them, collects the entries of the bins in
//      question and ends the filters and the draw in them.  One CU reads no more
//      than some 30 GB/s, so while there are few rows several blocks share a row's
//      reading: each merges for itself, and the last to be done (none waits) goes on.
//
// Bound by the two readings where there are many rows: 256 rows of 151936, 156 MB,
// bins 41 us (3.8 TB/s; some 25 vector operations and an LDS addition an entry take
// nearly as long), draw 60, of which reading 36 (a broad distribution's ends lie in
// bins that nearly all subsets reach into; of a peaked one it reads a few).  Few rows:
// by latencies, one row 8.5 + 12.5 us: merging 2, scans 2, bins in question 1, their
// entries 3, the last of the row's blocks 2, ends of the filters 2.
// With unaligned rows (not WIDE) / WIDE, us: one row 22.1 / 20.7, 256 105.7 / 98.5.
// Where the bins in question hold more than SMP_LIST entries one block reads the row again
// for every split, at a CU's rate: rows of 262144 nearly equal logits with a nucleus of
// 0.95, one row 519 us (of N(0, 1) 37), 16 rows 606 (419), 256 rows of 151936 564 (114).
#include <algorithm>
#include "vte_common.h"

#define SMP_THREADS 1024
#define SMP_WAVES (SMP_THREADS / 64)
#define SMP_SUB 256         // entries whose largest one is kept (one wave's 16-byte load)
#define SMP_BINS 1024       // one a thread
#define SMP_PER_UNIT 32.0   // bins per unit of x / T
#define SMP_ONE 17592186044416.0  // 2^44
#define SMP_IDX_BITS 18
#define SMP_DIGIT 10
#define SMP_LEVELS 5        // 32 + 18 bits of (key, index) in digits of 10
#define SMP_LIST 8192       // entries that are collected at most; more: the row is read again
#define SMP_SMALL 1024      // entries of a bin that are ordered by counting
#define SMP_FEW 128         // .. without a split first
#define SMP_AHEAD 4         // subsets a wave of the draw has in flight (8: one row 16.1 -> 18.6 us, 256 rows the same)
#define SMP_SPLIT 8         // blocks of a row at most (2 / 8, us: one row 30.6 / 22.5, 16 rows 37.8 / 30.9; 16 as 8)

// Scratch of a row.
struct SmpScratch {
    uint64_t* mass;  // [blocks][SMP_BINS]
    uint32_t* count; // [blocks][SMP_BINS], rows with a top-k only
    float* sub;      // [entries / SMP_SUB] largest entry of each
    float* max;      // [blocks]
    int* shared;     // entries collected, blocks of the draw that are done
    uint32_t* list;  // [SMP_LIST] their indices
};
__host__ __device__ inline size_t smp_row_bytes(int blocks, int subs) {
    return (size_t)blocks * SMP_BINS * 12 + (SMP_SPLIT + 4 + SMP_LIST) * 4 + ((size_t)subs * 4 + 15) / 16 * 16;
}
__device__ __forceinline__ SmpScratch smp_scratch(uint8_t* base, int row, int blocks, int subs) {
    uint8_t* p = base + (size_t)row * smp_row_bytes(blocks, subs);
    SmpScratch s;
    s.mass = reinterpret_cast<uint64_t*>(p);
    s.count = reinterpret_cast<uint32_t*>(p + (size_t)blocks * SMP_BINS * 8);
    s.max = reinterpret_cast<float*>(p + (size_t)blocks * SMP_BINS * 12);
    s.shared = reinterpret_cast<int*>(s.max + SMP_SPLIT);
    s.list = reinterpret_cast<uint32_t*>(s.shared + 4);
    s.sub = reinterpret_cast<float*>(s.list + SMP_LIST);
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
__device__ __forceinline__ float smp_value(uint64_t place) {
    const uint32_t k = (uint32_t)(place >> SMP_IDX_BITS);
    return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k);
}
__device__ __forceinline__ int smp_index(uint64_t place) {
    return ((1 << SMP_IDX_BITS) - 1) - (int)(place & ((1 << SMP_IDX_BITS) - 1));
}
// A drawn entry's token; -1 where none was found, which takes logits that change under the call.
__device__ __forceinline__ int smp_token(uint64_t place, int vocab) {
    const int i = smp_index(place);
    return place != 0 && i < vocab ? i : -1;
}

// Where a row's bins lie: the largest value (of the row or of a part), 32 / T, and the low word of round(32 max / T).
// Rounding adds 1.5 2^52, whose low word then holds the whole number: differences of up to 2^31 bins are right, and
// values that lie further down are raised to `low`, which is out of every bin.
#define SMP_ROUND 6755399441055744.0
struct SmpScale {
    float max, low;
    double s;
    int top;
    bool whole;  // 32 max / T is a place on this scale
    bool flat;   // if not: every finite value weighs the same (T infinite); else the largest is alone
};
__device__ __forceinline__ SmpScale smp_scale(float max, float T) {
    SmpScale c;
    c.max = max;
    c.s = SMP_PER_UNIT / (double)T;
    const double y = (double)max * c.s;
    c.whole = fabs(y) < 35184372088832.0 && c.s > 0.0;  // 2^45: from 2^40 on neighbours are 2^16 bins apart
    c.flat = !c.whole && !(c.s > 0.0) && max < INFINITY;
    // (As smp_bin rounds the largest entry itself.  The product rounded first comes to lie on a half for 1 of 30000 values at
    // T = 1e-9, and the largest entry then lay above the first bin, out of every one.)
    c.top = c.whole ? __double2loint(fma((double)max, c.s, SMP_ROUND)) : 0;
    const double low = c.whole ? (y - 1.5 * SMP_BINS) / c.s : 0.0;
    c.low = fmaxf(low < -3.4e38 ? -3.4e38f : (float)(low - 1.2e-7 * fabs(low) - 1e-45), -3.4028234664e38f);
    return c;
}
// fma with its constants in registers: the two-operand form that the compiler takes moves one there each time.
__device__ __forceinline__ double smp_fma(double a, double b, double c) {
    double d;
    asm("v_fma_f64 %0, %1, %2, %3" : "=v"(d) : "v"(a), "v"(b), "v"(c));
    return d;
}
// Bin of x (false: no weight, NaN among them) and its weight in the bin, in units of 2^-44: the series of e^(r / 32)
// for y = round(y) + r (the next term is below 2^-45).
// ABOVE: bins above the scale's largest value that count too (g is below 0 there).
template <int ABOVE = 0>
__device__ __forceinline__ bool smp_bin(const SmpScale& c, float x, int& g, uint64_t& m) {
    constexpr double H = 1.0 / SMP_PER_UNIT;
    double r = 0.0;
    bool in = x > -INFINITY;
    if (c.whole) {
        const double v = (double)fmaxf(x, c.low);
        const double t = fma(v, c.s, SMP_ROUND);
        r = fma(v, c.s, SMP_ROUND - t);
        g = c.top - __double2loint(t);
        in = in && (unsigned)(g + ABOVE) < SMP_BINS + ABOVE;
    } else {
        in = in && (c.flat || x == c.max);
        g = 0;
    }
    double p = smp_fma(r, H * H * H * H * H / 120.0, H * H * H * H / 24.0);
    p = smp_fma(r, p, H * H * H / 6.0);
    p = fma(r, p, H * H / 2.0);
    p = fma(r, p, H);
    p = fma(r, p, 1.0);
    // 2^52 + p 2^44 holds the whole number in its low bits
    m = (uint64_t)__double_as_longlong(smp_fma(p, SMP_ONE, 4503599627370496.0)) & 0xFFFFFFFFFFFFFull;
    return in;
}
// Place of x inside its bin, from the largest value on, in 1024 steps.
__device__ __forceinline__ int smp_inside(const SmpScale& c, float x) {
    if (!c.whole) return 0;
    const double t = fma((double)x, c.s, SMP_ROUND), r = fma((double)x, c.s, SMP_ROUND - t);
    return min(max((int)((0.5 - r) * (double)SMP_THREADS), 0), SMP_THREADS - 1);
}
// Bins from the scale's largest value up to a larger one; SMP_ROOM + 1 where that is more than SMP_ROOM.
__device__ __forceinline__ int smp_above(const SmpScale& c, float top) {
    const double d = fma((double)top, c.s, SMP_ROUND) - fma((double)c.max, c.s, SMP_ROUND);  // (differences of bins as smp_bin has them)
    return d <= (double)SMP_BINS ? (int)d : SMP_BINS + 1;
}
// Bins between the largest values of a part and of the row; SMP_BINS or more: none of the part's matter.
__device__ __forceinline__ int smp_apart(const SmpScale& c, float part) {
    if (part == c.max) return 0;
    if (!c.whole) return c.flat ? 0 : SMP_BINS;
    const int d = c.top - __double2loint(fma((double)fmaxf(part, c.low), c.s, SMP_ROUND));
    return (unsigned)d < SMP_BINS ? d : SMP_BINS;
}

// Four entries of a subset: lane's 16 bytes where every row is 16-byte aligned and whole (WIDE), else one of each 64.
// The load itself asks nothing of its values and takes no branch, so that several stay in flight; places behind the
// row's end hold an entry of the row until smp_cut.
struct SmpFour {
    float x[4];
};
template <bool WIDE>
__device__ __forceinline__ int smp_at(int sub, int lane, int e) {
    return sub * SMP_SUB + (WIDE ? 4 * lane + e : 64 * e + lane);
}
template <bool WIDE>
__device__ __forceinline__ SmpFour smp_load(const float* row, int vocab, int sub, int lane) {
    SmpFour r;
    if constexpr (WIDE) {
        const float4 v = *reinterpret_cast<const float4*>(row + min(smp_at<WIDE>(sub, lane, 0), vocab - 4));
        r.x[0] = v.x; r.x[1] = v.y; r.x[2] = v.z; r.x[3] = v.w;
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) r.x[e] = row[min(smp_at<WIDE>(sub, lane, e), vocab - 1)];
    }
    return r;
}
template <bool WIDE>
__device__ __forceinline__ void smp_cut(SmpFour& f, int vocab, int sub, int lane) {
    if ((sub + 1) * SMP_SUB <= vocab) return;  // (the same for a wave)
#pragma unroll
    for (int e = 0; e < 4; ++e) f.x[e] = smp_at<WIDE>(sub, lane, e) < vocab ? f.x[e] : -INFINITY;
}
__device__ __forceinline__ float smp_max4(const SmpFour& r) {  // NaN counts as nothing
    return fmaxf(fmaxf(fmaxf(r.x[0], -INFINITY), r.x[1]), fmaxf(r.x[2], r.x[3]));
}

// Largest of the wave's values of four subsets at once: lane 16 i has subset i's (halves, then rows of 16 lanes change
// places and carry two subsets each on; inside a row as whole numbers in the same order, which need no quieting).
typedef unsigned smp_u2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ float smp_max_of_four(float a, float b, float c, float d) {
    auto two = [](smp_u2 w) { return fmaxf(__uint_as_float(w[0]), __uint_as_float(w[1])); };
    const float ac = two(__builtin_amdgcn_permlane32_swap(__float_as_uint(a), __float_as_uint(c), false, false));
    const float bd = two(__builtin_amdgcn_permlane32_swap(__float_as_uint(b), __float_as_uint(d), false, false));
    const float x = two(__builtin_amdgcn_permlane16_swap(__float_as_uint(ac), __float_as_uint(bd), false, false));
    int i = (int)__float_as_uint(x);
    i ^= (i >> 31) & 0x7FFFFFFF;
    i = max(i, __builtin_amdgcn_update_dpp(i, i, 0xB1, 0xF, 0xF, false));
    i = max(i, __builtin_amdgcn_update_dpp(i, i, 0x4E, 0xF, 0xF, false));
    i = max(i, __builtin_amdgcn_update_dpp(i, i, 0x141, 0xF, 0xF, false));
    i = max(i, __builtin_amdgcn_update_dpp(i, i, 0x140, 0xF, 0xF, false));
    return __uint_as_float((uint32_t)(i ^ ((i >> 31) & 0x7FFFFFFF)));
}

// grid (blocks of a row, rows).  A part of at most KEEP subsets a wave (few rows) stays in registers while its largest
// entry is found.  A longer one is read once: its bins are laid from the largest entry of those first subsets on, with
// SMP_ROOM bins above it for what follows; if that is not enough (a much larger entry comes later) it is read again.
#define SMP_KEEP 8
#define SMP_ROOM SMP_BINS
template <bool WIDE>
__global__ __launch_bounds__(SMP_THREADS) void sample_bins_kernel(const float* __restrict__ logits, int vocab,
                                                                  const float* __restrict__ temperature,
                                                                  const int* __restrict__ top_k, uint8_t* scratch,
                                                                  int subs) {
    __shared__ unsigned long long mass[SMP_ROOM + SMP_BINS];
    __shared__ unsigned count[SMP_ROOM + SMP_BINS];
    __shared__ float wmax[2][SMP_WAVES];
    const int row = blockIdx.y, blocks = gridDim.x, tid = threadIdx.x, lane = tid & 63;
    const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    const float* x = logits + (size_t)row * vocab;
    const SmpScratch sc = smp_scratch(scratch, row, blocks, subs);
    const int lo = (int)((long long)subs * blockIdx.x / blocks), hi = (int)((long long)subs * (blockIdx.x + 1) / blocks);
    // subset j of this wave, one of the block's where there are fewer (lo < hi: no more blocks than subsets)
    auto nth = [&](int j) { return lo + wv + SMP_WAVES * j; };
    auto load = [&](int j) { return smp_load<WIDE>(x, vocab, min(nth(j), hi - 1), lane); };
    SmpFour keep[SMP_KEEP];
#pragma unroll
    for (int j = 0; j < SMP_KEEP; ++j) keep[j] = load(j);
    const float T = temperature ? temperature[row] : 1.f;
    const bool counts = top_k != nullptr && top_k[row] > 0;
    for (int i = tid; i < SMP_ROOM + SMP_BINS; i += SMP_THREADS) {
        mass[i] = 0;
        count[i] = 0;
    }
    float best = -INFINITY;
    auto first = [&](SmpFour* f, int j) {  // subsets j .. j + 3
        float m[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            smp_cut<WIDE>(f[i], vocab, min(nth(j + i), hi - 1), lane);
            m[i] = smp_max4(f[i]);
        }
        const float x = smp_max_of_four(m[0], m[1], m[2], m[3]);
        const int at = nth(j + (lane >> 4));
        if ((lane & 15) == 0 && at < hi) sc.sub[at] = x;
        best = fmaxf(best, x);  // (a subset twice changes nothing)
    };
    auto largest = [&](int i) {  // of all waves'
        const float m = fmaxf(fmaxf(wave_rows4(best, 0), wave_rows4(best, 1)), fmaxf(wave_rows4(best, 2), wave_rows4(best, 3)));
        if (lane == 0) wmax[i][wv] = m;
        __syncthreads();
        float x = wmax[i][0];
#pragma unroll
        for (int w = 1; w < SMP_WAVES; ++w) x = fmaxf(x, wmax[i][w]);
        return x;
    };
    const int n = (hi - lo + SMP_WAVES - 1) / SMP_WAVES;
#pragma unroll
    for (int j = 0; j < SMP_KEEP; j += 4) first(keep + j, j);
    const float ref = largest(0);
    const bool draws = T > 0.f;  // greedy rows need the maxima only
    const SmpScale c = smp_scale(ref, T);
    auto add = [&](const SmpScale& s, const SmpFour& f, int j) {
        if (nth(j) >= hi) return;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            int g;
            uint64_t m;
            if (!smp_bin<SMP_ROOM>(s, f.x[e], g, m)) continue;
            atomicAdd(&mass[SMP_ROOM + g], (unsigned long long)m);
            if (counts) atomicAdd(&count[SMP_ROOM + g], 1u);
        }
    };
    float top = ref;
    int shift = 0;
    if (n <= SMP_KEEP) {
        if (draws && ref > -INFINITY) {
#pragma unroll
            for (int j = 0; j < SMP_KEEP; ++j) add(c, keep[j], j);
        }
    } else {
        const bool lay = draws && c.whole;
        SmpFour f[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = load(SMP_KEEP + i);
        if (lay) {
#pragma unroll
            for (int j = 0; j < SMP_KEEP; ++j) add(c, keep[j], j);
        }
        for (int j = SMP_KEEP; j < n; j += 4) {
            SmpFour ahead[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) ahead[i] = load(j + 4 + i);
            first(f, j);
            if (lay) {
#pragma unroll
                for (int i = 0; i < 4; ++i) add(c, f[i], j + i);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) f[i] = ahead[i];
        }
        top = largest(1);
        shift = lay ? smp_above(c, top) : SMP_ROOM + 1;
        if (shift > SMP_ROOM && draws && top > -INFINITY) {  // once more, from the largest entry on
            for (int i = tid; i < SMP_ROOM + SMP_BINS; i += SMP_THREADS) {
                mass[i] = 0;
                count[i] = 0;
            }
            __syncthreads();
            const SmpScale t = smp_scale(top, T);
            for (int j = 0; j < n; j += 4) {
#pragma unroll
                for (int i = 0; i < 4; ++i) f[i] = load(j + i);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    smp_cut<WIDE>(f[i], vocab, min(nth(j + i), hi - 1), lane);
                    add(t, f[i], j + i);
                }
            }
            shift = 0;
        }
    }
    if (tid == 0) sc.max[blockIdx.x] = top;
    if (tid < 2 && blockIdx.x == 0) sc.shared[tid] = 0;
    if (!draws || !(top > -INFINITY)) return;
    __syncthreads();
    sc.mass[(size_t)blockIdx.x * SMP_BINS + tid] = mass[SMP_ROOM - shift + tid];
    if (counts) sc.count[(size_t)blockIdx.x * SMP_BINS + tid] = count[SMP_ROOM - shift + tid];
}

// Sum over the threads up to and with this one; `sh` holds one value a wave.  Inside a wave: shifts by 1, 2, 4 and 8
// in rows of 16 lanes, then the rows' last lanes into the rows behind them.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t smp_from(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xF, false);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ uint64_t smp_from(uint64_t v) {
    return (uint64_t)smp_from<CTRL, ROWS>((uint32_t)v) | (uint64_t)smp_from<CTRL, ROWS>((uint32_t)(v >> 32)) << 32;
}
__device__ __forceinline__ uint32_t smp_lane(uint32_t v, int l) { return (uint32_t)__builtin_amdgcn_readlane((int)v, l); }
__device__ __forceinline__ uint64_t smp_lane(uint64_t v, int l) {
    return (uint64_t)smp_lane((uint32_t)v, l) | (uint64_t)smp_lane((uint32_t)(v >> 32), l) << 32;
}
template <typename V>
__device__ __forceinline__ V smp_rows_scan(V v) {  // in rows of 16 lanes
    v += smp_from<0x111, 0xF>(v);
    v += smp_from<0x112, 0xF>(v);
    v += smp_from<0x114, 0xF>(v);
    v += smp_from<0x118, 0xF>(v);
    return v;
}
template <typename V>
__device__ __forceinline__ V smp_wave_scan(V v) {
    v = smp_rows_scan(v);
    v += smp_from<0x142, 0xA>(v);
    v += smp_from<0x143, 0xC>(v);
    return v;
}
template <typename V>
__device__ __forceinline__ V smp_join(V v, const V* sh, V& all) {  // with the waves' sums
    const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const V w = smp_rows_scan(sh[threadIdx.x & 15]);
    all = smp_lane(w, 15);
    return v + (wv > 0 ? smp_lane(w, wv - 1) : 0);
}
template <typename V>
__device__ __forceinline__ V smp_scan(V v, V* sh) {
    V all;
    v = smp_wave_scan(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 63) sh[threadIdx.x >> 6] = v;
    __syncthreads();
    return smp_join(v, sh, all);
}

struct SmpRow {
    const float* x;
    int vocab;
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
    uint64_t wave[SMP_WAVES], before[2];
    uint32_t wave_n[SMP_WAVES];
    uint64_t found, found_m;
    int n, n_need, n_match, overflow, hit[2];
};

__device__ __forceinline__ double smp_middle(int g) { return exp(-(double)g / SMP_PER_UNIT); }  // weight at the bin's middle
// First bin whose running weight exceeds t0 (t1): the last one with weight if none does.  Thread t holds the running
// weight with and before bin t, and that of all.
struct SmpMine {
    double before, with, all;
};
__device__ __forceinline__ void smp_find(SmpShared& S, const SmpMine& v, double t0, double t1, int& g0, int& g1) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const double t = i ? t1 : t0;
        const bool none = !(v.all > t);
        if (none ? v.before < v.all && v.with >= v.all : v.before <= t && v.with > t) S.hit[i] = threadIdx.x;
    }
    __syncthreads();
    g0 = S.hit[0];
    g1 = S.hit[1];
}
__device__ __forceinline__ double smp_before(const SmpShared& S, int g) { return g ? (double)S.mass[g - 1] : 0.0; }

// f(place, bin, weight) for the entries in question: the collected ones, or where there were too many all of the row's.
template <typename F>
__device__ __forceinline__ void smp_each(const SmpShared& S, const SmpRow& r, F f) {
    int g;
    uint64_t m;
    if (!S.overflow) {
        for (int i = threadIdx.x; i < S.n; i += SMP_THREADS) {
            const uint64_t c = S.list[i];  // (0 has the value of a NaN)
            if (smp_bin(r.c, smp_value(c), g, m)) f(c, g, m);
        }
        return;
    }
    for (int i = threadIdx.x; i < r.vocab; i += SMP_THREADS) {
        const float x = r.x[i];
        if (smp_bin(r.c, x, g, m)) f(smp_place(x, i), g, m);
    }
}

// Sum over the 16 lanes of a row: every lane gets it.
template <typename V>
__device__ __forceinline__ V smp_row_sum(V v) {
    v += smp_from<0xB1, 0xF>(v);
    v += smp_from<0x4E, 0xF>(v);
    v += smp_from<0x141, 0xF>(v);
    v += smp_from<0x140, 0xF>(v);
    return v;
}
// Ends in the n <= SMP_SMALL entries of S.place and S.m, `sum0` and `rank0` before them: as smp_end.  16 lanes count
// what is before an entry.
template <bool COUNT>
__device__ __forceinline__ void smp_end_few(SmpShared& S, int n, double t, uint64_t sum0, uint64_t rank0) {
    const int part = threadIdx.x & 15;
    for (int at = threadIdx.x >> 4; at < n; at += SMP_THREADS / 16) {
        const uint64_t mine = S.place[at], w = S.m[at];
        uint64_t sum = 0;
        uint32_t r = 0;
        for (int i = part; i < n; i += 16) {
            const bool before = S.place[i] >= mine;
            sum += before ? S.m[i] : 0;
            r += before;
        }
        sum = sum0 + smp_row_sum(sum);
        const uint64_t rank = rank0 + smp_row_sum(r);
        const bool passes = COUNT ? (double)rank >= t : (double)sum > t;
        const bool passed = COUNT ? (double)(rank - 1) >= t : (double)(sum - w) > t;
        if (part == 0 && ((passes && !passed) || (!passes && rank == rank0 + n))) {
            S.found = mine;
            S.found_m = sum;
        }
    }
}

// In bin b (one with entries): the first entry in the order at which the running weight exceeds t (COUNT: the t-th
// entry, from 1), the bin's last one if none does.  Its place, and the bin's weight up to and with it.  All threads.
// Up to 128 entries count those before them; more are first split into 1024 steps of the bin; where one of these holds
// more than SMP_SMALL (a flat row, ties), digit by digit over the places.
template <bool COUNT>
__device__ uint64_t smp_end(SmpShared& S, const SmpRow& r, int b, double t, uint64_t& upto) {
    const int tid = threadIdx.x;
    t = fmax(t, COUNT ? 1.0 : 0.0);
    auto collect = [&](int step) {  // the bin's entries (of one step) into place and m, SMP_SMALL at most
        __syncthreads();
        if (tid == 0) {
            S.n_match = 0;
            S.found = 0;  // (no entry's place; what a split found has been read)
        }
        __syncthreads();
        smp_each(S, r, [&](uint64_t c, int g, uint64_t m) {
            if (g != b || (step >= 0 && smp_inside(r.c, smp_value(c)) != step)) return;
            const int at = atomicAdd(&S.n_match, 1);
            if (at < SMP_SMALL) {
                S.place[at] = c;
                S.m[at] = m;
            }
        });
        __syncthreads();
        return S.n_match;
    };
    // sums over 1024 classes of entries, class `of` each (< 0: not in question): the class in which it ends
    uint64_t sum0 = 0, rank0 = 0;
    auto split = [&](auto of) {
        __syncthreads();
        S.m[tid] = 0;
        S.digit_n[tid] = 0;
        __syncthreads();
        smp_each(S, r, [&](uint64_t c, int g, uint64_t m) {
            const int d = g == b ? of(c) : -1;
            if (d < 0) return;
            atomicAdd((unsigned long long*)&S.m[d], (unsigned long long)m);
            atomicAdd(&S.digit_n[d], 1u);
        });
        __syncthreads();
        const uint64_t m = S.m[tid];
        const uint32_t n = S.digit_n[tid];
        uint64_t sum = smp_wave_scan(m), all;
        uint32_t rank32 = smp_wave_scan(n), all_n;
        if ((tid & 63) == 63) {
            S.wave[tid >> 6] = sum;
            S.wave_n[tid >> 6] = rank32;
        }
        __syncthreads();
        sum = sum0 + smp_join(sum, S.wave, all);
        rank32 = smp_join(rank32, S.wave_n, all_n);
        const uint64_t rank = rank0 + rank32;
        const bool passes = COUNT ? (double)rank >= t : (double)sum > t;
        const bool passed = COUNT ? (double)(rank - n) >= t : (double)(sum - m) > t;
        const bool none = COUNT ? !((double)(rank0 + all_n) >= t) : !((double)(sum0 + all) > t);
        if (n && (none ? rank32 == all_n : passes && !passed)) {  // none passes: the last class
            S.found = (uint64_t)tid;
            S.found_m = sum;
            S.before[0] = sum - m;
            S.before[1] = rank - n;
        }
        __syncthreads();
        sum0 = S.before[0];
        rank0 = S.before[1];
        return (int)S.found;
    };
    int n = S.n > 4 * SMP_FEW ? SMP_SMALL + 1 : collect(-1);  // (of many collected ones most bins have more)
    if (n > SMP_FEW) {
        const int step = split([&](uint64_t c) { return smp_inside(r.c, smp_value(c)); });
        n = collect(step);
        if (n > SMP_SMALL) {
            uint64_t prefix = 0;
            sum0 = rank0 = 0;
            for (int level = 0; level < SMP_LEVELS; ++level) {
                const int shift = (SMP_LEVELS - 1 - level) * SMP_DIGIT;
                const int d = split([&](uint64_t c) {
                    return level > 0 && (c >> (shift + SMP_DIGIT)) != prefix
                               ? -1 : SMP_THREADS - 1 - ((int)(c >> shift) & (SMP_THREADS - 1));  // largest first
                });
                prefix = (prefix << SMP_DIGIT) | (uint64_t)(SMP_THREADS - 1 - d);
            }
            upto = S.found_m;
            return prefix;
        }
    }
    smp_end_few<COUNT>(S, n, t, sum0, rank0);
    __syncthreads();
    upto = S.found_m;
    return S.found;
}

// The kernel's last part for at most 64 collected entries, in one wave: the token.
template <typename F>
__device__ __forceinline__ int smp_end_wave(const SmpShared& S, const SmpRow& r, int lane, int kb, int k, bool has_p, double p,
                                            int p0, int p1, bool has_m, int m0, int m1, double floor_w, double z_lo,
                                            double z_hi, double k_lo, double k_hi, int u0, int u1, F drawn) {
    const uint64_t c = lane < S.n ? S.list[lane] : 0;
    int g;
    uint64_t m;
    if (!smp_bin(r.c, smp_value(c), g, m)) g = -1;
    auto end = [&](int b, double t, bool count, uint64_t& upto) {  // as smp_end
        t = fmax(t, count ? 1.0 : 0.0);
        uint64_t sum = 0;
        int rank = 0;
        const uint64_t in = __ballot(g == b);
        for (uint64_t left = in; left != 0; left &= left - 1) {
            const int l = __ffsll((unsigned long long)left) - 1;
            const bool before = smp_lane(c, l) >= c;
            sum += before ? smp_lane(m, l) : 0;
            rank += before;
        }
        const bool passes = count ? (double)rank >= t : (double)sum > t;
        const bool passed = count ? (double)(rank - 1) >= t : (double)(sum - m) > t;
        const uint64_t here = __ballot(g == b && ((passes && !passed) || (!passes && rank == __popcll(in))));
        const int l = here ? __ffsll((unsigned long long)here) - 1 : 0;
        upto = here ? smp_lane(sum, l) : 0;
        return here ? smp_lane(c, l) : 0;
    };
    auto find = [&](double t) {  // as smp_find: bins whose running weight does not exceed t (is below all) come before
        const double all = (double)S.mass[SMP_BINS - 1];
        int n = 0;
        for (int i = 0; i < SMP_BINS; i += 64) {
            const double w = (double)S.mass[i + lane];
            n += __popcll(__ballot(all > t ? w <= t : w < all));
        }
        return n;
    };
    uint64_t upto;
    double z = z_hi;
    if (kb >= 0) {
        end(kb, (double)((uint32_t)k - (kb ? S.count[kb - 1] : 0)), true, upto);
        z = fmin(fmax(smp_before(S, kb) + (double)upto * smp_middle(kb), z_lo), z_hi);  // roundings apart it lies there
    }
    double kept = z;
    if (has_p) {
        const int b = p0 != p1 ? find(p * z) : p0;
        end(b, (p * z - smp_before(S, b)) / smp_middle(b), false, upto);
        kept = fmin(kept, smp_before(S, b) + (double)upto * smp_middle(b));
    }
    if (has_m) {  // the weights in bins m0 and m1 that reach the least one
        const double e0 = smp_middle(m0), e1 = smp_middle(m1);
        const bool reach = (g == m0 && (double)m * e0 >= floor_w) || (g == m1 && (double)m * e1 >= floor_w);
        uint64_t s0 = 0, s1 = 0;
        for (uint64_t left = __ballot(reach); left != 0; left &= left - 1) {
            const int l = __ffsll((unsigned long long)left) - 1;
            const bool first = __builtin_amdgcn_readlane(g, l) == m0;
            s0 += first ? smp_lane(m, l) : 0;
            s1 += first ? 0 : smp_lane(m, l);
        }
        kept = fmin(kept, smp_before(S, m0) + (double)s0 * e0 + (double)s1 * e1);
    }
    const double t = drawn(fmin(fmax(kept, k_lo), k_hi));
    const int b = u0 != u1 ? find(t) : u0;
    return smp_token(end(b, (t - smp_before(S, b)) / smp_middle(b), false, upto), r.vocab);
}

template <bool WIDE>
__global__ __launch_bounds__(SMP_THREADS) void sample_draw_kernel(const float* __restrict__ logits, int vocab,
                                                                  const float* __restrict__ temperature,
                                                                  const int* __restrict__ top_k,
                                                                  const float* __restrict__ top_p,
                                                                  const float* __restrict__ min_p,
                                                                  const double* __restrict__ u, int* __restrict__ tokens,
                                                                  uint8_t* scratch, int blocks, int subs) {
    __shared__ SmpShared S;
    const int row = blockIdx.y, tid = threadIdx.x, lane = tid & 63;
    const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    const SmpScratch sc = smp_scratch(scratch, row, blocks, subs);
    const float T = temperature ? temperature[row] : 1.f;
    float part[SMP_SPLIT];  // largest of each part, requested together (past the last one: the last again)
#pragma unroll
    for (int i = 0; i < SMP_SPLIT; ++i) part[i] = sc.max[min(i, blocks - 1)];
    float top = part[0];
#pragma unroll
    for (int i = 1; i < SMP_SPLIT; ++i) top = fmaxf(top, part[i]);
    SmpRow r;
    r.x = logits + (size_t)row * vocab;
    r.vocab = vocab;
    if (!(top > -INFINITY)) {  // nothing to draw from
        if (tid == 0 && blockIdx.x == 0) tokens[row] = -1;
        return;
    }
    if (!(T > 0.f)) {  // greedy: the first subset with the maximum, its first entry
        if (blockIdx.x > 0) return;
        if (tid == 0) S.n = subs;
        __syncthreads();
        for (int s = tid; s < subs; s += SMP_THREADS)
            if (sc.sub[s] == top) atomicMin(&S.n, s);
        __syncthreads();
        if (wv == 0) {
            SmpFour f = smp_load<WIDE>(r.x, vocab, S.n, lane);
            smp_cut<WIDE>(f, vocab, S.n, lane);
            int at = vocab;
#pragma unroll
            for (int e = 3; e >= 0; --e) at = f.x[e] == top ? min(at, smp_at<WIDE>(S.n, lane, e)) : at;
            for (int d = 1; d < 64; d *= 2) at = min(at, __shfl_xor(at, d, 64));
            if (lane == 0) tokens[row] = at < vocab ? at : -1;
        }
        return;
    }
    r.c = smp_scale(top, T);
    const int k = top_k ? top_k[row] : 0;
    const double uu = fmin(fmax(u[row], 0.0), 1.0);  // NaN: 0
    const double p = top_p ? (double)top_p[row] : 1.0, mp = min_p ? (double)min_p[row] : 0.0;
    const bool has_k = k > 0, has_p = p > 0.0 && p < 1.0, has_m = mp > 0.0;

    // ---- the row's bins: thread t sums bin t over the parts, all of them requested together ----
    uint64_t m = 0;
    uint32_t n = 0;
    {
        uint64_t mm[SMP_SPLIT];
        uint32_t nn[SMP_SPLIT];
        int at[SMP_SPLIT];
#pragma unroll
        for (int i = 0; i < SMP_SPLIT; ++i) {
            at[i] = i < blocks && part[i] > -INFINITY ? tid - smp_apart(r.c, part[i]) : -1;
            const size_t o = (size_t)(i < blocks ? i : 0) * SMP_BINS + max(at[i], 0);
            mm[i] = sc.mass[o];
            nn[i] = has_k ? sc.count[o] : 0;
        }
#pragma unroll
        for (int i = 0; i < SMP_SPLIT; ++i)
            if (at[i] >= 0) {
                m += mm[i];
                n += nn[i];
            }
    }
    SmpMine mine;
    {
        // whole numbers again, so that running sums do not fall and an empty bin adds nothing
        const uint64_t w = (uint64_t)rint((double)m * smp_middle(tid));
        const uint64_t sum = smp_scan<uint64_t>(w, S.wave);
        mine.before = (double)(sum - w);
        mine.with = (double)sum;
        S.mass[tid] = sum;
        if (has_k) {
            __syncthreads();
            const uint32_t c = smp_scan<uint32_t>(n, (uint32_t*)S.wave);
            S.count[tid] = c;
            if (c - n < (uint32_t)k && c >= (uint32_t)k) S.hit[0] = tid;
        }
    }
    if (tid == 0) {
        S.n = 0;
        S.n_need = 0;
        S.overflow = 0;
    }
    __syncthreads();

    // ---- in which bins the filters and the draw may end ----
    mine.all = (double)S.mass[SMP_BINS - 1];
    double z_lo = mine.all, z_hi = mine.all;  // mass of the top-k
    int kb = -1;
    if (has_k && (uint32_t)k < S.count[SMP_BINS - 1]) {
        const int g = S.hit[0];  // the first bin whose running count reaches k
        z_hi = (double)S.mass[g];
        z_lo = z_hi;
        if (S.count[g] != (uint32_t)k) {
            kb = g;
            z_lo = smp_before(S, g);
        }
    }
    int last = kb, p0 = 0, p1 = -1, m0 = 0, m1 = -1;
    double k_lo = z_lo, k_hi = z_hi;  // kept mass
    if (has_p) {
        smp_find(S, mine, p * z_lo, p * z_hi, p0, p1);
        k_lo = fmin(k_lo, smp_before(S, p0));
        k_hi = fmin(k_hi, (double)S.mass[p1]);
        last = max(last, p1);
    }
    double floor_w = 0.0;
    if (has_m) {  // bins around the least weight's
        int g = 0;
        uint64_t w = 0;
        smp_bin(r.c, top, g, w);
        floor_w = fmin(mp, 1.0) * (double)w;  // in units of 2^-44 of bin 0's middle
        // (in 32 bits: within 2e-4 of a bin, as log2 is at most 47 there)
        const float y = __log2f((float)(floor_w / SMP_ONE)) * (float)(-0.69314718055994530942 * SMP_PER_UNIT) + 0.5f;
        m0 = (int)fminf(fmaxf(floorf(y - 1e-3f), 0.f), (float)(SMP_BINS - 1));
        m1 = (int)fminf(fmaxf(floorf(y + 1e-3f), 0.f), (float)(SMP_BINS - 1));
        k_lo = fmin(k_lo, smp_before(S, m0));
        k_hi = fmin(k_hi, (double)S.mass[m1]);
        last = max(last, m1);
    }
    // the draw lies before the end of the kept mass even where u is 1
    auto drawn = [&](double mass) { return fmin(uu * mass, mass * (1.0 - 1e-15)); };
    int u0, u1;
    smp_find(S, mine, drawn(k_lo), drawn(k_hi), u0, u1);
    last = max(last, u1);
    // as ranges of values in fp32, wider than the bins by more than its roundings: what else they hold goes by bin later
    const double y_top = fma((double)top, r.c.s, SMP_ROUND) - SMP_ROUND, unit = (double)T / SMP_PER_UNIT;
    struct Range {
        float low, high;
    };
    auto want = [&](int a, int b) {
        const double lo = (y_top - (double)b - 0.5) * unit, hi = (y_top - (double)a + 0.5) * unit;
        Range w;
        w.low = a > b ? INFINITY : r.c.whole ? (float)(lo - 1e-6 * fabs(lo)) : -INFINITY;
        w.high = a > b ? -INFINITY : r.c.whole ? (float)(hi + 1e-6 * fabs(hi)) : INFINITY;
        return w;
    };
    const Range wk = want(max(kb, 0), kb), wp = want(p0, p1), wm = want(m0, m1), wu = want(u0, u1);
    // ---- collect their entries, from the subsets whose largest one is not behind the last of these bins ----
    const int s0 = (int)((long long)subs * blockIdx.x / gridDim.x), s1 = (int)((long long)subs * (blockIdx.x + 1) / gridDim.x);
    for (int s = s0 + tid; s < s1; s += SMP_THREADS) {  // (at most one a thread)
        int g;
        uint64_t w;
        if (smp_bin(r.c, sc.sub[s], g, w) && g <= last) S.need[atomicAdd(&S.n_need, 1)] = (uint16_t)s;
    }
    __syncthreads();
    const int n_need = S.n_need;
    SmpFour f[SMP_AHEAD];  // subsets a wave and round, the next round's requested ahead
    auto fetch = [&](int i, int j) {
        return smp_load<WIDE>(r.x, vocab, S.need[min(i + j * SMP_WAVES, n_need - 1)], lane);
    };
    if (n_need > 0) {
#pragma unroll
        for (int j = 0; j < SMP_AHEAD; ++j) f[j] = fetch(wv, j);
    }
    for (int i = wv; i < n_need; i += SMP_AHEAD * SMP_WAVES) {
        uint32_t in = 0;  // bit 4 j + e: entry e of subset j
#pragma unroll
        for (int j = 0; j < SMP_AHEAD; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float x = f[j].x[e];
                bool y = x >= wu.low && x <= wu.high;
                if (has_p) y = y || (x >= wp.low && x <= wp.high);
                if (kb >= 0) y = y || (x >= wk.low && x <= wk.high);
                if (has_m) y = y || (x >= wm.low && x <= wm.high);
                in |= y ? 1u << (4 * j + e) : 0u;
            }
#pragma unroll
        for (int j = 0; j < SMP_AHEAD; ++j) f[j] = fetch(i + SMP_AHEAD * SMP_WAVES, j);
#pragma unroll
        for (int j = 1; j < SMP_AHEAD; ++j)
            if (i + j * SMP_WAVES >= n_need) in &= (1u << (4 * j)) - 1;  // the last subset again
        int at = in ? atomicAdd(&S.n, __popc(in)) : 0;
        while (in) {
            const int b = __ffs(in) - 1, idx = smp_at<WIDE>(S.need[i + (b >> 2) * SMP_WAVES], lane, b & 3);
            in &= in - 1;
            if (at < SMP_LIST) S.list[at] = (uint64_t)min(idx, vocab);  // vocab: nothing
            ++at;
        }
    }
    __syncthreads();
    if (gridDim.x > 1) {  // all blocks' entries together; the last one goes on with them
        const int n = S.n;
        if (tid == 0) S.hit[0] = atomicAdd(&sc.shared[0], n);
        __syncthreads();
        const int at = S.hit[0];
        for (int i = tid; i < min(n, SMP_LIST); i += SMP_THREADS)
            if (at + i < SMP_LIST)
                __hip_atomic_store(&sc.list[at + i], (uint32_t)S.list[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        // device-coherent stores, waited for by each wave before the block is counted, and device-coherent loads by the
        // last block: no cache is written back (fences on both sides took 7 us more)
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (tid == 0) S.hit[1] = atomicAdd(&sc.shared[1], 1);
        __syncthreads();
        if (S.hit[1] != (int)gridDim.x - 1) return;
        if (tid == 0) S.n = __hip_atomic_load(&sc.shared[0], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __syncthreads();
        for (int i = tid; i < min(S.n, SMP_LIST); i += SMP_THREADS)
            S.list[i] = __hip_atomic_load(&sc.list[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    for (int i = tid; i < min(S.n, SMP_LIST); i += SMP_THREADS) {
        const int idx = (int)S.list[i];
        S.list[i] = idx < vocab ? smp_place(r.x[idx], idx) : 0;
    }
    __syncthreads();
    if (tid == 0 && S.n > SMP_LIST) S.overflow = 1;
    __syncthreads();

    // ---- end the filters, then the draw ----
    if (S.n <= 64) {  // one wave, an entry a lane, nothing to wait for
        if (wv == 0) {
            const int token = smp_end_wave(S, r, lane, kb, k, has_p, p, p0, p1, has_m, m0, m1, floor_w, z_lo, z_hi, k_lo, k_hi,
                                           u0, u1, drawn);
            if (lane == 0) tokens[row] = token;
        }
        return;
    }
    uint64_t upto;
    double z = z_hi;
    if (kb >= 0) {
        smp_end<true>(S, r, kb, (double)((uint32_t)k - (kb ? S.count[kb - 1] : 0)), upto);
        z = fmin(fmax(smp_before(S, kb) + (double)upto * smp_middle(kb), z_lo), z_hi);  // roundings apart it lies there
    }
    double kept = z;
    if (has_p) {
        int b = p0, same;
        if (p0 != p1) smp_find(S, mine, p * z, p * z, b, same);
        smp_end<false>(S, r, b, (p * z - smp_before(S, b)) / smp_middle(b), upto);
        kept = fmin(kept, smp_before(S, b) + (double)upto * smp_middle(b));
    }
    if (has_m) {  // the weights in bins m0 and m1 that reach the least one
        __syncthreads();
        if (tid < 2) S.m[tid] = 0;
        __syncthreads();
        const double e0 = smp_middle(m0), e1 = smp_middle(m1);
        smp_each(S, r, [&](uint64_t, int g, uint64_t w) {
            if ((g == m0 && (double)w * e0 >= floor_w) || (g == m1 && (double)w * e1 >= floor_w))
                atomicAdd((unsigned long long*)&S.m[g == m0 ? 0 : 1], (unsigned long long)w);
        });
        __syncthreads();
        kept = fmin(kept, smp_before(S, m0) + (double)S.m[0] * e0 + (double)S.m[1] * e1);
    }
    const double t = drawn(fmin(fmax(kept, k_lo), k_hi));
    int b = u0, same;
    if (u0 != u1) smp_find(S, mine, t, t, b, same);
    const uint64_t place = smp_end<false>(S, r, b, (t - smp_before(S, b)) / smp_middle(b), upto);
    if (tid == 0) tokens[row] = smp_token(place, vocab);
}

namespace vte {
// Blocks of a row: as many as find a CU each (their registers let one lie on a CU; 256 rows in 512 blocks 47.5 us, in 256
// 41.2 us).
static int sample_blocks(int rows) { return std::max(1, std::min(SMP_SPLIT, device_cus() / rows)); }
// Blocks that share the reading of a row, while they fit on the CUs at once: one / 16, us: 16 rows 55.6 / 30.9, one peaked
// row, of which little is read, 21.8 / 22.5.
static int draw_blocks(int rows) { return std::max(1, std::min(16, device_cus() / rows)); }

// What a call of any number of rows up to `rows` takes: fewer rows have more parts, so each number of parts at the most rows
// that have it (33 rows of 7 parts are less than 32 of 8).
long long sample_scratch_bytes(int rows) {
    long long most = 0;
    for (int b = 1; b <= SMP_SPLIT; ++b) {
        const int r = std::max(1, std::min(rows, device_cus() / b));
        most = std::max(most, (long long)r * (long long)smp_row_bytes(sample_blocks(r), (1 << SMP_IDX_BITS) / SMP_SUB));
    }
    return std::max(most, (long long)rows * (long long)smp_row_bytes(sample_blocks(rows), (1 << SMP_IDX_BITS) / SMP_SUB));
}
hipError_t sample(const float* logits, int rows, int vocab, const float* temperature, const int* top_k,
                  const float* top_p, const float* min_p, const double* u, int* tokens, void* scratch,
                  hipStream_t st) {
    const int subs = (vocab + SMP_SUB - 1) / SMP_SUB, blocks = std::min(sample_blocks(rows), subs);
    const bool wide = vocab % 4 == 0 && (reinterpret_cast<uintptr_t>(logits) & 15) == 0;
    auto bins = wide ? sample_bins_kernel<true> : sample_bins_kernel<false>;
    auto draw = wide ? sample_draw_kernel<true> : sample_draw_kernel<false>;
    hipLaunchKernelGGL(bins, dim3(blocks, rows), dim3(SMP_THREADS), 0, st, logits, vocab, temperature, top_k,
                       (uint8_t*)scratch, subs);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    const int share = std::min(draw_blocks(rows), subs);
    hipLaunchKernelGGL(draw, dim3(share, rows), dim3(SMP_THREADS), 0, st, logits, vocab, temperature, top_k, top_p, min_p, u,
                       tokens, (uint8_t*)scratch, blocks, subs);
    return hipGetLastError();
}
}  // namespace vte
