// Norm of a head and its rotation by position, shared by the kernels that write q
// and k (qk_norm.hip, the append of kv_pages.hip), gfx950.
//
//   y = x w / sqrt(mean(x^2) + eps), then of the first `rot` dims pair i = (a, b)
//   becomes A (a cos t - b sin t, a sin t + b cos t), t = position * freq[i].
//
// No tables: far positions would need long ones, and fp16 ones hold a cosine to
// 2^-12 only.  The angle is formed in 64 bits (a position of 2^20 times a frequency
// near 1 leaves 2^-32 of a turn of error; in 32 bits it would be 2^-5), reduced to
// within half a quarter turn there, and the rest is two short polynomials in fp32.
#pragma once
#include "vte_common.h"

struct HeadForm {
    const __half *q_norm, *k_norm;  // null: not normed
    const double* freq;             // radians a position; null: no rotation
    float eps, amplitude;
    int rot, inter;                 // dims that rotate; whether pairs are neighbours (else half of `rot` apart)
};

// Eight consecutive elements.
template <typename T>
__device__ __forceinline__ void kvp_ld8(const T* p, float (&v)[8]) {
    if constexpr (sizeof(T) == 2) {
        const uint4 t = *reinterpret_cast<const uint4*>(p);
        const uint32_t w[4] = {t.x, t.y, t.z, t.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = h2f_bits(w[i]);
            v[2 * i + 1] = h2f_bits(w[i] >> 16);
        }
    } else {
        const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
        v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    }
}
template <typename T>
__device__ __forceinline__ void kvp_st8(T* p, const float (&v)[8]) {
    if constexpr (sizeof(T) == 2) {
        union {
            __half h[8];
            uint4 u;
        } r;
#pragma unroll
        for (int i = 0; i < 8; ++i) r.h[i] = __float2half(v[i]);
        *reinterpret_cast<uint4*>(p) = r.u;
    } else {
        reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
        reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
    }
}

// amplitude * (cos, sin) of position * freq, with `turns` = freq / (2 pi).  The angle in quarter turns is n + r, |r| <= 1/2;
// Taylor series of sin(pi/2 r) and cos(pi/2 r) to r^9 and r^10 (what is left out is below 2^-28 of either).
__device__ __forceinline__ double ht_turns(double freq) { return freq * 0.15915494309189533577; }
__device__ __forceinline__ void ht_angle(double position, double turns, float amplitude, float& c, float& s) {
    double t = position * turns;
    t = 4.0 * (t - rint(t));
    const double n = rint(t);
    const float r = (float)(t - n), x = r * r;
    const float sn = r * fmaf(fmaf(fmaf(fmaf(1.60441185e-4f, x, -4.68175414e-3f), x, 7.96926262e-2f), x, -6.45964098e-1f), x,
                              1.57079633f);
    const float cs = fmaf(fmaf(fmaf(fmaf(fmaf(-2.52020424e-5f, x, 9.19260274e-4f), x, -2.08634807e-2f), x, 2.53669508e-1f), x,
                               -1.23370055f), x, 1.f);
    const int q = (int)n;  // -2 .. 2
    c = (q & 1 ? sn : cs) * ((q + 1) & 2 ? -amplitude : amplitude);
    s = (q & 1 ? cs : sn) * (q & 2 ? -amplitude : amplitude);
}
__device__ __forceinline__ void ht_turn(float& a, float& b, float c, float s) {
    const float x = a, y = b;
    a = fmaf(x, c, -(y * s));
    b = fmaf(x, s, y * c);
}

// N consecutive elements, 8 or 4.
template <typename T, int N>
__device__ __forceinline__ void ht_ld(const T* p, float (&v)[N]) {
    if constexpr (N == 8) {
        kvp_ld8(p, v);
    } else {
        static_assert(N == 4 && sizeof(T) == 4, "");
        const float4 a = *reinterpret_cast<const float4*>(p);
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    }
}
template <typename T, int N>
__device__ __forceinline__ void ht_st(T* p, const float (&v)[N]) {
    if constexpr (N == 8) kvp_st8(p, v);
    else *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
}

// ---- Two runs of V dims a thread: HD / (2 V) neighbouring lanes hold a head.  Needs rot % (2 V) = 0 or neighbouring pairs.
// A run of the neighbouring lane begins where the lane's ends, so that a load touches whole lines.
template <int HD, int V>
__device__ __forceinline__ void ht_runs(const HeadForm& f, int u, int& d0, int& d1) {
    const int n = f.inter ? 0 : f.rot;  // dims whose pairs lie half of them apart
    d0 = V * u;
    d1 = d0 + (V * u < n / 2 ? n : HD) / 2;
    if (d0 >= n / 2) d0 += n / 2;  // (behind them the rest in two halves: d1 - d0 = (HD - n) / 2)
}
// Sum over N neighbouring lanes (4, 8, 16 or 32).
template <int N>
__device__ __forceinline__ float ht_sum(float v) {
    v += VTE_DPP_F(v, 0xB1);
    v += VTE_DPP_F(v, 0x4E);
    if constexpr (N >= 8) v += VTE_DPP_F(v, 0x141);
    if constexpr (N >= 16) v += VTE_DPP_F(v, 0x140);
    if constexpr (N >= 32) v += __shfl_xor(v, 16, 64);
    return v;
}
template <int HD, int V>
__device__ __forceinline__ void ht_norm(const __half* w, float eps, int d0, int d1, float (&x)[V], float (&y)[V]) {
    __half a[V], b[V];
    if constexpr (V == 8) {
        *reinterpret_cast<uint4*>(a) = *reinterpret_cast<const uint4*>(w + d0);
        *reinterpret_cast<uint4*>(b) = *reinterpret_cast<const uint4*>(w + d1);
    } else {
        *reinterpret_cast<uint2*>(a) = *reinterpret_cast<const uint2*>(w + d0);
        *reinterpret_cast<uint2*>(b) = *reinterpret_cast<const uint2*>(w + d1);
    }
    float sum = 0.f;
#pragma unroll
    for (int e = 0; e < V; ++e) sum = fmaf(x[e], x[e], fmaf(y[e], y[e], sum));
    const float inv = rsqrtf(ht_sum<HD / (2 * V)>(sum) * (1.f / HD) + eps);
#pragma unroll
    for (int e = 0; e < V; ++e) {
        x[e] *= inv * h2f(a[e]);
        y[e] *= inv * h2f(b[e]);
    }
}
// Cosines and sines of a block's rows, once for all their heads: turn[row][pair], rows at positions pos(row).  (By each
// thread for its own eight pairs they cost as much time as the bytes: see the kernels.)  A thread keeps to one pair,
// whose frequency it asks for before the positions are there.
template <int NT>
struct HtPair {
    int row, pair, step;  // its first row, and the rows between its rows
    double freq;
    __device__ __forceinline__ explicit HtPair(const HeadForm& f) : row(0), pair(0), step(0), freq(0.) {
        if (f.freq == nullptr) return;
        const int pairs = f.rot / 2, tid = threadIdx.x;
        step = NT / pairs;
        row = tid / pairs;
        pair = tid - row * pairs;
        if (row < step) freq = f.freq[pair];
    }
    template <int NP, class Pos>
    __device__ __forceinline__ void fill(const HeadForm& f, float2 (*turn)[NP], int rows, Pos pos) const {
        if (row >= step) return;
        const double turns = ht_turns(freq);
        for (int r = row; r < rows; r += step) {
            float2 t;
            ht_angle((double)pos(r), turns, f.amplitude, t.x, t.y);
            turn[r][pair] = t;
        }
    }
};
// A barrier for what stands in LDS only: loads from memory stay under way.
__device__ __forceinline__ void ht_barrier() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}
// (Pairs that do not rotate are left alone: times 0 an infinite neighbour would make NaN of them.)
template <int V>
__device__ __forceinline__ void ht_turn_runs(const HeadForm& f, int d0, int d1, const float2* turn, float (&x)[V], float (&y)[V]) {
    if (f.inter) {  // each run holds pairs
#pragma unroll
        for (int e = 0; e < V; e += 2) {
            if (d0 + e < f.rot) ht_turn(x[e], x[e + 1], turn[(d0 + e) / 2].x, turn[(d0 + e) / 2].y);
            if (d1 + e < f.rot) ht_turn(y[e], y[e + 1], turn[(d1 + e) / 2].x, turn[(d1 + e) / 2].y);
        }
    } else if (d0 < f.rot / 2) {
#pragma unroll
        for (int e = 0; e < V; ++e) ht_turn(x[e], y[e], turn[d0 + e].x, turn[d0 + e].y);
    }
}

// ---- one pair a thread: any rotation.
// Dims of pair i of a head, and whether it rotates.
__device__ __forceinline__ bool ht_pair(const HeadForm& f, int i, int& d0, int& d1) {
    const bool turns = f.freq != nullptr && i < f.rot / 2;
    if (turns && !f.inter) {
        d0 = i;
        d1 = i + f.rot / 2;
    } else {
        d0 = 2 * i;
        d1 = 2 * i + 1;
    }
    return turns;
}
// Sum over N neighbouring lanes (32 or 64).
template <int N>
__device__ __forceinline__ float ht_sum_lanes(float v) {
#pragma unroll
    for (int d = 1; d < N; d <<= 1) v += __shfl_xor(v, d, 64);
    return v;
}
