// Queries and keys normed head by head and rotated by their positions (head_turn.h), gfx950.
// The reference has the two steps apart, for heads that are not normed:
// vte/compiler/templates/rdna/rope.hip.template:17-137.
#include "head_turn.h"
#include "launch.h"

// q and k of one call: rows of heads.
template <typename T>
struct QkRows {
    const T* x;
    T* y;
    int heads;
    long long in, out;  // elements between rows
};

// A thread takes two 16-byte runs of a head; q heads of a row, then its k heads.  A block's rows share their cosines and
// sines.
//
// A value is read once and written once: bound by bytes where there are many rows, 134 MB of 4096 fp32 rows of 32 heads of
// 128 in 27.7 to 28.7 us, 4.7 to 4.8 TB/s (a large copy reaches 5.1 to 5.2; 24 where two inputs take turns, which the
// memory-side cache holds in part), by latency where there are few (one row 2.6 to 2.9 us).  With cosines by each thread 39.1, with a thread's dims side by side (half a line a load
// in fp32) 33.5; stores past the caches, of which such a load's are parts of lines, took 84.
template <typename T, int HD>
__global__ __launch_bounds__(256) void qk_norm_rope_kernel(HeadForm f, QkRows<T> q, QkRows<T> k, int rows,
                                                           const int* __restrict__ positions) {
    constexpr int V = 16 / sizeof(T), NU = HD / (2 * V), HEADS = vte::qk_norm_heads(true, HD, sizeof(T));
    static_assert(HEADS * NU == 256, "");
    __shared__ __align__(16) float2 turn[HEADS][HD / 2];
    __shared__ int pos_sh[HEADS];
    const int heads = q.heads + k.heads, tid = threadIdx.x, u = tid % NU;
    const int first = (blockIdx.x + gridDim.x * blockIdx.y) * HEADS, all = rows * heads;  // (2^27 at most, and a row of blocks more)
    if (first >= all) return;
    const bool in = first + tid / NU < all;
    const int item = in ? first + tid / NU : first;
    const int row0 = first / heads, row_n = (min(first + HEADS, all) - 1) / heads - row0 + 1;
    const int row = item / heads, hh = item - row * heads;
    const bool is_q = hh < q.heads;
    const int h = is_q ? hh : hh - q.heads;
    const QkRows<T>& r = is_q ? q : k;
    const T* src = r.x + row * r.in + h * HD;
    T* dst = r.y + row * r.out + h * HD;
    const HtPair<256> mine(f);
    int d0, d1;
    ht_runs<HD, V>(f, u, d0, d1);
    float x[V], y[V];
    ht_ld(src + d0, x);
    ht_ld(src + d1, y);
    if (positions != nullptr) {
        if (tid < row_n) pos_sh[tid] = positions[row0 + tid];
        ht_barrier();
        if (f.freq != nullptr) {
            mine.fill(f, turn, row_n, [&](int i) { return pos_sh[i]; });
            ht_barrier();
        }
        if (pos_sh[row - row0] < 0) return;
    }
    if (!in) return;
    const __half* w = is_q ? f.q_norm : f.k_norm;
    if (w != nullptr) ht_norm<HD, V>(w, f.eps, d0, d1, x, y);
    if (f.freq != nullptr) ht_turn_runs<V>(f, d0, d1, turn[row - row0], x, y);
    ht_st(dst + d0, x);
    ht_st(dst + d1, y);
}

// Any alignment and rotation: a wave takes a head, a lane one pair of dims (heads of 256: two).  Values are loaded one by
// one and every head forms its row's angles again, which bound it: 4096 rows of 32 heads of 128, the first 40 dims rotated in
// halves (fp32: 20), 38.7 us fp16 and 41.6 fp32, against 13.8 and 22.9 of the kernel above with 64 (two inputs in turn).
template <typename T, int HD>
__global__ __launch_bounds__(256) void qk_norm_rope_pairs_kernel(HeadForm f, QkRows<T> q, QkRows<T> k, int rows,
                                                                 const int* __restrict__ positions) {
    constexpr int NP = HD / 2, EACH = NP > 64 ? NP / 64 : 1;
    const int heads = q.heads + k.heads, lane = threadIdx.x & 63;
    const int item = (blockIdx.x + gridDim.x * blockIdx.y) * 4 + (threadIdx.x >> 6);
    if (item >= rows * heads) return;  // (2^27 at most, and a row of blocks more)
    const int row = item / heads, hh = item - row * heads;
    const int pos = positions != nullptr ? positions[row] : 0;
    if (pos < 0) return;
    const bool is_q = hh < q.heads;
    const int h = is_q ? hh : hh - q.heads;
    const QkRows<T>& r = is_q ? q : k;
    const T* src = r.x + row * r.in + h * HD;
    T* dst = r.y + row * r.out + h * HD;
    const __half* w = is_q ? f.q_norm : f.k_norm;
    float a[EACH], b[EACH], sum = 0.f;
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
        a[e] = b[e] = 0.f;
        if (lane < NP) {
            int d0, d1;
            ht_pair(f, lane + 64 * e, d0, d1);
            a[e] = ld_act<T>(src + d0);
            b[e] = ld_act<T>(src + d1);
        }
        sum = fmaf(a[e], a[e], fmaf(b[e], b[e], sum));
    }
    sum = wave_sum(sum);
    const float inv = rsqrtf(sum * (1.f / HD) + f.eps);
    if (lane >= NP) return;
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
        int d0, d1;
        const bool turns = ht_pair(f, lane + 64 * e, d0, d1);
        if (w != nullptr) {
            a[e] *= inv * h2f(w[d0]);
            b[e] *= inv * h2f(w[d1]);
        }
        if (turns) {
            float c, s;
            ht_angle((double)pos, ht_turns(f.freq[lane + 64 * e]), f.amplitude, c, s);
            ht_turn(a[e], b[e], c, s);
        }
        st_act<T>(dst + d0, a[e]);
        st_act<T>(dst + d1, b[e]);
    }
}

namespace vte {

template <typename T, int HD>
static hipError_t norm_hd(const HeadForm& f, const void* q, void* q_out, int n_q, long long qs, const void* k, void* k_out,
                          int n_kv, long long ks, int rows, const int* positions, hipStream_t st) {
    const QkRows<T> Q{(const T*)q, (T*)q_out, n_q, qs, q == q_out ? qs : (long long)n_q * HD};
    const QkRows<T> K{(const T*)k, (T*)k_out, n_kv, ks, k == k_out ? ks : (long long)n_kv * HD};
    auto fits = [](const void* p, long long stride) {
        return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && stride * (long long)sizeof(T) % 16 == 0;
    };
    const bool wide = fits(q, qs) && fits(q_out, 0) && fits(k, ks) && fits(k_out, 0) && fits(f.q_norm, 0) &&
                      fits(f.k_norm, 0) && (f.freq == nullptr || f.inter || f.rot % (32 / (int)sizeof(T)) == 0);
    const long long items = (long long)rows * (n_q + n_kv), per = qk_norm_heads(wide, HD, sizeof(T));
    const BlockGrid g = block_grid((items + per - 1) / per);
    if (wide)
        hipLaunchKernelGGL((qk_norm_rope_kernel<T, HD>), dim3(g.x, g.y), dim3(256), 0, st, f, Q, K, rows, positions);
    else
        hipLaunchKernelGGL((qk_norm_rope_pairs_kernel<T, HD>), dim3(g.x, g.y), dim3(256), 0, st, f, Q, K, rows, positions);
    return hipGetLastError();
}
hipError_t qk_norm_rope(const HeadForm& f, int hd, bool f16, const void* q, void* q_out, int n_q, long long qs, const void* k,
                        void* k_out, int n_kv, long long ks, int rows, const int* positions, hipStream_t st) {
#define QK_NORM(T, HD) norm_hd<T, HD>(f, q, q_out, n_q, qs, k, k_out, n_kv, ks, rows, positions, st)
    if (hd == 64) return f16 ? QK_NORM(__half, 64) : QK_NORM(float, 64);
    if (hd == 128) return f16 ? QK_NORM(__half, 128) : QK_NORM(float, 128);
    return f16 ? QK_NORM(__half, 256) : QK_NORM(float, 256);
#undef QK_NORM
}

}  // namespace vte
