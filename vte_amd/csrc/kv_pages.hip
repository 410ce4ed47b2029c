// Append and read of the 8-bit paged KV cache (layout: kv_pages.h), gfx950.
// No counterpart in the reference, whose cache is one fp16 range per sequence
// (vte/compiler/templates/rdna/kv_cache_append.hip.template:13-39).
#include <algorithm>
#include "kv_pages.h"

// ---------------------------------------------------------------------------
// Append.  One wave writes the K or the V part of one 16-token block of one
// head, so no two waves share a block: blocks of a sequence grid.x, heads
// grid.y, sequences grid.z; wave 0 K (rotated), wave 1 V.  Behind them grid.x
// holds the blocks that rotate q.
//
// A lane holds dims (d0, d1) of a rotation pair for 16 tokens (heads of 64: 8
// tokens, the upper 32 lanes the later ones).  The block's exponent is that of
// the largest new value, and no smaller than what the block has while tokens
// before the new ones live in it; if it grows, their bytes are shifted.
// ---------------------------------------------------------------------------
struct KvRope {
    const __half *cosc, *sinc;
    int rows, type, dim;  // table rows, rotation type (as rope_kernel), its dims
};

// Dims of pair i of a head, and whether the pair rotates.
template <int HD>
__device__ __forceinline__ bool kvp_pair(int i, const KvRope& rp, int& d0, int& d1) {
    if (rp.type == 1) {
        d0 = 2 * i;
        d1 = 2 * i + 1;
    } else if (rp.type == 2) {
        const int hr = rp.dim / 2;
        d0 = i < hr ? i : 2 * i;
        d1 = i < hr ? i + hr : 2 * i + 1;
        return i < hr;
    } else {
        d0 = i;
        d1 = i + HD / 2;
    }
    return true;
}
// The products and the sum are rounded one by one, as separate operations round
// them: a contracted form could move a value over the border between two codes.
__device__ __forceinline__ void kvp_rotate(float& a, float& b, float c, float s) {
#pragma clang fp contract(off)
    const float x = a, y = b;
    const float xc = x * c, ys = y * s, xs = x * s, yc = y * c;
    a = xc - ys;
    b = xs + yc;
}

template <typename T, int HD>
__global__ __launch_bounds__(128) void kv_pages_append_kernel(KvPages c, KvRows r, KvRope rp, const T* __restrict__ k,
                                                              const T* __restrict__ v, const T* q, T* q_out, int n_q,
                                                              long long k_stride, long long v_stride,
                                                              long long q_stride, int seq_blocks) {
    constexpr int NP = HD / 2;           // pairs of a head
    constexpr int TOK = KVP_BLOCK * NP / 64;  // tokens a lane holds
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    const int cap = kvp_capacity(c, r);
    const int limit = rp.cosc != nullptr ? min(cap, rp.rows) : cap;  // positions from here on are dropped
    const int tab = rp.type == 2 ? rp.dim : HD;                      // row of a table

    if ((int)blockIdx.x >= seq_blocks) {  // q: one pair a thread
        const int per_row = n_q * NP;
        const long long gid =
            ((long long)(blockIdx.x - seq_blocks) + (long long)(gridDim.x - seq_blocks) *
             (blockIdx.y + (long long)gridDim.y * blockIdx.z)) * 128 + threadIdx.x;
        const int row = (int)(gid / per_row), h = (int)(gid % per_row) / NP, i = (int)(gid % NP);
        if (row >= r.rows) return;
        const int b = kvp_row_seq(r, row);
        if (b < 0) return;
        const KvSeq s = kvp_seq(r, b);
        const int at = row - s.first;
        if (at < 0 || at >= s.n || s.pos >= limit - at) return;
        const int pos = s.pos + at;
        int d0, d1;
        const bool turns = kvp_pair<HD>(i, rp, d0, d1);
        const T* src = q + row * q_stride + h * HD;
        float x = ld_act<T>(src + d0), y = ld_act<T>(src + d1);
        if (turns) kvp_rotate(x, y, h2f(rp.cosc[(size_t)pos * tab + i]), h2f(rp.sinc[(size_t)pos * tab + i]));
        T* dst = q_out + ((size_t)row * n_q + h) * HD;
        st_act<T>(dst + d0, x);
        st_act<T>(dst + d1, y);
        return;
    }

    const int b = blockIdx.z, h = blockIdx.y;
    const KvSeq s = kvp_seq(r, b);
    if (s.n == 0 || s.pos >= limit) return;
    const int t_end = s.n < limit - s.pos ? s.pos + s.n : limit;   // new positions [s.pos, t_end)
    const int blk = s.pos / KVP_BLOCK + blockIdx.x, t0 = blk * KVP_BLOCK;
    if (t0 >= t_end) return;
    const int page = kvp_page(c, r, b, t0 >> c.page_log2);
    if (page < 0) return;
    const int j0 = max(s.pos - t0, 0), j1 = min(t_end - t0, KVP_BLOCK);  // new places of the block
    const int in_page = blk & ((1 << (c.page_log2 - 4)) - 1);
    const size_t at = (((size_t)page * c.n_kv + h) << (c.page_log2 - 4)) + in_page;  // the block's place in the cache
    const bool is_v = wv != 0;
    int8_t* exps = is_v ? c.v_exp : c.k_exp;
    uint8_t* codes = (is_v ? c.v : c.k) + at * (KVP_BLOCK * HD);

    const int i = lane & (NP - 1), jb = (lane / NP) * TOK;  // pair, first place
    int d0, d1;
    const bool turns = kvp_pair<HD>(i, rp, d0, d1) && !is_v && rp.cosc != nullptr;
    const T* src = (is_v ? v : k) + (long long)(s.first + t0 - s.pos) * (is_v ? v_stride : k_stride) + h * HD;
    const long long stride = is_v ? v_stride : k_stride;
    float x[TOK], y[TOK];
    float amax = 0.f;
    bool bad = false;
#pragma unroll
    for (int j = 0; j < TOK; ++j) {
        const int p = jb + j;
        const bool in = p >= j0 && p < j1;
        x[j] = in ? ld_act<T>(src + p * stride + d0) : 0.f;
        y[j] = in ? ld_act<T>(src + p * stride + d1) : 0.f;
    }
#pragma unroll
    for (int j = 0; j < TOK; ++j) {
        const int p = jb + j;
        if (turns && p >= j0 && p < j1) {
            const size_t row = (size_t)(t0 + p) * tab + i;
            kvp_rotate(x[j], y[j], h2f(rp.cosc[row]), h2f(rp.sinc[row]));
        }
        bad = bad || !(fabsf(x[j]) < INFINITY) || !(fabsf(y[j]) < INFINITY);
        amax = fmaxf(amax, fmaxf(fabsf(x[j]), fabsf(y[j])));
    }
    amax = wave_max(amax);
    const int e_old = j0 > 0 ? exps[at] : KVP_E_MIN;
    int e = KVP_E_NAN;
    if (!__any(bad) && e_old != KVP_E_NAN) e = max(e_old, kvp_exponent(amax));
    const float inv = e == KVP_E_NAN ? 0.f : ldexpf(1.f, -e);
    const int shift = e - e_old;  // > 0: the old bytes move
    if (lane == 0) exps[at] = (int8_t)e;
    const bool move = j0 > 0 && e != KVP_E_NAN && shift > 0;
#pragma unroll
    for (int j = 0; j < TOK; ++j) {
        const int p = jb + j;
        const bool in = p >= j0 && p < j1;
        if (!in && !(move && p < j0)) continue;
        uint8_t* a0 = is_v ? codes + d0 * KVP_BLOCK + p : codes + p * HD + d0;
        uint8_t* a1 = is_v ? codes + d1 * KVP_BLOCK + p : codes + p * HD + d1;
        if (in) {
            *a0 = e == KVP_E_NAN ? KVP_ZERO : (uint8_t)kvp_code(x[j], inv);
            *a1 = e == KVP_E_NAN ? KVP_ZERO : (uint8_t)kvp_code(y[j], inv);
        } else {
            *a0 = (uint8_t)(__float2int_rn(ldexpf((float)((int)*a0 - KVP_ZERO), -shift)) + KVP_ZERO);
            *a1 = (uint8_t)(__float2int_rn(ldexpf((float)((int)*a1 - KVP_ZERO), -shift)) + KVP_ZERO);
        }
    }
}

// ---------------------------------------------------------------------------
// Read: rows 0 .. end - 1 of every sequence as T [batch][out_rows][n_kv][HD].
// One block of threads per (16-token block, sequence); a thread takes (token,
// dim) values of every head.
// ---------------------------------------------------------------------------
template <typename T, int HD>
__global__ __launch_bounds__(256) void kv_pages_read_kernel(KvPages c, KvRows r, T* __restrict__ k_out,
                                                            T* __restrict__ v_out, int out_rows) {
    const int b = blockIdx.y, blk = blockIdx.x, t0 = blk * KVP_BLOCK;
    const KvSeq s = kvp_seq(r, b);
    if (s.pos < 0) return;
    const int cap = min(kvp_capacity(c, r), out_rows);
    const int end = s.n < cap - s.pos ? s.pos + s.n : cap;
    if (t0 >= end) return;
    const int page = kvp_page(c, r, b, t0 >> c.page_log2);
    const int in_page = blk & ((1 << (c.page_log2 - 4)) - 1);
    for (int i = threadIdx.x; i < c.n_kv * KVP_BLOCK * HD; i += 256) {
        const int d = i % HD, h = i / HD % c.n_kv, p = i / (HD * c.n_kv);
        if (t0 + p >= end) break;
        float kv = 0.f, vv = 0.f;
        if (page >= 0) {
            const size_t at = (((size_t)page * c.n_kv + h) << (c.page_log2 - 4)) + in_page;
            kv = ((int)c.k[at * (KVP_BLOCK * HD) + p * HD + d] - KVP_ZERO) * kvp_scale(c.k_exp[at]);
            vv = ((int)c.v[at * (KVP_BLOCK * HD) + d * KVP_BLOCK + p] - KVP_ZERO) * kvp_scale(c.v_exp[at]);
        }
        const size_t o = (((size_t)b * out_rows + t0 + p) * c.n_kv + h) * HD + d;
        st_act<T>(k_out + o, kv);
        st_act<T>(v_out + o, vv);
    }
}

// ---------------------------------------------------------------------------
// Host launchers
// ---------------------------------------------------------------------------
namespace vte {

template <typename T, int HD>
static hipError_t append_hd(const KvPages& c, const KvRows& r, const KvRope& rp, const void* k, const void* v,
                            const void* q, void* q_out, int n_q, long long ks, long long vs, long long qs,
                            hipStream_t st) {
    // a run of max_rows tokens touches at most this many blocks of 16
    const int seq_blocks = r.max_rows == 1 ? 1 : (r.max_rows + KVP_BLOCK - 1) / KVP_BLOCK + 1;
    const long long grid_yz = (long long)c.n_kv * r.batch;
    const long long q_blocks = q ? ((long long)r.rows * n_q * (HD / 2) + 127) / 128 : 0;
    const int qx = (int)((q_blocks + grid_yz - 1) / grid_yz);
    hipLaunchKernelGGL((kv_pages_append_kernel<T, HD>), dim3(seq_blocks + qx, c.n_kv, r.batch), dim3(128), 0, st, c, r,
                       rp, (const T*)k, (const T*)v, (const T*)q, (T*)q_out, n_q, ks, vs, qs, seq_blocks);
    return hipGetLastError();
}
hipError_t kv_pages_append(const KvPages& c, const KvRows& r, int hd, bool f16, const void* k, const void* v,
                           const void* q, void* q_out, int n_q, long long ks, long long vs, long long qs,
                           const void* cosc, const void* sinc, int rope_rows, int rope_type, int rotary_dim,
                           hipStream_t st) {
    const KvRope rp{(const __half*)cosc, (const __half*)sinc, rope_rows, rope_type, rotary_dim};
#define KVP_APPEND(T, HD) append_hd<T, HD>(c, r, rp, k, v, q, q_out, n_q, ks, vs, qs, st)
    if (hd == 128) return f16 ? KVP_APPEND(__half, 128) : KVP_APPEND(float, 128);
    return f16 ? KVP_APPEND(__half, 64) : KVP_APPEND(float, 64);
#undef KVP_APPEND
}

template <typename T, int HD>
static hipError_t read_hd(const KvPages& c, const KvRows& r, void* k_out, void* v_out, int out_rows, hipStream_t st) {
    const int rows = (int)std::min<long long>(out_rows, (long long)r.max_pages << c.page_log2);
    hipLaunchKernelGGL((kv_pages_read_kernel<T, HD>), dim3((rows + KVP_BLOCK - 1) / KVP_BLOCK, r.batch), dim3(256), 0,
                       st, c, r, (T*)k_out, (T*)v_out, out_rows);
    return hipGetLastError();
}
hipError_t kv_pages_read(const KvPages& c, const KvRows& r, int hd, bool f16, void* k_out, void* v_out, int out_rows,
                         hipStream_t st) {
    if (hd == 128)
        return f16 ? read_hd<__half, 128>(c, r, k_out, v_out, out_rows, st)
                   : read_hd<float, 128>(c, r, k_out, v_out, out_rows, st);
    return f16 ? read_hd<__half, 64>(c, r, k_out, v_out, out_rows, st)
               : read_hd<float, 64>(c, r, k_out, v_out, out_rows, st);
}

}  // namespace vte
