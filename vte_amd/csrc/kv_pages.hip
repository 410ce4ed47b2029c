// Append and read of the 8-bit paged KV cache (layout: kv_pages.h), gfx950.
// No counterpart in the reference, whose cache is one fp16 range per sequence
// (vte/compiler/templates/rdna/kv_cache_append.hip.template:13-39).
#include <algorithm>
#include "kv_pages.h"

// ---------------------------------------------------------------------------
// Append.  One block of threads writes one 16-token block of one head, K and V
// (blocks of a sequence grid.x, heads grid.y, sequences grid.z); behind them
// grid.x holds the blocks that rotate q.  A block's exponent is that of the
// largest new value, and no smaller than what the block has while tokens before
// the new ones live in it; if it grows, their bytes are shifted.
//
// WIDE: rows and tables 16-byte aligned and every pair rotates (rope_type 0, 1 or
// none).  HD threads take K, each 8 rotation pairs of one token, HD threads V,
// each 16 dims of one token, whose bytes change places in LDS.  Otherwise one wave
// takes K and one V, a lane holding one pair of dims for all 16 tokens (heads of
// 64: 8 tokens, the upper 32 lanes the later ones): 2-byte loads and single bytes
// stored, but any alignment and the partial rotation.
//
// A value is read once and a byte written once; a block of the cache is whole in
// its block of threads because the scale needs its largest value first.  Few tokens:
// a launch and four loads in a row (position, page, old exponent and bytes), 3.7 us
// for one token.  Prompts: bytes, 41 MB of four chunks of 700 to 2048 tokens with
// their q in 10.7 us, 3.9 TB/s (a large copy reaches 5.0).  With the read-back of the
// chunks, us: 14.7 WIDE, 44.0 otherwise; one token each of 64 sequences 12.6 / 13.9.
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

// Eight bytes to the left of a grown scale: rounded shifts of the whole numbers.
__device__ __forceinline__ uint32_t kvp_shift4(uint32_t w, float f) {
    uint32_t r = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) r |= kvp_code((float)((int)(w >> (8 * i) & 0xFFu) - KVP_ZERO), f) << (8 * i);
    return r;
}
__device__ __forceinline__ uint2 kvp_code8(const float (&v)[8], float inv) {
    uint2 r = make_uint2(0, 0);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        r.x |= kvp_code(v[i], inv) << (8 * i);
        r.y |= kvp_code(v[4 + i], inv) << (8 * i);
    }
    return r;
}

template <typename T, int HD, bool WIDE>
__global__ __launch_bounds__(WIDE ? 2 * HD : 128) void kv_pages_append_kernel(KvPages c, KvRows r, KvRope rp, const T* __restrict__ k,
                                                              const T* __restrict__ v, const T* q, T* q_out, int n_q,
                                                              long long k_stride, long long v_stride,
                                                              long long q_stride, int seq_blocks) {
    constexpr int NP = HD / 2;           // pairs of a head
    constexpr int TOK = KVP_BLOCK * NP / 64;  // tokens a lane holds
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    const int cap = kvp_capacity(c, r);
    const int limit = rp.cosc != nullptr ? min(cap, rp.rows) : cap;  // positions from here on are dropped
    const int tab = rp.type == 2 ? rp.dim : HD;                      // row of a table

    if ((int)blockIdx.x >= seq_blocks) {  // q: one pair a thread, or eight
        constexpr int NU = WIDE ? NP / 8 : NP;
        const int per_row = n_q * NU;
        const long long gid =
            ((long long)(blockIdx.x - seq_blocks) + (long long)(gridDim.x - seq_blocks) *
             (blockIdx.y + (long long)gridDim.y * blockIdx.z)) * (WIDE ? 2 * HD : 128) + threadIdx.x;
        if (gid >= (long long)r.rows * per_row) return;
        const int row = (int)(gid / per_row), hu = (int)(gid - (long long)row * per_row), h = hu / NU, i = hu % NU;
        const int b = kvp_row_seq(r, row);
        if (b < 0) return;
        const KvSeq s = kvp_seq(r, b);
        const int at = row - s.first;
        if (at < 0 || at >= s.n || s.pos >= limit - at) return;
        const int pos = s.pos + at;
        const T* src = q + row * q_stride + h * HD;
        T* dst = q_out + ((size_t)row * n_q + h) * HD;
        if constexpr (WIDE) {
            const int d0 = rp.type == 1 ? 16 * i : 8 * i, d1 = rp.type == 1 ? 16 * i + 8 : 8 * i + NP;
            float x[8], y[8], c8[8], s8[8];
            kvp_ld8(src + d0, x);
            kvp_ld8(src + d1, y);
            kvp_ld8(rp.cosc + (size_t)pos * HD + 8 * i, c8);
            kvp_ld8(rp.sinc + (size_t)pos * HD + 8 * i, s8);
            if (rp.type == 1) {  // pairs lie side by side: x holds the first four of them, y the others
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    kvp_rotate(x[2 * e], x[2 * e + 1], c8[e], s8[e]);
                    kvp_rotate(y[2 * e], y[2 * e + 1], c8[4 + e], s8[4 + e]);
                }
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) kvp_rotate(x[e], y[e], c8[e], s8[e]);
            }
            kvp_st8(dst + d0, x);
            kvp_st8(dst + d1, y);
        } else {
            int d0, d1;
            const bool turns = kvp_pair<HD>(i, rp, d0, d1);
            float x = ld_act<T>(src + d0), y = ld_act<T>(src + d1);
            if (turns) kvp_rotate(x, y, h2f(rp.cosc[(size_t)pos * tab + i]), h2f(rp.sinc[(size_t)pos * tab + i]));
            st_act<T>(dst + d0, x);
            st_act<T>(dst + d1, y);
        }
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
    const bool is_v = WIDE ? (int)threadIdx.x >= HD : wv != 0;
    int8_t* exps = is_v ? c.v_exp : c.k_exp;
    uint8_t* codes = (is_v ? c.v : c.k) + at * (KVP_BLOCK * HD);
    const int e_old = j0 > 0 ? exps[at] : KVP_E_MIN;

    if constexpr (WIDE) {
        __shared__ float top[4];
        __shared__ int odd[4];
        __shared__ __align__(16) uint8_t turned[HD][KVP_BLOCK];  // V: a dim's tokens together
        const int id = threadIdx.x % HD, i = id % (HD / 16), p = id / (HD / 16);  // unit of 16 dims, place
        const bool in = p >= j0 && p < j1, old = p < j0;
        const int d0 = is_v || rp.type == 1 ? 16 * i : 8 * i, d1 = is_v || rp.type == 1 ? 16 * i + 8 : 8 * i + NP;
        float x[8], y[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = y[e] = 0.f;
        if (in) {
            const T* src = (is_v ? v + (s.first + t0 - s.pos + p) * v_stride : k + (s.first + t0 - s.pos + p) * k_stride) +
                           h * HD;
            kvp_ld8(src + d0, x);
            kvp_ld8(src + d1, y);
            if (!is_v && rp.cosc != nullptr) {
                float c8[8], s8[8];
                kvp_ld8(rp.cosc + (size_t)(t0 + p) * HD + 8 * i, c8);
                kvp_ld8(rp.sinc + (size_t)(t0 + p) * HD + 8 * i, s8);
                if (rp.type == 1) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        kvp_rotate(x[2 * e], x[2 * e + 1], c8[e], s8[e]);
                        kvp_rotate(y[2 * e], y[2 * e + 1], c8[4 + e], s8[4 + e]);
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e) kvp_rotate(x[e], y[e], c8[e], s8[e]);
                }
            }
        }
        // old tokens' bytes: K this thread's own, V those of dim id
        uint2 k0 = make_uint2(0, 0), k1 = k0;
        uint4 v0 = make_uint4(0, 0, 0, 0);
        if (j0 > 0 && is_v) v0 = *reinterpret_cast<const uint4*>(codes + id * KVP_BLOCK);
        if (old && !is_v) {
            k0 = *reinterpret_cast<const uint2*>(codes + p * HD + d0);
            k1 = *reinterpret_cast<const uint2*>(codes + p * HD + d1);
        }
        float amax = 0.f;
        bool bad = false;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            bad = bad || !(fabsf(x[e]) < INFINITY) || !(fabsf(y[e]) < INFINITY);
            amax = fmaxf(amax, fmaxf(fabsf(x[e]), fabsf(y[e])));
        }
        amax = wave_max(amax);
        const bool any_bad = __any(bad);
        if (lane == 0) {
            top[wv] = amax;
            odd[wv] = any_bad;
        }
        __syncthreads();
        constexpr int W = HD / 64;  // waves of K, of V
        bool not_finite = false;
        amax = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) {
            amax = fmaxf(amax, top[(is_v ? W : 0) + w]);
            not_finite = not_finite || odd[(is_v ? W : 0) + w];
        }
        const int e = not_finite || e_old == KVP_E_NAN ? KVP_E_NAN : max(e_old, kvp_exponent(amax));
        const float inv = e == KVP_E_NAN ? 0.f : ldexpf(1.f, -e);
        const bool move = j0 > 0 && e != KVP_E_NAN && e > e_old;
        const float down = move ? ldexpf(1.f, e_old - e) : 1.f;
        if (e == KVP_E_NAN) {
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = y[j] = 0.f;
        }
        if (id == 0) exps[at] = (int8_t)e;
        if (!is_v) {
            if (in) {
                *reinterpret_cast<uint2*>(codes + p * HD + d0) = kvp_code8(x, inv);
                *reinterpret_cast<uint2*>(codes + p * HD + d1) = kvp_code8(y, inv);
            } else if (old && move) {
                *reinterpret_cast<uint2*>(codes + p * HD + d0) = make_uint2(kvp_shift4(k0.x, down), kvp_shift4(k0.y, down));
                *reinterpret_cast<uint2*>(codes + p * HD + d1) = make_uint2(kvp_shift4(k1.x, down), kvp_shift4(k1.y, down));
            }
        } else if (in) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                turned[d0 + j][p] = (uint8_t)kvp_code(x[j], inv);
                turned[d1 + j][p] = (uint8_t)kvp_code(y[j], inv);
            }
        }
        __syncthreads();
        if (!is_v) return;
        uint8_t* dst = codes + id * KVP_BLOCK;
        const uint4 n = *reinterpret_cast<const uint4*>(turned[id]);
        if (j0 == 0 && j1 == KVP_BLOCK) {
            *reinterpret_cast<uint4*>(dst) = n;
            return;
        }
        const uint32_t o[4] = {v0.x, v0.y, v0.z, v0.w}, w[4] = {n.x, n.y, n.z, n.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {  // places 4 j .. 4 j + 3: old ones, new ones, and those of nobody as they are
            if (4 * j >= j1 || (4 * j + 4 <= j0 && !move)) continue;
            const uint32_t moved = move ? kvp_shift4(o[j], down) : o[j];
            const int a = min(max(j0 - 4 * j, 0), 4), b4 = min(j1 - 4 * j, 4);
            const uint32_t below = a == 4 ? ~0u : (1u << (8 * a)) - 1, upto = b4 == 4 ? ~0u : (1u << (8 * b4)) - 1;
            uint32_t tail = 0;
            if (b4 < 4) tail = *reinterpret_cast<const uint32_t*>(dst + 4 * j) & ~upto;
            *reinterpret_cast<uint32_t*>(dst + 4 * j) = (moved & below) | (w[j] & upto & ~below) | tail;
        }
        return;
    }

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
// HD threads turn one block of one head of K (16 dims of a token each), HD threads
// the same of V (4 dims of 4 tokens each, whose bytes change places by permutes: a
// row's stores are then 8 or 16 bytes, as K's; with single values they took twice as
// long) and pass the caches by, which 68 MB of rows would fill for nobody: 102 MB read
// and written for a ragged batch of 16 sequences of up to 8192 tokens in 21.5 us, 4.8
// TB/s, against 28 (a copy: 5.0).  Loads that pass them by took 32: V's are 4 bytes each.
// ---------------------------------------------------------------------------
template <typename T, int N>
__device__ __forceinline__ void kvp_put(T* dst, const uint32_t (&w)[N], float f) {  // 4 N bytes as values
    static_assert(N == 1 || N == 4, "");
    union {
        T t[4 * N];
        uint4 u4[N * sizeof(T) / 4 < 1 ? 1 : N * sizeof(T) / 4];
        uint2 u2[1];
    } r;
#pragma unroll
    for (int i = 0; i < 4 * N; ++i) st_act<T>(&r.t[i], (float)((int)(w[i / 4] >> (8 * (i % 4)) & 0xFFu) - KVP_ZERO) * f);
    if constexpr (4 * N * sizeof(T) == 8) {
        typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
        __builtin_nontemporal_store(u32x2{r.u2[0].x, r.u2[0].y}, reinterpret_cast<u32x2*>(dst));
    } else {
#pragma unroll
        for (int i = 0; i < (int)(4 * N * sizeof(T) / 16); ++i)
            __builtin_nontemporal_store(vte_u32x4{r.u4[i].x, r.u4[i].y, r.u4[i].z, r.u4[i].w}, reinterpret_cast<vte_u32x4*>(dst) + i);
    }
}

template <typename T, int HD>
__global__ __launch_bounds__(256) void kv_pages_read_kernel(KvPages c, KvRows r, T* __restrict__ k_out,
                                                            T* __restrict__ v_out, int out_rows) {
    constexpr int ITEM = 2 * HD;  // threads of an item (block, head)
    const int b = blockIdx.y;
    const KvSeq s = kvp_seq(r, b);
    if (s.pos < 0) return;
    const int cap = min(kvp_capacity(c, r), out_rows);
    const int end = s.n < cap - s.pos ? s.pos + s.n : cap;
    const int item = blockIdx.x * (256 / ITEM) + threadIdx.x / ITEM, i = threadIdx.x % HD;
    const bool is_v = threadIdx.x / HD & 1;
    const int blk = item / c.n_kv, h = item - blk * c.n_kv, t0 = blk * KVP_BLOCK;
    if (t0 >= end) return;
    const int page = kvp_page(c, r, b, t0 >> c.page_log2);
    const size_t at = (((size_t)max(page, 0) * c.n_kv + h) << (c.page_log2 - 4)) +
                      (blk & ((1 << (c.page_log2 - 4)) - 1));
    const size_t row = (size_t)c.n_kv * HD;
    T* dst = (is_v ? v_out : k_out) + (((size_t)b * out_rows + t0) * c.n_kv + h) * HD;
    const float f = page >= 0 ? kvp_scale((is_v ? c.v_exp : c.k_exp)[at]) : 0.f;
    if (!is_v) {
        const int p = i / (HD / 16), d = i % (HD / 16) * 16;
        const uint4 x = ldg_g16(c.k + at * (KVP_BLOCK * HD) + p * HD + d);
        const uint32_t w[4] = {x.x, x.y, x.z, x.w};
        if (t0 + p < end) kvp_put<T>(dst + p * row + d, w, f);
    } else {
        const int d = i % (HD / 4) * 4, p = i / (HD / 4) * 4;
        uint32_t x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e)
            x[e] = *reinterpret_cast<const uint32_t*>(c.v + at * (KVP_BLOCK * HD) + (d + e) * KVP_BLOCK + p);
        // bytes (dim, token) -> (token, dim)
        const uint32_t a = __builtin_amdgcn_perm(x[1], x[0], 0x05010400u), e = __builtin_amdgcn_perm(x[1], x[0], 0x07030602u);
        const uint32_t g = __builtin_amdgcn_perm(x[3], x[2], 0x05010400u), k = __builtin_amdgcn_perm(x[3], x[2], 0x07030602u);
        const uint32_t y[4] = {__builtin_amdgcn_perm(g, a, 0x05040100u), __builtin_amdgcn_perm(g, a, 0x07060302u),
                               __builtin_amdgcn_perm(k, e, 0x05040100u), __builtin_amdgcn_perm(k, e, 0x07060302u)};
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            const uint32_t w[1] = {y[t]};
            if (t0 + p + t < end) kvp_put<T>(dst + (p + t) * row + d, w, f);
        }
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
    auto fits = [](const void* p, long long stride) {
        return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && stride * (long long)sizeof(T) % 16 == 0;
    };
    const bool wide = (rp.cosc == nullptr || (rp.type != 2 && fits(rp.cosc, 0) && fits(rp.sinc, 0))) && fits(k, ks) &&
                      fits(v, vs) && (!q || (fits(q, qs) && fits(q_out, 0)));
    const int nt = wide ? 2 * HD : 128;
    const long long q_blocks = q ? ((long long)r.rows * n_q * (HD / (wide ? 16 : 2)) + nt - 1) / nt : 0;
    const int qx = (int)((q_blocks + grid_yz - 1) / grid_yz);
    auto kernel = wide ? kv_pages_append_kernel<T, HD, true> : kv_pages_append_kernel<T, HD, false>;
    hipLaunchKernelGGL(kernel, dim3(seq_blocks + qx, c.n_kv, r.batch), dim3(nt), 0, st, c, r,
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
    const int items = (rows + KVP_BLOCK - 1) / KVP_BLOCK * c.n_kv, per = 128 / HD;
    hipLaunchKernelGGL((kv_pages_read_kernel<T, HD>), dim3((items + per - 1) / per, r.batch), dim3(256), 0, st, c, r,
                       (T*)k_out, (T*)v_out, out_rows);
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
