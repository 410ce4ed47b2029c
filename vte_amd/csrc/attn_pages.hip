// Attention over the 8-bit paged KV cache (layout: kv_pages.h), gfx950: few rows
// of each sequence (decoded tokens) or many (prompt chunks).
//
// Algorithm: online softmax per chunk and log-sum-exp combine as in
// vte/compiler/templates/rdna/flash_attention_split_kv_partial.hip.template:31-120
// and flash_attention_split_kv_reduce.hip.template:14-67, with
//   s_t = scale 2^ek(t) q.K_t,  out = sum_t p_t 2^ev(t) V_t / sum_t p_t,  p_t = exp(s_t - max)
// over whole-number K and V.  Bytes become fp16 exactly (0x6400 | byte is 1024 +
// byte; minus 1152), so both products run on 16x16x32 or 32x32x16 fp16 MFMAs with
// no rounding of K or V.  The V scale is folded into the probability, relative to
// the largest exponent seen (2^14 p 2^(ev - ref), at most 2^14), which is why
// byte 0..255 of a masked token times probability 0 is the only thing a place that
// nobody sees can add: its exponent, which may be anything, is never used.
#include <algorithm>
#include <type_traits>

#include "attn_tile.h"
#include "kv_pages.h"

#define PA_TILE 64       // tokens of a wave's step: a lane group of 16 holds one block of 16
#define PA_P_LOG2 14     // probabilities are held as 2^14 p
#define PA_NONE (-1e30f) // running maximum before anything is seen

typedef _Float16 pa_h2 __attribute__((ext_vector_type(2)));
typedef unsigned pa_u2 __attribute__((ext_vector_type(2)));

// 8 bytes as 8 fp16 whole numbers (byte - 128).
__device__ __forceinline__ half8_t pa_half8(uint32_t a, uint32_t b) {
    union {
        uint32_t u[4];
        pa_h2 h[4];
        half8_t v;
    } r;
    r.u[0] = __builtin_amdgcn_perm(0x64646464u, a, 0x04010400u);
    r.u[1] = __builtin_amdgcn_perm(0x64646464u, a, 0x04030402u);
    r.u[2] = __builtin_amdgcn_perm(0x64646464u, b, 0x04010400u);
    r.u[3] = __builtin_amdgcn_perm(0x64646464u, b, 0x04030402u);
    const pa_h2 z = {(_Float16)1152.f, (_Float16)1152.f};
#pragma unroll
    for (int i = 0; i < 4; ++i) r.h[i] = r.h[i] - z;
    return r.v;
}
// Over the lanes that differ in lane group (16 lanes each): every lane gets the result.
__device__ __forceinline__ float pa_max4(float v) {
    pa_u2 a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}
__device__ __forceinline__ int pa_max4(int v) {
    pa_u2 a = __builtin_amdgcn_permlane16_swap((unsigned)v, (unsigned)v, false, false);
    v = max((int)a[0], (int)a[1]);
    a = __builtin_amdgcn_permlane32_swap((unsigned)v, (unsigned)v, false, false);
    return max((int)a[0], (int)a[1]);
}
__device__ __forceinline__ float pa_sum4(float v) {
    pa_u2 a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}
// 2^d for d <= 0 (0 below the smallest normal).
__device__ __forceinline__ float pa_pow2(int d) { return d < -126 ? 0.f : __uint_as_float((uint32_t)(d + 127) << 23); }

// ---------------------------------------------------------------------------
// Few rows.  A segment is one (sequence, KV head): its n rows of G heads each are
// at most 16 columns of one MFMA tile, its tokens ceil(len / 64) tiles.  The
// tiles of all segments, one after the other, are cut into equal shares, one per
// block, so a ragged batch keeps every block as busy as the others; a block walks
// the segments its share touches, its four waves taking every fourth tile.  A
// segment that lies in one share is done there; one that is cut leaves a record in
// each: it is its first block's last piece and the first piece of the others, so
// two records a block are enough.
// ---------------------------------------------------------------------------
struct PaPlan {
    int blocks;  // grid of the main launch
    int ncol;    // columns (rows of the second form) of a record
    float* ml;   // [2 blocks][ncol][2]: maximum (log2), sum
    int* ev;     // [2 blocks]: exponent the record's sums are relative to
    float* o;    // [2 blocks][ncol][HD]
    int2* seg;   // [segments]: first block, pieces
};
// Record of piece i of a segment whose first block is `first`.
__device__ __forceinline__ size_t pa_rec(int first, int i) { return i == 0 ? 2 * (size_t)first + 1 : 2 * ((size_t)first + i); }

// Tokens that any row of sequence b sees.
__device__ __forceinline__ int pa_tokens(const KvSeq& s, int cap) {
    return s.n == 0 ? 0 : (s.n < cap - s.pos ? s.pos + s.n : cap);
}

// The block's share [t, t_end) of all tiles, and the sequence that t lies in with
// the number of tiles before it.
struct PaShare {
    long long t, t_end, before;
    long long share;
    int b;
};
__device__ __forceinline__ PaShare pa_share(const KvPages& c, const KvRows& r, int cap, int block, int blocks) {
    __shared__ long long wsum[4];
    __shared__ long long found[2];
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    const int per = (r.batch + 255) / 256;
    long long mine = 0;
    for (int b = tid * per; b < min(r.batch, tid * per + per); ++b)
        mine += (long long)c.n_kv * ((pa_tokens(kvp_seq(r, b), cap) + PA_TILE - 1) / PA_TILE);
    long long incl = mine;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const long long up = __shfl_up(incl, d, 64);
        if (lane >= d) incl += up;
    }
    if (lane == 63) wsum[wv] = incl;
    __syncthreads();
    for (int w = 0; w < wv; ++w) incl += wsum[w];
    const long long total = wsum[0] + wsum[1] + wsum[2] + wsum[3];
    PaShare s;
    s.share = ((total + blocks - 1) / blocks + 3) / 4 * 4;
    s.t = s.share * block;
    s.t_end = min(total, s.t + s.share);
    if (mine > 0 && s.t >= incl - mine && s.t < incl) {
        long long before = incl - mine;
        int b = tid * per;
        for (;; ++b) {
            const long long n = (long long)c.n_kv * ((pa_tokens(kvp_seq(r, b), cap) + PA_TILE - 1) / PA_TILE);
            if (s.t < before + n) break;
            before += n;
        }
        found[0] = b;
        found[1] = before;
    }
    __syncthreads();
    s.b = (int)found[0];
    s.before = found[1];
    return s;
}

// One wave's tile: K rows (lane: row col of each of the four 16-row tiles) and V (lane: dim col, block grp).
template <int HD>
struct PaTile {
    uint4 k[4][HD / 64], v[HD / 16];
    int ek, ev;
    bool has;  // the lane's block has a page
};

template <typename T, int HD>
__global__ __launch_bounds__(256, 2) void attn_pages_rows_kernel(KvPages c, KvRows r, PaPlan pl,
                                                                 const T* __restrict__ q, T* __restrict__ out, int n_q,
                                                                 float scale) {
    constexpr int PARTS = sizeof(T) == 4 ? 2 : 1;  // fp16 parts of q and of the probabilities
    constexpr int KC = HD / 64;                    // 16-byte pieces of a K row that a lane holds
    constexpr int DT = HD / 16;
    __shared__ float m_sh[4][16], l_sh[4][16];
    __shared__ int ev_sh[4];
    __shared__ __align__(16) float o_sh[4][16][HD + 4];
    const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 15, grp = lane >> 4;
    const int G = n_q / c.n_kv, cap = kvp_capacity(c, r);
    const int bl = c.page_log2 - 4;  // log2 of a page's blocks
    PaShare sh = pa_share(c, r, cap, blockIdx.x, pl.blocks);
    int b = sh.b;
    long long t = sh.t, before = sh.before;

    while (t < sh.t_end) {
        const KvSeq s = kvp_seq(r, b);
        const int len = pa_tokens(s, cap), nt = (len + PA_TILE - 1) / PA_TILE;
        if (t - before >= (long long)nt * c.n_kv) {  // the next sequence
            before += (long long)nt * c.n_kv;
            ++b;
            continue;
        }
        const int h = (int)((t - before) / nt), a = (int)((t - before) - (long long)h * nt);
        const int z = (int)min((long long)nt, a + (sh.t_end - t));  // tiles [a, z) of the segment
        const long long seg_t = before + (long long)h * nt;         // its first tile among all
        const int* table = r.page_table + (size_t)b * r.max_pages;

        // ---- this lane's column: query, tokens it sees ----
        const int ncol = s.n * G, ci = min(col, ncol - 1);
        const int qi = ci / G, qh = h * G + ci - qi * G;
        const int end = col < ncol ? kvp_len(s.pos + qi, cap) : 0;
        half8_t qb[PARTS][2 * KC];
        float q_unit = 1.f;  // of the values in qb
        {
            const T* qp = q + ((size_t)(s.first + qi) * n_q + qh) * HD + 16 * grp;
            if constexpr (PARTS == 1) {
#pragma unroll
                for (int i = 0; i < 2 * KC; ++i)
                    qb[0][i] = *reinterpret_cast<const half8_t*>(qp + 64 * (i >> 1) + 8 * (i & 1));
            } else {  // scaled by a power of two so that the second part keeps its bits too
                float x[2 * KC][8], amax = 0.f;
#pragma unroll
                for (int i = 0; i < 2 * KC; ++i) {
                    const float4* p4 = reinterpret_cast<const float4*>(qp + 64 * (i >> 1) + 8 * (i & 1));
                    *reinterpret_cast<float4*>(&x[i][0]) = p4[0];
                    *reinterpret_cast<float4*>(&x[i][4]) = p4[1];
#pragma unroll
                    for (int j = 0; j < 8; ++j) amax = fmaxf(amax, fabsf(x[i][j]));
                }
                amax = pa_max4(amax);
                const int e = min(max((int)(__float_as_uint(amax) >> 23) - 127, -110), 126);  // 2^e <= amax
                const float up = __uint_as_float((uint32_t)(127 + 13 - e) << 23);
                q_unit = __uint_as_float((uint32_t)(127 - 13 + e) << 23);
#pragma unroll
                for (int i = 0; i < 2 * KC; ++i)
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const float y = x[i][j] * up;
                        qb[0][i][j] = (_Float16)y;
                        qb[1][i][j] = (_Float16)(y - (float)qb[0][i][j]);
                    }
            }
        }
        const float c2 = scale * 1.44269504088896340736f * q_unit;  // exp(scale s) = 2^(c2 s)

        float m_run = PA_NONE, l_run = 0.f;
        int ev_ref = KVP_E_MIN;
        floatx4_t o[DT];  // lane: column col, dims 16 dt + 4 grp + i
#pragma unroll
        for (int i = 0; i < DT; ++i) o[i] = floatx4_t{0.f, 0.f, 0.f, 0.f};

        // K row of 16-row tile tt: token 16 (col / 4) + 4 tt + col % 4, so that the scores a lane gets from the four
        // tiles are those of block grp in order, which is the order V's 16 bytes hold its tokens in.
        auto load = [&](PaTile<HD>& x, int tile) {
            const int t0 = tile * PA_TILE;
            const int last = (len - 1) >> 4;  // blocks past the end read the last one (their tokens are masked)
            const int kb = min((t0 >> 4) + (col >> 2), last), vb = min((t0 >> 4) + grp, last);
            const int kp = table[kb >> bl], vp = table[vb >> bl];
            x.has = (unsigned)vp < (unsigned)c.n_pages;
            const size_t ka = ((((size_t)((unsigned)kp < (unsigned)c.n_pages ? kp : 0) * c.n_kv + h) << bl) +
                               (kb & ((1 << bl) - 1))) * (KVP_BLOCK * HD);
            const size_t vi = (((size_t)(x.has ? vp : 0) * c.n_kv + h) << bl) + (vb & ((1 << bl) - 1));
            const uint8_t* kr = c.k + ka + (col & 3) * HD + 16 * grp;
#pragma unroll
            for (int tt = 0; tt < 4; ++tt)
#pragma unroll
                for (int j = 0; j < KC; ++j) x.k[tt][j] = ldg_g16(kr + 4 * tt * HD + 64 * j);
            x.ek = c.k_exp[vi];
            x.ev = c.v_exp[vi];
            const uint8_t* vr = c.v + vi * (KVP_BLOCK * HD) + col * KVP_BLOCK;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) x.v[dt] = ldg_g16(vr + 256 * dt);
        };
        auto step = [&](const PaTile<HD>& x, int tile) {
            const int p0 = tile * PA_TILE + 16 * grp;  // this lane group's block
            floatx4_t sc[4];
#pragma unroll
            for (int tt = 0; tt < 4; ++tt) {
                sc[tt] = floatx4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int j = 0; j < KC; ++j) {
                    const half8_t k0 = pa_half8(x.k[tt][j].x, x.k[tt][j].y), k1 = pa_half8(x.k[tt][j].z, x.k[tt][j].w);
#pragma unroll
                    for (int p = 0; p < PARTS; ++p) {
                        sc[tt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, qb[p][2 * j], sc[tt], 0, 0, 0);
                        sc[tt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1, qb[p][2 * j + 1], sc[tt], 0, 0, 0);
                    }
                }
            }
            const float kf = kvp_scale(x.ek) * c2;
            const int live = x.has ? end - p0 : 0;  // places of the block that this column sees
            float mx = m_run;
#pragma unroll
            for (int tt = 0; tt < 4; ++tt)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    sc[tt][i] = 4 * tt + i < live ? sc[tt][i] * kf : -INFINITY;
                    mx = fmaxf(mx, sc[tt][i]);
                }
            mx = pa_max4(mx);
            const bool in_use = x.has && p0 < len;
            const int evm = max(ev_ref, pa_max4(in_use ? x.ev : KVP_E_MIN));
            if (__any(mx > m_run) || evm > ev_ref) {
                const float corr = __builtin_amdgcn_exp2f(m_run - mx);
                l_run *= corr;
                const float both = corr * pa_pow2(ev_ref - evm);
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) o[dt] *= both;
                m_run = mx;
                ev_ref = evm;
            }
            // (a NaN block's tokens are NaN to the columns that see them and nothing to the others)
            const float vf = x.ev == KVP_E_NAN ? NAN : pa_pow2(min(x.ev - evm, 0)) * (float)(1 << PA_P_LOG2);
            half8_t pa[PARTS][2];
#pragma unroll
            for (int tt = 0; tt < 4; ++tt)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float p = __builtin_amdgcn_exp2f(sc[tt][i] - mx);
                    l_run += p;
                    const float w = 4 * tt + i < live ? p * vf : 0.f;
                    const int u = tt >> 1, j = 4 * (tt & 1) + i;
                    pa[0][u][j] = (_Float16)w;
                    if constexpr (PARTS == 2) pa[1][u][j] = (_Float16)(w - (float)pa[0][u][j]);
                }
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
                const half8_t v0 = pa_half8(x.v[dt].x, x.v[dt].y), v1 = pa_half8(x.v[dt].z, x.v[dt].w);
#pragma unroll
                for (int p = 0; p < PARTS; ++p) {
                    o[dt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, pa[p][0], o[dt], 0, 0, 0);
                    o[dt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, pa[p][1], o[dt], 0, 0, 0);
                }
            }
        };

        // ---- the wave's tiles, the next one's loads under this one's work ----
        PaTile<HD> A, B;
        int tile = a + wv;
        if (tile < z) load(A, tile);
        while (tile < z) {
            if (tile + 4 < z) load(B, tile + 4);
            step(A, tile);
            tile += 4;
            if (tile >= z) break;
            if (tile + 4 < z) load(A, tile + 4);
            step(B, tile);
            tile += 4;
        }

        // ---- the four waves together ----
        l_run = pa_sum4(l_run);
        if (grp == 0) {
            m_sh[wv][col] = m_run;
            l_sh[wv][col] = l_run;
        }
        if (lane == 0) ev_sh[wv] = ev_ref;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) *reinterpret_cast<floatx4_t*>(&o_sh[wv][col][16 * dt + 4 * grp]) = o[dt];
        __syncthreads();
        const int seg = b * c.n_kv + h;
        const int first = (int)(seg_t / sh.share), pieces = (int)((seg_t + nt - 1) / sh.share) - first + 1;
        const size_t rec = pa_rec(first, blockIdx.x - first);
        const int EV = max(max(ev_sh[0], ev_sh[1]), max(ev_sh[2], ev_sh[3]));
        for (int i = tid; i < ncol * (HD / 4); i += 256) {
            const int cc = i / (HD / 4), d = i % (HD / 4) * 4;
            const float M = fmaxf(fmaxf(m_sh[0][cc], m_sh[1][cc]), fmaxf(m_sh[2][cc], m_sh[3][cc]));
            float L = 0.f;
            floatx4_t O = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const float f = __builtin_amdgcn_exp2f(m_sh[w][cc] - M);
                L = fmaf(l_sh[w][cc], f, L);
                O += *reinterpret_cast<const floatx4_t*>(&o_sh[w][cc][d]) * (f * pa_pow2(ev_sh[w] - EV));
            }
            if (pieces == 1) {
                const int i_row = cc / G;
                T* dst = out + ((size_t)(s.first + i_row) * n_q + h * G + cc - i_row * G) * HD + d;
#pragma unroll
                for (int e = 0; e < 4; ++e) st_act<T>(dst + e, L == 0.f ? 0.f : ldexpf(O[e] / L, EV - PA_P_LOG2));
            } else {
                *reinterpret_cast<floatx4_t*>(pl.o + (rec * pl.ncol + cc) * HD + d) = O;
                if (d == 0) {
                    pl.ml[(rec * pl.ncol + cc) * 2] = M;
                    pl.ml[(rec * pl.ncol + cc) * 2 + 1] = L;
                }
            }
        }
        if (tid == 0) {
            if (pieces > 1) pl.ev[rec] = EV;
            if (a == 0) pl.seg[seg] = make_int2(first, pieces);
        }
        __syncthreads();
        t += z - a;
    }
}

// Combine of the segments that were cut, and zeros for the rows that see nothing:
// grid (segments, ncol), HD / 4 threads per group of pieces.
template <typename T, int HD>
__global__ __launch_bounds__(256) void attn_pages_combine_kernel(KvPages c, KvRows r, PaPlan pl, T* __restrict__ out,
                                                                 int n_q) {
    constexpr int TD = HD / 4, GR = 256 / TD;  // threads of a row, groups of pieces
    __shared__ float w_sh[256];
    __shared__ __align__(16) float o_sh[GR][HD + 4];
    __shared__ float red[2][4];
    __shared__ int red_ev[4];
    const int seg = blockIdx.x, cc = blockIdx.y, b = seg / c.n_kv, h = seg - b * c.n_kv, tid = threadIdx.x;
    const int lane = tid & 63, wv = tid >> 6, g = tid / TD, d = tid % TD * 4;
    const int G = n_q / c.n_kv, cap = kvp_capacity(c, r);
    const KvSeq s = kvp_place(r, b);
    if (cc >= s.n * G) return;
    T* dst = out + ((size_t)(s.first + cc / G) * n_q + h * G + cc % G) * HD;
    if (s.pos < 0) {
        if (tid < HD) st_act<T>(dst + tid, 0.f);
        return;
    }
    const int2 sg = pl.seg[seg];
    if (sg.y == 1) return;
    float M = PA_NONE;
    int EV = KVP_E_MIN;
    for (int i = tid; i < sg.y; i += 256) {
        const size_t rec = pa_rec(sg.x, i);
        M = fmaxf(M, pl.ml[(rec * pl.ncol + cc) * 2]);
        EV = max(EV, pl.ev[rec]);
    }
    M = wave_max(M);
    for (int x = 1; x < 64; x *= 2) EV = max(EV, __shfl_xor(EV, x, 64));
    if (lane == 0) {
        red[0][wv] = M;
        red_ev[wv] = EV;
    }
    __syncthreads();
    M = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
    EV = max(max(red_ev[0], red_ev[1]), max(red_ev[2], red_ev[3]));
    float l = 0.f;
    floatx4_t O = {0.f, 0.f, 0.f, 0.f};
    for (int i0 = 0; i0 < sg.y; i0 += 256) {  // 256 pieces at a time
        const int n = min(256, sg.y - i0);
        if (tid < n) {
            const size_t rec = pa_rec(sg.x, i0 + tid);
            const float f = __builtin_amdgcn_exp2f(pl.ml[(rec * pl.ncol + cc) * 2] - M);
            l = fmaf(pl.ml[(rec * pl.ncol + cc) * 2 + 1], f, l);
            w_sh[tid] = f * pa_pow2(pl.ev[rec] - EV);
        }
        __syncthreads();
#pragma unroll 4
        for (int i = g; i < n; i += GR)
            O += *reinterpret_cast<const floatx4_t*>(pl.o + (pa_rec(sg.x, i0 + i) * pl.ncol + cc) * HD + d) * w_sh[i];
        __syncthreads();
    }
    l = wave_sum(l);
    if (lane == 0) red[1][wv] = l;
    *reinterpret_cast<floatx4_t*>(&o_sh[g][d]) = O;
    __syncthreads();
    const float L = (red[1][0] + red[1][1]) + (red[1][2] + red[1][3]);
    if (tid < HD) {
        float x = 0.f;
#pragma unroll
        for (int i = 0; i < GR; ++i) x += o_sh[i][tid];
        st_act<T>(dst + tid, L == 0.f ? 0.f : ldexpf(x / L, EV - PA_P_LOG2));
    }
}

// ---------------------------------------------------------------------------
// Many rows.  Rows of a KV head are numbered (new row, query head of the group),
// so a group of any size fills 32-row MFMA tiles; 128 of them are a row block and
// see tokens up to their last row's position.  A segment is (KV head, row block);
// shares of 64-token steps are cut as above, from a plan that a first launch
// writes (row blocks of a ragged batch and the steps before each).
//
// A block's four waves own 32 rows each and walk the same steps.  The bytes of a
// step become fp16 once per block on their way into LDS, times 2^(e - ref) with
// ref the largest exponent so far (exact down to 2^-24 of the largest block's
// step), so a step's scores and sums have one scale.  Scores are K.Q^T, sums are
// V^T.P^T (a lane is a row in both), K rows are read with token bits 2 and 3
// swapped so that a lane's scores are its operand of the second product as they
// stand.
// ---------------------------------------------------------------------------
#define PA_ROWS 128  // rows of a row block

typedef float floatx16_t __attribute__((ext_vector_type(16)));

struct PaRowBlock {
    int b, rb;      // sequence, row block of it
    int steps;      // 64-token steps that its rows see
    int before;     // steps of the row blocks before it
};
struct PaStart {
    int block, h, at, pad;  // row block, KV head and step of it that a share starts with
};
struct PaPrompt {
    PaRowBlock* rb;  // [row blocks]
    PaStart* start;  // [blocks]
    int* total;      // row blocks, steps of one KV head, steps of a share
};

// One block: row blocks of every sequence, their steps, and where each share starts.
__global__ __launch_bounds__(1024) void attn_pages_plan_kernel(KvPages c, KvRows r, PaPlan pl, PaPrompt pp, int n_q) {
    __shared__ int wsum[16];
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    const int G = n_q / c.n_kv, cap = kvp_capacity(c, r);
    auto scan = [&](int mine, int& total) {  // sum over the threads before this one
        int incl = mine;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const int up = __shfl_up(incl, d, 64);
            if (lane >= d) incl += up;
        }
        __syncthreads();
        if (lane == 63) wsum[wv] = incl;
        __syncthreads();
        int before = 0;
        total = 0;
        for (int w = 0; w < 16; ++w) {
            before += w < wv ? wsum[w] : 0;
            total += wsum[w];
        }
        return before + incl - mine;
    };
    // row blocks, in the sequences' order
    const int per = (r.batch + 1023) / 1024;
    int mine = 0, n_rb, steps;
    for (int b = tid * per; b < min(r.batch, tid * per + per); ++b) mine += (kvp_place(r, b).n * G + PA_ROWS - 1) / PA_ROWS;
    int at = scan(mine, n_rb);
    for (int b = tid * per; b < min(r.batch, tid * per + per); ++b) {
        const int n = (kvp_place(r, b).n * G + PA_ROWS - 1) / PA_ROWS;
        for (int i = 0; i < n; ++i) pp.rb[at++] = PaRowBlock{b, i, 0, 0};
    }
    __threadfence_block();
    __syncthreads();
    // steps of each
    const int per2 = (n_rb + 1023) / 1024, lo = min(n_rb, tid * per2), hi = min(n_rb, lo + per2);
    mine = 0;
    for (int i = lo; i < hi; ++i) {
        const int b = pp.rb[i].b;
        const KvSeq s = kvp_place(r, b);
        const int last = min((pp.rb[i].rb * PA_ROWS + PA_ROWS - 1) / G, s.n - 1);
        const int n = s.pos < 0 ? 0 : ((s.pos < cap - last ? s.pos + last + 1 : cap) + PA_TILE - 1) / PA_TILE;
        pp.rb[i].steps = n;
        mine += n;
    }
    int before = scan(mine, steps);
    const int share = max(1, (int)(((long long)steps * c.n_kv + pl.blocks - 1) / pl.blocks));
    for (int i = lo; i < hi; ++i) {
        const int n = pp.rb[i].steps;
        pp.rb[i].before = before;
        for (int h = 0; h < c.n_kv; ++h) {  // shares that start in this segment
            const long long t0 = (long long)h * steps + before;
            for (long long k = (t0 + share - 1) / share; k * share < t0 + n; ++k)
                pp.start[k] = PaStart{i, h, (int)(k * share - t0), 0};
        }
        before += n;
    }
    if (tid == 0) {
        pp.total[0] = n_rb;
        pp.total[1] = steps;
        pp.total[2] = share;
    }
}

template <typename T, int HD>
__global__ __launch_bounds__(256, 2) void attn_pages_prompt_kernel(KvPages c, KvRows r, PaPlan pl, PaPrompt pp,
                                                                   const T* __restrict__ q, T* __restrict__ out,
                                                                   int n_q, float scale) {
    constexpr int PARTS = sizeof(T) == 4 ? 2 : 1;
    constexpr int KS = HD / 16, DT = HD / 32, U = HD / 64;  // 16-dim steps of a score, 32-dim tiles, staged pieces a thread
    constexpr int KROW = PA_TILE * 16 + 8;                  // halves of a 16-dim column of K, 16 bytes apart in banks
    struct alignas(16) Tile {
        _Float16 k[KS * KROW];
        _Float16 v[4 * HD * 16];
    };
    __shared__ Tile tiles[2];
    const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int row = lane & 31, half = lane >> 5;
    const int G = n_q / c.n_kv, cap = kvp_capacity(c, r), bl = c.page_log2 - 4;
    const int steps = pp.total[1], share = pp.total[2];
    const long long all = (long long)steps * c.n_kv;
    long long t = (long long)blockIdx.x * share;
    const long long t_end = min(all, t + share);
    if (t >= t_end) return;
    const PaStart st = pp.start[blockIdx.x];
    int rbi = __builtin_amdgcn_readfirstlane(st.block), h = __builtin_amdgcn_readfirstlane(st.h);
    int a = __builtin_amdgcn_readfirstlane(st.at);

    while (t < t_end) {
        const PaRowBlock R = pp.rb[rbi];
        const int b = __builtin_amdgcn_readfirstlane(R.b), nt = __builtin_amdgcn_readfirstlane(R.steps);
        if (a >= nt) {  // a row block that sees nothing, or the end of this one
            a = 0;
            if (++rbi == pp.total[0]) {
                rbi = 0;
                ++h;
            }
            continue;
        }
        const int z = (int)min((long long)nt, a + (t_end - t));
        const KvSeq s = kvp_seq(r, b);
        const int* table = r.page_table + (size_t)b * r.max_pages;

        // ---- this lane's row ----
        const int r0 = R.rb * PA_ROWS + wv * 32, rows = s.n * G;
        const int ri = min(r0 + row, rows - 1), qi = ri / G, qh = h * G + ri - qi * G;
        const int end = r0 + row < rows ? kvp_len(s.pos + qi, cap) : 0;
        const int seg_end = kvp_len(s.pos + min((R.rb * PA_ROWS + PA_ROWS - 1) / G, s.n - 1), cap);  // of the row block
        const int longest = r0 < rows ? kvp_len(s.pos + min(r0 + 31, rows - 1) / G, cap) : 0;       // of the wave
        const int shortest = r0 + 31 < rows ? kvp_len(s.pos + r0 / G, cap) : 0;
        half8_t qb[PARTS][KS];
        float q_unit = 1.f;
        {
            const T* qp = q + ((size_t)(s.first + qi) * n_q + qh) * HD + 8 * half;
            if constexpr (PARTS == 1) {
#pragma unroll
                for (int i = 0; i < KS; ++i) qb[0][i] = *reinterpret_cast<const half8_t*>(qp + 16 * i);
            } else {  // scaled by a power of two so that the second part keeps its bits too
                float amax = 0.f;
#pragma unroll
                for (int i = 0; i < KS; ++i)
#pragma unroll
                    for (int j = 0; j < 8; ++j) amax = fmaxf(amax, fabsf(qp[16 * i + j]));
                amax = fmaxf(amax, __shfl_xor(amax, 32, 64));
                const int e = min(max((int)(__float_as_uint(amax) >> 23) - 127, -110), 126);  // 2^e <= amax
                const float up = __uint_as_float((uint32_t)(127 + 13 - e) << 23);
                q_unit = __uint_as_float((uint32_t)(127 - 13 + e) << 23);
#pragma unroll
                for (int i = 0; i < KS; ++i)
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const float y = qp[16 * i + j] * up;
                        qb[0][i][j] = (_Float16)y;
                        qb[1][i][j] = (_Float16)(y - (float)qb[0][i][j]);
                    }
            }
        }
        const float c2 = scale * 1.44269504088896340736f * q_unit;

        float m_run = PA_NONE, l_run = 0.f;
        floatx16_t o[DT];  // lane: row, dims 32 dt + 8 (i / 4) + 4 half + i % 4
#pragma unroll
        for (int i = 0; i < DT; ++i)
#pragma unroll
            for (int j = 0; j < 16; ++j) o[i][j] = 0.f;
        int o_ref = KVP_E_MIN;                              // exponent that o is relative to
        int k_ref = KVP_E_MIN, v_ref = KVP_E_MIN;           // of the step staged last
        int cur_k = KVP_E_MIN, cur_v = KVP_E_MIN, cur_odd = 0;  // of the step in work; its blocks without a page, NaN in V

        // Staging: registers, then LDS.  Lane j & 3 knows block j's page and exponents; a wave's pieces lie in one block.
        uint4 kx[U], vx[U];
        int ek, ev, page;
        bool used;
        auto find = [&](int step) {
            const int blk = 4 * step + (lane & 3);
            used = blk * KVP_BLOCK < seg_end;
            page = used ? table[blk >> bl] : -1;
            used = used && (unsigned)page < (unsigned)c.n_pages;
        };
        auto load = [&](int step) {
            const int blk = 4 * step + (lane & 3);
            const size_t i = (((size_t)(used ? page : 0) * c.n_kv + h) << bl) + (blk & ((1 << bl) - 1));
            ek = c.k_exp[i];
            ev = c.v_exp[i];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int j = U == 2 ? 2 * u + (wv >> 1) : wv;  // the block of this wave's pieces
                const int p = __builtin_amdgcn_readlane(used ? page : 0, j);
                const size_t at = (((size_t)p * c.n_kv + h) << bl) + ((4 * step + j) & ((1 << bl) - 1));
                const int piece = U == 2 ? (wv & 1) * 64 + lane : lane;  // of the block's HD pieces
                kx[u] = ldg_g16(c.k + at * (KVP_BLOCK * HD) + piece * 16);
                vx[u] = ldg_g16(c.v + at * (KVP_BLOCK * HD) + piece * 16);
            }
        };
        auto scaled = [&](const uint4& x, _Float16 f, _Float16* dst) {
            const half8_t lo = pa_half8(x.x, x.y) * f, hi = pa_half8(x.z, x.w) * f;
            *reinterpret_cast<half8_t*>(dst) = lo;
            *reinterpret_cast<half8_t*>(dst + 8) = hi;
        };
        int next_odd = 0;
        auto put = [&](Tile& D) {
            next_odd = 0;
            int e[4], f[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const bool in = __builtin_amdgcn_readlane((int)used, j);
                e[j] = in ? __builtin_amdgcn_readlane(ek, j) : -1000;
                f[j] = in ? __builtin_amdgcn_readlane(ev, j) : -1000;
                if (!in) next_odd |= 1 << j;
                if (f[j] == KVP_E_NAN) next_odd |= 16 << j;
                k_ref = max(k_ref, e[j]);
                v_ref = max(v_ref, f[j]);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int j = U == 2 ? 2 * u + (wv >> 1) : wv;
                int ej = e[0], fj = f[0];
#pragma unroll
                for (int i = 1; i < 4; ++i) {
                    ej = i == j ? e[i] : ej;
                    fj = i == j ? f[i] : fj;
                }
                const _Float16 kf = ej == KVP_E_NAN ? (_Float16)NAN : (_Float16)pa_pow2(ej - k_ref);
                const _Float16 vf = fj == KVP_E_NAN ? (_Float16)0.f : (_Float16)pa_pow2(fj - v_ref);
                const int piece = U == 2 ? (wv & 1) * 64 + lane : lane;
                // K piece: token piece / KS of the block, dims 16 (piece % KS) ..; V piece: dim `piece`
                scaled(kx[u], kf, D.k + (piece % KS) * KROW + (16 * j + piece / KS) * 16);
                scaled(vx[u], vf, D.v + (j * HD + piece) * 16);
            }
        };

        // K row of 32-token tile tt: token with bits 2 and 3 of the lane's row swapped
        const int kt = (row & 0x13) | (row & 4) << 1 | (row & 8) >> 1;
        auto work = [&](const Tile& S, int step, auto ends) {
            constexpr bool ENDS = decltype(ends)::value;
            floatx16_t sc[2];
#pragma unroll
            for (int tt = 0; tt < 2; ++tt) {
#pragma unroll
                for (int j = 0; j < 16; ++j) sc[tt][j] = 0.f;
#pragma unroll
                for (int i = 0; i < KS; ++i) {
                    const half8_t k = *reinterpret_cast<const half8_t*>(S.k + i * KROW + (32 * tt + kt) * 16 + 8 * half);
#pragma unroll
                    for (int p = 0; p < PARTS; ++p)
                        sc[tt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, qb[p][i], sc[tt], 0, 0, 0);
                }
            }
            // lane: its row's scores of tokens 32 tt + 16 (j / 8) + 8 half + j % 8
            const int live = end - step * PA_TILE - 8 * half;
            if constexpr (ENDS) {
#pragma unroll
                for (int tt = 0; tt < 2; ++tt)
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        const bool in = 32 * tt + 16 * (j >> 3) + (j & 7) < live && !(cur_odd >> (2 * tt + (j >> 3)) & 1);
                        sc[tt][j] = in ? sc[tt][j] : -INFINITY;
                    }
            }
            float mx = sc[0][0];
#pragma unroll
            for (int tt = 0; tt < 2; ++tt)
#pragma unroll
                for (int j = 0; j < 16; ++j) mx = fmaxf(mx, sc[tt][j]);
            {
                const pa_u2 w = __builtin_amdgcn_permlane32_swap(__float_as_uint(mx), __float_as_uint(mx), false, false);
                mx = fmaxf(__uint_as_float(w[0]), __uint_as_float(w[1]));
            }
            const float kf = kvp_scale(cur_k) * c2;
            mx = fmaxf(m_run, mx * kf);
            if (__any(mx > m_run) || cur_v > o_ref) {
                const float corr = __builtin_amdgcn_exp2f(m_run - mx);
                l_run *= corr;
                const float both = corr * pa_pow2(o_ref - cur_v);
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) o[dt] *= both;
                m_run = mx;
                o_ref = cur_v;
            }
            const float shift = (float)PA_P_LOG2 - mx;
            half8_t pf[PARTS][4];
#pragma unroll
            for (int tt = 0; tt < 2; ++tt)
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    const float p = __builtin_amdgcn_exp2f(fmaf(sc[tt][j], kf, shift));
                    l_run += p;
                    const int kb = 2 * tt + (j >> 3);
                    float w = p;
                    if constexpr (ENDS) w = (cur_odd >> (4 + kb) & 1) && !(sc[tt][j] == -INFINITY) ? NAN : p;
                    pf[0][kb][j & 7] = (_Float16)w;
                    if constexpr (PARTS == 2) pf[1][kb][j & 7] = (_Float16)(w - (float)pf[0][kb][j & 7]);
                }
#pragma unroll
            for (int kb = 0; kb < 4; ++kb)
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) {
                    const half8_t v = *reinterpret_cast<const half8_t*>(S.v + (kb * HD + 32 * dt + row) * 16 + 8 * half);
#pragma unroll
                    for (int p = 0; p < PARTS; ++p)
                        o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, pf[p][kb], o[dt], 0, 0, 0);
                }
        };

        find(a);
        load(a);
        put(tiles[0]);
        cur_k = k_ref;
        cur_v = v_ref;
        cur_odd = next_odd;
        if (a + 1 < z) find(a + 1);
        __syncthreads();
        int buf = 0;
        for (int step = a; step < z; ++step) {
            const bool more = step + 1 < z;
            if (more) load(step + 1);
            if (step * PA_TILE < longest) {
                if (step * PA_TILE + PA_TILE <= shortest && cur_odd == 0) work(tiles[buf], step, std::false_type{});
                else work(tiles[buf], step, std::true_type{});
            }
            if (more) {
                put(tiles[buf ^ 1]);
                cur_k = k_ref;
                cur_v = v_ref;
                cur_odd = next_odd;
                if (step + 2 < z) find(step + 2);
            }
            __syncthreads();
            buf ^= 1;
        }

        // ---- results ----
        const long long seg_t = (long long)h * steps + R.before;
        const int first = (int)(seg_t / share), pieces = (int)((seg_t + nt - 1) / share) - first + 1;
        {
            const pa_u2 w = __builtin_amdgcn_permlane32_swap(__float_as_uint(l_run), __float_as_uint(l_run), false, false);
            l_run = __uint_as_float(w[0]) + __uint_as_float(w[1]);
        }
        const size_t rec = pa_rec(first, blockIdx.x - first);
        if (pieces > 1) {
            float* po = pl.o + (rec * PA_ROWS + wv * 32 + row) * HD + 4 * half;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    *reinterpret_cast<floatx4_t*>(po + 32 * dt + 8 * j) =
                        floatx4_t{o[dt][4 * j], o[dt][4 * j + 1], o[dt][4 * j + 2], o[dt][4 * j + 3]};
            if (half == 0) {
                pl.ml[(rec * PA_ROWS + wv * 32 + row) * 2] = m_run;
                pl.ml[(rec * PA_ROWS + wv * 32 + row) * 2 + 1] = l_run;
            }
            if (lane == 0) pl.ev[4 * rec + wv] = o_ref;
        } else if (r0 + row < rows) {
            T* po = out + ((size_t)(s.first + qi) * n_q + qh) * HD + 4 * half;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                for (int j = 0; j < 16; ++j)
                    st_act<T>(po + 32 * dt + 8 * (j >> 2) + (j & 3), l_run == 0.f ? 0.f : ldexpf(o[dt][j] / l_run, o_ref));
        }
        t += z - a;
        a = z;
    }
}

// Combine of the cut row blocks, and zeros for the rows that see nothing: grid (row blocks, n_kv, PA_ROWS / rows of a
// block), HD / 4 threads a row.
template <typename T, int HD>
__global__ __launch_bounds__(256) void attn_pages_prompt_combine_kernel(KvPages c, KvRows r, PaPlan pl, PaPrompt pp,
                                                                        T* __restrict__ out, int n_q) {
    constexpr int TD = HD / 4;
    if ((int)blockIdx.x >= pp.total[0]) return;
    const PaRowBlock R = pp.rb[blockIdx.x];
    const int h = blockIdx.y, G = n_q / c.n_kv, share = pp.total[2];
    const int rr = blockIdx.z * (256 / TD) + threadIdx.x / TD, d = threadIdx.x % TD * 4;
    const KvSeq s = kvp_place(r, R.b);
    const int ri = R.rb * PA_ROWS + rr;
    if (ri >= s.n * G) return;
    T* dst = out + ((size_t)(s.first + ri / G) * n_q + h * G + ri % G) * HD + d;
    if (R.steps == 0) {
        for (int e = 0; e < 4; ++e) st_act<T>(dst + e, 0.f);
        return;
    }
    const long long seg_t = (long long)h * pp.total[1] + R.before;
    const int first = (int)(seg_t / share), pieces = (int)((seg_t + R.steps - 1) / share) - first + 1;
    if (pieces == 1) return;
    float M = PA_NONE, L = 0.f;
    int EV = KVP_E_MIN;
    for (int i = 0; i < pieces; ++i) {
        const size_t rec = pa_rec(first, i);
        M = fmaxf(M, pl.ml[(rec * PA_ROWS + rr) * 2]);
        EV = max(EV, pl.ev[4 * rec + rr / 32]);
    }
    floatx4_t O = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int i = 0; i < pieces; ++i) {
        const size_t rec = pa_rec(first, i);
        const float f = __builtin_amdgcn_exp2f(pl.ml[(rec * PA_ROWS + rr) * 2] - M);
        L = fmaf(pl.ml[(rec * PA_ROWS + rr) * 2 + 1], f, L);
        O += *reinterpret_cast<const floatx4_t*>(pl.o + (rec * PA_ROWS + rr) * HD + d) *
             (f * pa_pow2(pl.ev[4 * rec + rr / 32] - EV));
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) st_act<T>(dst + e, L == 0.f ? 0.f : ldexpf(O[e] / L, EV));
}

// ---------------------------------------------------------------------------
// Host launchers
// ---------------------------------------------------------------------------
namespace vte {

static long long pa_up(long long x) { return (x + 15) / 16 * 16; }

// Blocks of the few-rows form: two per CU (their registers allow no more), and
// no more than the table's capacity has shares of four tiles.
static PaPlan rows_plan(const KvPages& c, const KvRows& r, int hd, int G, void* scratch, long long* bytes) {
    const long long segments = (long long)r.batch * c.n_kv;
    const long long tiles = segments * ((((long long)r.max_pages << c.page_log2) + PA_TILE - 1) / PA_TILE);
    PaPlan p;
    p.blocks = (int)std::min<long long>(2 * device_cus(), (tiles + 3) / 4);
    p.ncol = r.max_rows * G;
    const long long recs = 2LL * p.blocks;
    uint8_t* at = static_cast<uint8_t*>(scratch);
    long long n = 0;
    p.o = reinterpret_cast<float*>(at);
    n += pa_up(recs * p.ncol * hd * 4);
    p.ml = reinterpret_cast<float*>(at + n);
    n += pa_up(recs * p.ncol * 8);
    p.ev = reinterpret_cast<int*>(at + n);
    n += pa_up(recs * 4);
    p.seg = reinterpret_cast<int2*>(at + n);
    n += pa_up(segments * 8);
    *bytes = n;
    return p;
}
// Blocks of the many-rows form, likewise; at most `rbs` row blocks.
static PaPlan prompt_plan(const KvPages& c, const KvRows& r, int hd, int G, void* scratch, PaPrompt* pp, long long* rbs,
                          long long* bytes) {
    *rbs = ((long long)r.rows * G + PA_ROWS - 1) / PA_ROWS + r.batch;
    const long long steps = *rbs * c.n_kv * ((((long long)r.max_pages << c.page_log2) + PA_TILE - 1) / PA_TILE);
    PaPlan p;
    p.blocks = (int)std::min<long long>(2 * device_cus(), steps);
    p.ncol = PA_ROWS;
    p.seg = nullptr;
    const long long recs = 2LL * p.blocks;
    uint8_t* at = static_cast<uint8_t*>(scratch);
    long long n = 0;
    p.o = reinterpret_cast<float*>(at);
    n += pa_up(recs * PA_ROWS * hd * 4);
    p.ml = reinterpret_cast<float*>(at + n);
    n += pa_up(recs * PA_ROWS * 8);
    p.ev = reinterpret_cast<int*>(at + n);
    n += pa_up(recs * 16);
    pp->rb = reinterpret_cast<PaRowBlock*>(at + n);
    n += pa_up(*rbs * sizeof(PaRowBlock));
    pp->start = reinterpret_cast<PaStart*>(at + n);
    n += pa_up(p.blocks * sizeof(PaStart));
    pp->total = reinterpret_cast<int*>(at + n);
    n += 16;
    *bytes = n;
    return p;
}
static bool rows_form(const KvRows& r, int G) { return r.max_rows * G <= 16; }

long long attn_pages_scratch_bytes(const KvPages& c, const KvRows& r, int hd, int n_q) {
    const int G = n_q / c.n_kv;
    long long n, rbs;
    PaPrompt pp;
    if (rows_form(r, G)) rows_plan(c, r, hd, G, nullptr, &n);
    else prompt_plan(c, r, hd, G, nullptr, &pp, &rbs, &n);
    return n;
}

template <typename T, int HD>
static hipError_t attn_hd(const KvPages& c, const KvRows& r, const void* q, void* out, int n_q, float scale,
                          void* scratch, hipStream_t st) {
    const int G = n_q / c.n_kv;
    long long bytes;
    if (rows_form(r, G)) {
        const PaPlan p = rows_plan(c, r, HD, G, scratch, &bytes);
        hipLaunchKernelGGL((attn_pages_rows_kernel<T, HD>), dim3(p.blocks), dim3(256), 0, st, c, r, p, (const T*)q,
                           (T*)out, n_q, scale);
        hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
        hipLaunchKernelGGL((attn_pages_combine_kernel<T, HD>), dim3(r.batch * c.n_kv, p.ncol), dim3(256), 0, st, c, r,
                           p, (T*)out, n_q);
        return hipGetLastError();
    }
    long long rbs;
    PaPrompt pp;
    const PaPlan p = prompt_plan(c, r, HD, G, scratch, &pp, &rbs, &bytes);
    hipLaunchKernelGGL(attn_pages_plan_kernel, dim3(1), dim3(1024), 0, st, c, r, p, pp, n_q);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((attn_pages_prompt_kernel<T, HD>), dim3(p.blocks), dim3(256), 0, st, c, r, p, pp, (const T*)q,
                       (T*)out, n_q, scale);
    e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((attn_pages_prompt_combine_kernel<T, HD>), dim3((unsigned)rbs, c.n_kv, PA_ROWS * HD / 1024),
                       dim3(256), 0, st, c, r, p, pp, (T*)out, n_q);
    return hipGetLastError();
}
hipError_t attn_pages(const KvPages& c, const KvRows& r, int hd, bool f16, const void* q, void* out, int n_q,
                      float scale, void* scratch, hipStream_t st) {
#define PA_ATTN(T, HD) attn_hd<T, HD>(c, r, q, out, n_q, scale, scratch, st)
    if (hd == 128) return f16 ? PA_ATTN(__half, 128) : PA_ATTN(float, 128);
    return f16 ? PA_ATTN(__half, 64) : PA_ATTN(float, 64);
#undef PA_ATTN
}

}  // namespace vte
