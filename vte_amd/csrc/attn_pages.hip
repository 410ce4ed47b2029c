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
// the segments its share touches, its four waves taking every fourth tile.  Block
// i's piece of segment s is record i + s (each next piece raises one of them), and
// a segment that lies in one share needs none.
// ---------------------------------------------------------------------------
struct PaPlan {
    int blocks;              // grid of the main launch
    int ncol;                // columns of a record: max_rows * G
    float* ml;               // [blocks + segments][16][2]: maximum (log2), sum
    int* ev;                 // [blocks + segments]: exponent the record's sums are relative to
    float* o;                // [blocks + segments][ncol][HD]
    int2* seg;               // [segments]: first block, pieces
};

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
        const int rec = blockIdx.x + seg;
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
                *reinterpret_cast<floatx4_t*>(pl.o + ((size_t)rec * pl.ncol + cc) * HD + d) = O;
                if (d == 0) {
                    pl.ml[(size_t)rec * 32 + 2 * cc] = M;
                    pl.ml[(size_t)rec * 32 + 2 * cc + 1] = L;
                }
            }
        }
        if (tid == 0) {
            pl.ev[rec] = EV;
            if (a == 0) pl.seg[seg] = make_int2(first, pieces);
        }
        __syncthreads();
        t += z - a;
    }
}

// Combine of the segments that lie in several shares, and zeros for the rows that see nothing: grid (segments,
// ncol), HD / 4 threads per group of pieces.
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
    KvSeq s = kvp_seq(r, b);
    if (s.pos < 0) {  // not running: its rows are zeros
        const int at = r.row_start ? max(r.row_start[b], 0) : b;
        s.first = at;
        s.n = r.row_start ? min(min(r.row_start[b + 1], r.rows) - at, r.max_rows) : r.max_rows;
    }
    if (cc >= s.n * G) return;
    T* dst = out + ((size_t)(s.first + cc / G) * n_q + h * G + cc % G) * HD;
    if (s.pos < 0 || pa_tokens(s, cap) == 0) {
        if (g == 0)
            for (int e = 0; e < 4; ++e) st_act<T>(dst + d + e, 0.f);
        return;
    }
    const int2 sg = pl.seg[seg];
    if (sg.y == 1) return;
    const size_t rec = (size_t)sg.x + seg;
    const float* ml = pl.ml + rec * 32 + 2 * cc;
    float M = PA_NONE;
    int EV = KVP_E_MIN;
    for (int i = tid; i < sg.y; i += 256) {
        M = fmaxf(M, ml[(size_t)i * 32]);
        EV = max(EV, pl.ev[rec + i]);
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
            const float f = __builtin_amdgcn_exp2f(ml[(size_t)(i0 + tid) * 32] - M);
            l = fmaf(ml[(size_t)(i0 + tid) * 32 + 1], f, l);
            w_sh[tid] = f * pa_pow2(pl.ev[rec + i0 + tid] - EV);
        }
        __syncthreads();
#pragma unroll 4
        for (int i = g; i < n; i += GR)
            O += *reinterpret_cast<const floatx4_t*>(pl.o + ((rec + i0 + i) * pl.ncol + cc) * HD + d) * w_sh[i];
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
// Attention, one wave per (row, query head): online softmax token by token,
// dims over the lanes.
// ---------------------------------------------------------------------------
template <typename T, int HD>
__global__ __launch_bounds__(64) void attn_pages_kernel(KvPages c, KvRows r, const T* __restrict__ q,
                                                        T* __restrict__ out, int n_q, float scale) {
    constexpr int PL = HD / 64;  // dims a lane holds: lane + 64 j
    const int row = blockIdx.x, qh = blockIdx.y, lane = threadIdx.x;
    const int b = kvp_row_seq(r, row);
    if (b < 0) return;
    const KvSeq s = kvp_seq(r, b);
    const int i = row - s.first;
    if (s.pos >= 0 && (i < 0 || i >= s.n)) return;
    const int h = qh / (n_q / c.n_kv);
    const int len = s.pos < 0 ? 0 : kvp_len(min(s.pos, 1 << 30) + i, kvp_capacity(c, r));
    float qv[PL], o[PL], m = -INFINITY, l = 0.f;
#pragma unroll
    for (int j = 0; j < PL; ++j) {
        qv[j] = ld_act<T>(q + ((size_t)row * n_q + qh) * HD + lane + 64 * j);
        o[j] = 0.f;
    }
    for (int t = 0; t < len; ++t) {
        const int page = kvp_page(c, r, b, t >> c.page_log2);
        if (page < 0) {
            t |= (1 << c.page_log2) - 1;
            continue;
        }
        const int in_page = (t & ((1 << c.page_log2) - 1)) / KVP_BLOCK, p = t % KVP_BLOCK;
        const size_t at = (((size_t)page * c.n_kv + h) << (c.page_log2 - 4)) + in_page;
        float dot = 0.f;
#pragma unroll
        for (int j = 0; j < PL; ++j)
            dot += qv[j] * (float)((int)c.k[at * (KVP_BLOCK * HD) + p * HD + lane + 64 * j] - KVP_ZERO);
        const float sc = wave_sum(dot) * kvp_scale(c.k_exp[at]) * scale;
        const float mn = sc > m || sc != sc ? sc : m;
        const float corr = m == -INFINITY ? 0.f : expf(m - mn), w = expf(sc - mn);
        l = l * corr + w;
        const float wv = w * kvp_scale(c.v_exp[at]);
#pragma unroll
        for (int j = 0; j < PL; ++j)
            o[j] = o[j] * corr +
                   wv * (float)((int)c.v[at * (KVP_BLOCK * HD) + (lane + 64 * j) * KVP_BLOCK + p] - KVP_ZERO);
        m = mn;
    }
#pragma unroll
    for (int j = 0; j < PL; ++j)
        st_act<T>(out + ((size_t)row * n_q + qh) * HD + lane + 64 * j, l == 0.f ? 0.f : o[j] / l);
}

// ---------------------------------------------------------------------------
// Host launchers
// ---------------------------------------------------------------------------
namespace vte {

// Blocks of the few-rows form: two per CU (their registers allow no more), and
// no more than the table's capacity has shares of four tiles.
static PaPlan rows_plan(const KvPages& c, const KvRows& r, int hd, int G, void* scratch, long long* bytes) {
    const long long segments = (long long)r.batch * c.n_kv;
    const long long tiles = segments * ((((long long)r.max_pages << c.page_log2) + PA_TILE - 1) / PA_TILE);
    PaPlan p;
    p.blocks = (int)std::min<long long>(2 * device_cus(), (tiles + 3) / 4);
    p.ncol = r.max_rows * G;
    const long long recs = p.blocks + segments;
    auto up = [](long long x) { return (x + 15) / 16 * 16; };
    uint8_t* at = static_cast<uint8_t*>(scratch);
    long long n = 0;
    p.o = reinterpret_cast<float*>(at);
    n += up(recs * p.ncol * hd * 4);
    p.ml = reinterpret_cast<float*>(at + n);
    n += up(recs * 32 * 4);
    p.ev = reinterpret_cast<int*>(at + n);
    n += up(recs * 4);
    p.seg = reinterpret_cast<int2*>(at + n);
    n += up(segments * 8);
    *bytes = n;
    return p;
}
static bool rows_form(const KvRows& r, int G) { return r.max_rows * G <= 16; }

long long attn_pages_scratch_bytes(const KvPages& c, const KvRows& r, int hd, int n_q) {
    const int G = n_q / c.n_kv;
    long long n = 16;
    if (rows_form(r, G)) rows_plan(c, r, hd, G, nullptr, &n);
    return n;
}

template <typename T, int HD>
static hipError_t attn_hd(const KvPages& c, const KvRows& r, const void* q, void* out, int n_q, float scale,
                          void* scratch, hipStream_t st) {
    const int G = n_q / c.n_kv;
    if (!rows_form(r, G)) {
        hipLaunchKernelGGL((attn_pages_kernel<T, HD>), dim3(r.rows, n_q), dim3(64), 0, st, c, r, (const T*)q, (T*)out,
                           n_q, scale);
        return hipGetLastError();
    }
    long long bytes;
    const PaPlan p = rows_plan(c, r, HD, G, scratch, &bytes);
    hipLaunchKernelGGL((attn_pages_rows_kernel<T, HD>), dim3(p.blocks), dim3(256), 0, st, c, r, p, (const T*)q,
                       (T*)out, n_q, scale);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((attn_pages_combine_kernel<T, HD>), dim3(r.batch * c.n_kv, p.ncol), dim3(256), 0, st, c, r, p,
                       (T*)out, n_q);
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
