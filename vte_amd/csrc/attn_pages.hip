// Attention over the 8-bit paged KV cache (layout: kv_pages.h), gfx950: few rows
// of each sequence (decoded tokens) or many (prompt chunks).
//
// Algorithm: online softmax per chunk and log-sum-exp combine as in
// vte/compiler/templates/rdna/flash_attention_split_kv_partial.hip.template:31-120
// and flash_attention_split_kv_reduce.hip.template:14-67, with
//   s_t = scale 2^ek(t) q.K_t,  out = sum_t p_t 2^ev(t) V_t / sum_t p_t,  p_t = exp(s_t - max)
// over whole-number K and V.  Bytes become fp16 exactly (0x6400 | byte is 1024 +
// byte; minus 1152), so both products run on 16x16x32 or 32x32x16 fp16 MFMAs with
// no rounding of K or V.  With few rows the V scale is folded into the probability, as
// 2^14 2^(s_t - max + ev(t) - e): e is a whole number, at most 1 above the largest of
// what stands before it, so that the heaviest token's is 2^13 to 2^14, half the smallest
// fp16 is 2^-38 of it, and V of vanishing weight costs the others nothing.  A token that
// nobody sees adds its byte, 0..255, times probability 0: its exponent, which may be
// anything, is never used.
#include <algorithm>
#include <type_traits>
#include "attn_tile.h"
#include "kv_pages.h"

#define PA_TILE 64       // tokens of a wave's step: a lane group of 16 holds one block of 16
#define PA_P_LOG2 14     // probabilities are held as 2^14 p
#define PA_P_PARTS 2     // fp16 parts of a probability, a rounded one and a rounded rest: with one, fp16 results were off by up
                         // to 2.8e-4 of them, with two by the 2.1e-4 of their own rounding
#define PA_NONE (-3e38f) // running maximum before anything is seen

typedef _Float16 pa_h2 __attribute__((ext_vector_type(2)));
typedef float pa_f2 __attribute__((ext_vector_type(2)));
typedef unsigned pa_u2 __attribute__((ext_vector_type(2)));

// 8 bytes as 8 fp16 whole numbers (byte - 128), or `by` times them (one rounded operation; exact for a power of two
// from 2^-24 on).
__device__ __forceinline__ half8_t pa_half8(uint32_t a, uint32_t b, _Float16 by) {
    union {
        uint32_t u[4];
        pa_h2 h[4];
        half8_t v;
    } r;
    r.u[0] = __builtin_amdgcn_perm(0x64646464u, a, 0x04010400u);
    r.u[1] = __builtin_amdgcn_perm(0x64646464u, a, 0x04030402u);
    r.u[2] = __builtin_amdgcn_perm(0x64646464u, b, 0x04010400u);
    r.u[3] = __builtin_amdgcn_perm(0x64646464u, b, 0x04030402u);
    const _Float16 z = (_Float16)-1152.f * by;
    const pa_h2 f = {by, by}, m = {z, z};
#pragma unroll
    for (int i = 0; i < 4; ++i) r.h[i] = __builtin_elementwise_fma(r.h[i], f, m);
    return r.v;
}
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
__device__ __forceinline__ float pa_sum4(float v) {
    pa_u2 a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}
// Sums O = sum 2^(s_t - m) 2^(ev_t - e) V_t of two or more parts of a row's tokens, each relative to its own maximum m and
// exponent e, are joined by what they contribute: with M the largest m, relative to E, the smallest whole number from every
// (m - M) + e on, so the factor 2^((m - M) + (e - E)) is 1 at most and what vanishes is below 2^-126 of the heaviest part.  (By
// the largest e alone a part of great V and no weight, or of no token that the row sees, took the others' sums with it.)
#define PA_E_NONE (-300) // e of a part of no tokens, below all others
__device__ __forceinline__ float pa_weight(float m, int e, float M) { return ceilf((m - M) + (float)e); }  // its lower bound for E
__device__ __forceinline__ float pa_joined(float m, int e, float M, int E) { return __builtin_amdgcn_exp2f((m - M) + (float)(e - E)); }
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
//
// Bound by the cache's bytes where contexts are long: eight documents of 16384 to
// 65536 tokens, 168 MB, 37.2 us in all, 4.5 TB/s (a copy moves 5.0; fp32 q 37.7); by
// latencies where they are short: 2049 tokens 11.9 us (fp32 q 13.9), two launches, in the
// first four loads one after the other (positions, page, bytes, q) and a tile's work.  Bytes go from memory to registers, where a lane's 16 are its operand
// once permuted: no LDS, each is used once, and a wave has the next tile's under way
// (two blocks of 256 threads a CU is all that those registers leave).
// ---------------------------------------------------------------------------
struct PaPlan {
    int blocks;  // grid of the main launch
    int ncol;    // columns (rows of the second form) of a record
    float* ml;   // [2 blocks][ncol][2]: maximum (log2), sum
    int* ev;     // [2 blocks][ncol]: exponent that the sums are relative to (PA_E_NONE: nothing seen)
    float* o;    // [2 blocks][ncol][HD]
    int2* seg;   // [segments]: first block, pieces
};
// Record of piece i of a segment whose first block is `first`.
__device__ __forceinline__ size_t pa_rec(int first, int i) { return i == 0 ? 2 * (size_t)first + 1 : 2 * ((size_t)first + i); }

// Tokens that any row of sequence b sees.
__device__ __forceinline__ int pa_tokens(const KvSeq& s, int cap) {
    return s.n == 0 ? 0 : (s.n < cap - s.pos ? s.pos + s.n : cap);
}

// Windows (WIN).  A row at position p sees the tokens from p + 1 - window on and the first `sinks` ones, none behind itself.  Tiles
// that none of the rows at hand sees are left out: those that are walked are numbered through, `head` at the front and from
// there on those `skip` further.  (WIN false: all of them, and the kernels are those of the attention without windows.)
// A tile that some see whole costs as before, one at a window's edge two operations a score more.  64 sequences of 1000 to
// 65000 tokens, window 4096, 28 and 4 heads: 264 MB in 53.4 (two inputs in turn) to 58.1 us, 4.6 to 4.9 TB/s (a copy 5.1);
// one sequence 12.3 us in two launches, whatever its length; a chunk of 512 tokens after 32256, window 4096, 33 us, 392
// TFLOP/s.
struct PaWindow {
    int window, sinks;
};
struct PaSpan {
    int n, head, skip;
    template <bool WIN>
    __device__ __forceinline__ int real(int i) const { return WIN && i >= head ? i + skip : i; }
};
// Of rows from position `first` on, which see tokens below `end` (`end` 0: no rows).
template <bool WIN>
__device__ __forceinline__ PaSpan pa_span(int first, int end, const PaWindow& w) {
    const int nt = (end + PA_TILE - 1) / PA_TILE;
    if constexpr (!WIN) return PaSpan{nt, nt, 0};
    const int low = min(max(first + 1 - w.window, 0) / PA_TILE, nt);
    const int head = min((min(w.sinks, end) + PA_TILE - 1) / PA_TILE, low);
    return PaSpan{nt - (low - head), head, low - head};
}
// Which of the 16 tokens from t0 on a row sees, one bit each, where it sees those in [low, end) and below `sinks`.
__device__ __forceinline__ uint32_t pa_below(int n) { return n >= 16 ? 0xFFFFu : n <= 0 ? 0u : (1u << n) - 1; }
__device__ __forceinline__ uint32_t pa_seen(int t0, int low, int end, int sinks) {
    return pa_below(end - t0) & (~pa_below(low - t0) | pa_below(sinks - t0));
}

// The block's share [t, t_end) of all tiles, and the sequence that t lies in with
// the number of tiles before it.
struct PaShare {
    long long t, t_end, before;
    long long share;
    int b;
    KvSeq s;
};
// Sum over the lanes up to and with this one: shifts by 1, 2, 4 and 8 in rows of 16 lanes, then the rows' last lanes into
// the rows behind them.
template <int CTRL, int ROWS>
__device__ __forceinline__ int pa_from(int v) {
    return __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xF, false);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ long long pa_from(long long v) {
    const unsigned lo = (unsigned)pa_from<CTRL, ROWS>((int)v);
    return (long long)((unsigned long long)(unsigned)pa_from<CTRL, ROWS>((int)(v >> 32)) << 32 | lo);
}
__device__ __forceinline__ long long pa_uniform(long long v) {  // the same in every lane: a scalar
    const unsigned lo = __builtin_amdgcn_readfirstlane((int)v);
    return (long long)((unsigned long long)(unsigned)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32 | lo);
}
template <typename V>
__device__ __forceinline__ V pa_scan(V v) {
    v += pa_from<0x111, 0xF>(v);
    v += pa_from<0x112, 0xF>(v);
    v += pa_from<0x114, 0xF>(v);
    v += pa_from<0x118, 0xF>(v);
    v += pa_from<0x142, 0xA>(v);
    v += pa_from<0x143, 0xC>(v);
    return v;
}
template <bool WIN>
__device__ __forceinline__ PaShare pa_share(const KvPages& c, const KvRows& r, int cap, int block, int blocks, const PaWindow& w) {
    __shared__ long long wsum[4];
    __shared__ long long found[5];
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    auto tiles = [&](const KvSeq& q) { return (long long)c.n_kv * pa_span<WIN>(q.pos, pa_tokens(q, cap), w).n; };
    auto cut = [&](PaShare& s, long long total) {
        // (a tile for each wave at least; whole rounds of four beyond that left CUs idle: eight documents of 16384 to
        // 65536 tokens 44.0 -> 41.3 us without, 16 ragged sequences 19.7 -> 18.3 us)
        s.share = max((total + blocks - 1) / blocks, 4LL);
        s.t = s.share * block;
        s.t_end = min(total, s.t + s.share);
    };
    if (r.batch <= 64) {  // every wave for itself, a sequence a lane
        const KvSeq q = kvp_seq(r, min(lane, r.batch - 1));
        const long long n = lane < r.batch ? tiles(q) : 0, incl = pa_scan(n);
        auto at = [](long long v, int l) {
            return (long long)((unsigned long long)(unsigned)__builtin_amdgcn_readlane((int)(v >> 32), l) << 32 |
                               (unsigned)__builtin_amdgcn_readlane((int)v, l));
        };
        PaShare s;
        cut(s, at(incl, 63));
        const uint64_t here = __ballot((s.t >= incl - n) & (s.t < incl));
        const int l = here ? __ffsll((unsigned long long)here) - 1 : 0;  // (none: a block without a share)
        s.b = l;
        s.before = at(incl - n, l);
        s.s.first = __builtin_amdgcn_readlane(q.first, l);
        s.s.n = __builtin_amdgcn_readlane(q.n, l);
        s.s.pos = __builtin_amdgcn_readlane(q.pos, l);
        return s;
    }
    const int per = (r.batch + 255) / 256;
    long long mine = 0;
    KvSeq mine_last = {0, 0, 0};
    for (int b = tid * per; b < min(r.batch, tid * per + per); ++b) {
        mine_last = kvp_seq(r, b);
        mine += tiles(mine_last);
    }
    long long incl = pa_scan(mine);
    if (lane == 63) wsum[wv] = incl;
    __syncthreads();
    const long long w4[4] = {wsum[0], wsum[1], wsum[2], wsum[3]};
    incl += wv > 2 ? w4[0] + w4[1] + w4[2] : wv > 1 ? w4[0] + w4[1] : wv > 0 ? w4[0] : 0;
    const long long total = pa_uniform(w4[0] + w4[1] + w4[2] + w4[3]);
    PaShare s;
    cut(s, total);
    if (mine > 0 && s.t >= incl - mine && s.t < incl) {
        long long before = incl - mine;
        int b = tid * per;
        KvSeq q = mine_last;
        if (per > 1)
            for (;; ++b) {
                q = kvp_seq(r, b);
                const long long n = tiles(q);
                if (s.t < before + n) break;
                before += n;
            }
        found[0] = b;
        found[1] = before;
        found[2] = q.first;
        found[3] = q.n;
        found[4] = q.pos;
    }
    __syncthreads();
    s.b = __builtin_amdgcn_readfirstlane((int)found[0]);
    s.before = pa_uniform(found[1]);
    s.s.first = __builtin_amdgcn_readfirstlane((int)found[2]);
    s.s.n = __builtin_amdgcn_readfirstlane((int)found[3]);
    s.s.pos = __builtin_amdgcn_readfirstlane((int)found[4]);
    return s;
}

// Bytes that are read once, whole lines at a time: not kept in the caches (V of the few-rows form: eight documents of 16384 to
// 65536 tokens 40.8 -> 36.0 us; K, of which a load takes half a line, 39.1).
__device__ __forceinline__ uint4 pa_once(const uint8_t* p) {
    const vte_u32x4 v = __builtin_nontemporal_load((vte_g_u32x4*)p);
    return make_uint4(v.x, v.y, v.z, v.w);
}

// One wave's tile: K rows (lane: row col of each of the four 16-row tiles) and V (lane: dim col, block grp).
template <int HD>
struct PaTile {
    uint4 k[4][HD / 64], v[HD / 16];
    int ek, ev;
    bool has;  // the lane's block has a page
};

template <typename T, int HD, bool WIN>
__global__ __launch_bounds__(256, 2) void attn_pages_rows_kernel(KvPages c, KvRows r, PaPlan pl,
                                                                 const T* q, T* out, int n_q,
                                                                 float scale, PaWindow w) {
    constexpr int PARTS = sizeof(T) == 4 ? 2 : 1;  // fp16 parts of q
    constexpr int KC = HD / 64;                    // 16-byte pieces of a K row that a lane holds
    constexpr int DT = HD / 16;
    __shared__ float m_sh[4][16], l_sh[4][16];
    __shared__ int ev_sh[4][16];
    __shared__ __align__(16) float o_sh[4][16][HD + 4];
    const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 15, grp = lane >> 4;
    const int G = n_q / c.n_kv, cap = kvp_capacity(c, r);
    const int bl = c.page_log2 - 4;  // log2 of a page's blocks
    PaShare sh = pa_share<WIN>(c, r, cap, blockIdx.x, pl.blocks, w);
    int b = sh.b;
    long long t = sh.t, before = sh.before;
    KvSeq s = sh.s;

    while (t < sh.t_end) {
        const int len = pa_tokens(s, cap);
        const PaSpan span = pa_span<WIN>(s.pos, len, w);
        const int nt = span.n;
        if (t - before >= (long long)nt * c.n_kv) {  // the next sequence
            before += (long long)nt * c.n_kv;
            s = kvp_seq(r, ++b);
            s.first = __builtin_amdgcn_readfirstlane(s.first);
            s.n = __builtin_amdgcn_readfirstlane(s.n);
            s.pos = __builtin_amdgcn_readfirstlane(s.pos);
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
        const int low = WIN ? max(s.pos + qi + 1 - w.window, 0) : 0;
        // K row of 16-row tile tt: token 16 (col / 4) + 4 tt + col % 4, so that the scores a lane gets from the four
        // tiles are those of block grp in order, which is the order V's 16 bytes hold its tokens in.
        auto load = [&](PaTile<HD>& x, int tile) {
            const int t0 = span.template real<WIN>(tile) * PA_TILE;
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
            for (int dt = 0; dt < DT; ++dt) x.v[dt] = pa_once(vr + 256 * dt);
        };
        PaTile<HD> A, B;
        int tile = a + wv;
        if (tile < z) load(A, tile);  // (asked for before q, whose turning into fp16 would hold it up)

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
        int ev_ref = PA_E_NONE;  // exponent that o is relative to
        floatx4_t o[DT];  // lane: column col, dims 16 dt + 4 grp + i
#pragma unroll
        for (int i = 0; i < DT; ++i) o[i] = floatx4_t{0.f, 0.f, 0.f, 0.f};

        auto step = [&](const PaTile<HD>& x, int tile) {
            const int p0 = span.template real<WIN>(tile) * PA_TILE + 16 * grp;  // this lane group's block
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
            uint32_t bits = 0;                      // (with a window)
            if constexpr (WIN) bits = x.has ? pa_seen(p0, low, end, w.sinks) : 0;
            // x where the column sees place i of the block, else `other`; with a window by the bit as a mask (one token of one
            // sequence 12.9 -> 12.4 us; with fp32 q and heads of 128, where masks cost registers that there are not, by the bit)
            auto seen_or = [&](int i, float x, uint32_t other) {
                if constexpr (WIN && PARTS * HD == 256) {
                    return (bits >> i & 1) != 0 ? x : __uint_as_float(other);
                } else if constexpr (WIN) {
                    const uint32_t m = (uint32_t)__builtin_amdgcn_sbfe((int)bits, i, 1);
                    return __uint_as_float((m & __float_as_uint(x)) | (~m & other));
                } else {
                    return i < live ? x : __uint_as_float(other);
                }
            };
            float top = -INFINITY;  // of this lane group's block
#pragma unroll
            for (int tt = 0; tt < 4; ++tt)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    sc[tt][i] = seen_or(4 * tt + i, sc[tt][i] * kf, 0xFF800000u);
                    top = fmaxf(top, sc[tt][i]);
                }
            const float mx = fmaxf(m_run, pa_max4(top));
            const int evm = (int)fmaxf(fmaxf(pa_max4(pa_weight(top, x.ev, mx)), pa_weight(m_run, ev_ref, mx)), (float)PA_E_NONE);
            if (__any((mx > m_run) | (evm > ev_ref))) {
                l_run *= __builtin_amdgcn_exp2f(m_run - mx);
                const float both = pa_joined(m_run, ev_ref, mx, evm);
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) o[dt] *= both;
                m_run = mx;
                ev_ref = evm;
            }
            // (a NaN block's tokens are NaN to the columns that see them and nothing to the others)
            const float d = x.ev == KVP_E_NAN ? NAN : (float)(x.ev - evm + PA_P_LOG2);
            half8_t pa[PA_P_PARTS][2];
#pragma unroll
            for (int tt = 0; tt < 4; ++tt)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float y = sc[tt][i] - mx;
                    l_run += __builtin_amdgcn_exp2f(y);
                    const float p = seen_or(4 * tt + i, __builtin_amdgcn_exp2f(y + d), 0u);
                    const int u = tt >> 1, j = 4 * (tt & 1) + i;
                    pa[0][u][j] = (_Float16)p;
                    pa[1][u][j] = (_Float16)(p - (float)pa[0][u][j]);
                }
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
                const half8_t v0 = pa_half8(x.v[dt].x, x.v[dt].y), v1 = pa_half8(x.v[dt].z, x.v[dt].w);
#pragma unroll
                for (int p = 0; p < PA_P_PARTS; ++p) {
                    o[dt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, pa[p][0], o[dt], 0, 0, 0);
                    o[dt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, pa[p][1], o[dt], 0, 0, 0);
                }
            }
        };

        // ---- the wave's tiles, the next one's loads under this one's work ----
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
            ev_sh[wv][col] = ev_ref;
        }
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) *reinterpret_cast<floatx4_t*>(&o_sh[wv][col][16 * dt + 4 * grp]) = o[dt];
        __syncthreads();
        const int seg = b * c.n_kv + h;
        const int first = (int)(seg_t / sh.share), pieces = (int)((seg_t + nt - 1) / sh.share) - first + 1;
        const size_t rec = pa_rec(first, blockIdx.x - first);
        for (int i = tid; i < ncol * (HD / 4); i += 256) {
            const int cc = i / (HD / 4), d = i % (HD / 4) * 4;
            const float M = fmaxf(fmaxf(m_sh[0][cc], m_sh[1][cc]), fmaxf(m_sh[2][cc], m_sh[3][cc]));
            float top = (float)PA_E_NONE;
#pragma unroll
            for (int w = 0; w < 4; ++w) top = fmaxf(top, pa_weight(m_sh[w][cc], ev_sh[w][cc], M));
            const int EV = (int)top;
            float L = 0.f;
            floatx4_t O = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                L = fmaf(l_sh[w][cc], __builtin_amdgcn_exp2f(m_sh[w][cc] - M), L);
                O += *reinterpret_cast<const floatx4_t*>(&o_sh[w][cc][d]) * pa_joined(m_sh[w][cc], ev_sh[w][cc], M, EV);
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
                    pl.ev[rec * pl.ncol + cc] = EV;
                }
            }
        }
        if (tid == 0 && a == 0) pl.seg[seg] = make_int2(first, pieces);
        __syncthreads();
        t += z - a;
    }
}

// Combine of the segments that were cut, and zeros for the rows that see nothing:
// grid (segments, ncol), HD / 4 threads per group of pieces.
template <typename T, int HD, bool WIN>
__global__ __launch_bounds__(256) void attn_pages_combine_kernel(KvPages c, KvRows r, PaPlan pl, T* __restrict__ out,
                                                                 int n_q, PaWindow win) {
    constexpr int TD = HD / 4, GR = 256 / TD;  // threads of a row, groups of pieces
    __shared__ float w_sh[256];
    __shared__ __align__(16) float o_sh[GR][HD + 4];
    __shared__ float red[4];
    const int seg = blockIdx.x, cc = blockIdx.y, b = seg / c.n_kv, h = seg - b * c.n_kv, tid = threadIdx.x;
    const int lane = tid & 63, wv = tid >> 6, g = tid / TD, d = tid % TD * 4;
    const int G = n_q / c.n_kv, cap = kvp_capacity(c, r);
    const KvSeq s = kvp_place(r, b);
    if (cc >= s.n * G) return;
    T* dst = out + ((size_t)(s.first + cc / G) * n_q + h * G + cc % G) * HD;
    // (a window may lie behind the table)
    if (s.pos < 0 || (WIN && pa_span<WIN>(s.pos, pa_tokens(s, cap), win).n == 0)) {
        if (tid < HD) st_act<T>(dst + tid, 0.f);
        return;
    }
    const int2 sg = pl.seg[seg];
    if (sg.y == 1) return;
    auto sums = [&](int i) {
        return *reinterpret_cast<const floatx4_t*>(pl.o + (pa_rec(sg.x, i) * pl.ncol + cc) * HD + d);
    };
    floatx4_t early[2];  // the group's first pieces, under the way to their weights
#pragma unroll
    for (int u = 0; u < 2; ++u) early[u] = sums(min(g + u * GR, sg.y - 1));
    // every wave for itself, its first 64 pieces requested together
    auto max_of = [&](int i) { return pl.ml[(pa_rec(sg.x, i) * pl.ncol + cc) * 2]; };
    auto exp_of = [&](int i) { return pl.ev[pa_rec(sg.x, i) * pl.ncol + cc]; };
    const float m0 = max_of(min(lane, sg.y - 1));
    const int e0 = exp_of(min(lane, sg.y - 1));
    float M = m0;
    for (int i = 64 + lane; i < sg.y; i += 64) M = fmaxf(M, max_of(i));
    M = wave_max(M);
    float top = fmaxf(pa_weight(m0, e0, M), (float)PA_E_NONE);
    for (int i = 64 + lane; i < sg.y; i += 64) top = fmaxf(top, pa_weight(max_of(i), exp_of(i), M));
    const int EV = (int)wave_max(top);
    float l = 0.f;
    floatx4_t O = {0.f, 0.f, 0.f, 0.f};
    for (int i0 = 0; i0 < sg.y; i0 += 256) {  // 256 pieces at a time
        const int n = min(256, sg.y - i0);
        if (tid < n) {
            const size_t rec = pa_rec(sg.x, i0 + tid);
            const float m = pl.ml[(rec * pl.ncol + cc) * 2];
            l = fmaf(pl.ml[(rec * pl.ncol + cc) * 2 + 1], __builtin_amdgcn_exp2f(m - M), l);
            w_sh[tid] = pa_joined(m, pl.ev[rec * pl.ncol + cc], M, EV);
        }
        __syncthreads();
        if (i0 == 0) {
#pragma unroll
            for (int u = 0; u < 2; ++u)
                if (g + u * GR < n) O += early[u] * w_sh[g + u * GR];
        }
#pragma unroll 4
        for (int i = g + (i0 == 0 ? 2 * GR : 0); i < n; i += GR) O += sums(i0 + i) * w_sh[i];
        __syncthreads();
    }
    l = wave_sum(l);
    if (lane == 0) red[wv] = l;
    *reinterpret_cast<floatx4_t*>(&o_sh[g][d]) = O;
    __syncthreads();
    const float L = (red[0] + red[1]) + (red[2] + red[3]);
    if (tid < HD) {
        float x = 0.f;
#pragma unroll
        for (int i = 0; i < GR; ++i) x += o_sh[i][tid];
        st_act<T>(dst + tid, L == 0.f ? 0.f : ldexpf(x / L, EV - PA_P_LOG2));
    }
}

// ---------------------------------------------------------------------------
// Many rows.  Rows of a KV head are numbered (new row, query head of the group),
// so a group of any size fills 32-row MFMA tiles; 256 or 128 of them are a row
// block and see tokens up to their last row's position, in steps of 64.  One block
// of threads takes a row block, or while these are fewer than the CUs one of nsp
// equal shares of its steps (joined by a second launch).
//
// The block's eight waves hold 32 rows each (GROUPS = 1; with short windows also
// four of them, blocks of which share a CU), or are two groups of
// four that take every other step and whose sums meet in LDS at the end (GROUPS =
// 2: half as many rows, so twice as many blocks or half as many shares).  The bytes
// of a step become fp16 once per group on their way into LDS, times 2^(e - ref)
// with ref the largest exponent of the step (K) or so far (V), so a step's scores
// and sums have one scale.  That is exact while no block lies below 2^-24 of ref
// (PA_APART).  A probability is off by up to 2^-34 of its row's largest (half the
// smallest fp16 of 2^9 p), times its V: V scales further apart than 2^12 in a group's
// steps (PA_APART_V; 2^-22 a token) would let that reach a result of smaller tokens.
// And a row's result must not depend on how large tokens are that it does not see.
// So a wave that met such blocks, or a score beyond 2^20, does its rows over, block by
// block (pa_apart, some ten times as long).  Scores are K.Q^T, sums are
// V^T.P^T (a lane is a row in both), K rows are read with token bits 2 and 3
// swapped so that a lane's scores are its operand of the second product as they
// stand.
//
// Bound by issue: a group's step is 48 products a wave (1500 cycles; fp32 q 64, heads of
// 64 half as many) beside some 500 cycles of turning bytes and 1200 of softmax and
// splitting probabilities, with two waves a SIMD, which overlap in part: 2.8 us for two
// groups' steps (fp32 q 3.0, heads of 64 2.1 and 2.2).  The runs below fix what stands between two products (left to
// itself the compiler read an operand right before each).  Beside that a block starts
// (3 us: sequence, page, bytes, the first tile) and ends (2 us), which weighs on short
// ones: four sequences of 2048 new tokens, 32 query and 8 KV heads of 128, 222 to 230 us,
// 600 to 620 TFLOP/s (a large fp16 matrix product: 1100 to 1200; the second part of the
// probabilities is not counted, but takes a third of the products); a chunk of 512 after
// 1536 tokens, in shares of 8 steps, 24.3 us, 232.
// ---------------------------------------------------------------------------
#define PA_SHARES 64
#define PA_APART 24 // scales of K blocks that are staged together, log2
#define PA_APART_V 12 // of V blocks whose sums are held together (below)
#define PA_LAG 6    // sums are rescaled when a maximum has grown by more than 2^6 ..
#define PA_Q_LOG2 9 // .. so probabilities are held as 2^9 p, at most 2^15

typedef float floatx16_t __attribute__((ext_vector_type(16)));
typedef float floatx8_t __attribute__((ext_vector_type(8), aligned(16)));

// Row block `slot` of all sequences' in their order: its sequence (-1: there are not so many) and number there.
// One wave, sequences over its lanes.
struct PaRowBlock {
    int b, rb;
    KvSeq s;  // with n the rows of a sequence that does not run, too
};
template <int ROWS>
__device__ __forceinline__ PaRowBlock pa_row_block(const KvRows& r, int G, int slot) {
    const int lane = threadIdx.x & 63;
    PaRowBlock R;
    R.b = -1;
    for (int b0 = 0; b0 < r.batch; b0 += 64) {
        const KvSeq s = kvp_place(r, min(b0 + lane, r.batch - 1));
        const int n = b0 + lane < r.batch ? (s.n * G + ROWS - 1) / ROWS : 0;
        const int incl = pa_scan(n);
        const uint64_t here = __ballot(slot < incl);
        if (here != 0) {
            const int l = __ffsll((unsigned long long)here) - 1;
            R.b = b0 + l;
            R.rb = slot - __builtin_amdgcn_readlane(incl - n, l);
            R.s.first = __builtin_amdgcn_readlane(s.first, l);
            R.s.n = __builtin_amdgcn_readlane(s.n, l);
            R.s.pos = __builtin_amdgcn_readlane(s.pos, l);
            return R;
        }
        slot -= __builtin_amdgcn_readlane(incl, 63);
    }
    return R;
}
// Steps of a row block, and the steps of one of its nsp shares (even: both groups get as many).
template <int ROWS, bool WIN>
__device__ __forceinline__ PaSpan pa_steps(const PaRowBlock& R, int G, int cap, const PaWindow& w) {
    if (R.s.pos < 0) return PaSpan{0, 0, 0};
    const int last = min((R.rb * ROWS + ROWS - 1) / G, R.s.n - 1);
    return pa_span<WIN>(R.s.pos + R.rb * ROWS / G, R.s.pos < cap - last ? R.s.pos + last + 1 : cap, w);
}
__device__ __forceinline__ int pa_share_of(int steps, int nsp) {
    return nsp == 1 ? steps : ((steps + nsp - 1) / nsp + 1) / 2 * 2;
}

struct PaPrompt {
    int nsp;    // shares of a row block
    float* ml;  // [row blocks][n_kv][nsp][128][2]: maximum (log2), sum
    int* ev;    // [row blocks][n_kv][nsp][128]: exponent that the row's sums are relative to (PA_E_NONE: it sees nothing)
    float* o;   // [row blocks][n_kv][nsp][HD / 8][32-row tile][4 dims of 8][row][4]
};

// A row's results: dims 32 i + 8 (j / 4) + j % 4 from dst on.
template <typename T, int N>
__device__ __forceinline__ void pa_store(T* dst, const floatx16_t (&o)[N], float l, int ref) {
    const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            union {
                T t[4];
                uint2 u2;
                uint4 u4[sizeof(T) / 4 < 1 ? 1 : sizeof(T) / 4];
            } r;
#pragma unroll
            for (int e = 0; e < 4; ++e) st_act<T>(&r.t[e], l == 0.f ? 0.f : ldexpf(o[i][4 * j + e] * inv, ref));
            if constexpr (sizeof(T) == 2) *reinterpret_cast<uint2*>(dst + 32 * i + 8 * j) = r.u2;
            else *reinterpret_cast<uint4*>(dst + 32 * i + 8 * j) = r.u4[0];
        }
}

// The sums of a wave's rows over steps first, first + GROUPS, .. below z with one scale per block and row: K and V as
// whole numbers, scores in fp32 by two-element products, each row's sums relative to its heaviest block's 2^(s - m + ev)
// (ev_row, as pa_weight has it), weights in fp32.
// Blocks of the least exponent hold zeros, or values below 2^-119 that count as zeros beside larger ones: they alone do
// not lead here.
template <typename T, int HD, int GROUPS, bool WIN, int PARTS, int KS, int DT>
__device__ __forceinline__ void pa_apart(const KvPages& c, const int* table, int max_pages, int h, int first, int z,
                                         const PaSpan& span, int seg_end, int low, int end, int sinks, int half,
                                         const half8_t (&qb)[PARTS][KS], float c2, float& m_run, float& l_run, int& ev_row,
                                         floatx16_t (&o)[DT]) {
    const int bl = c.page_log2 - 4;
    m_run = PA_NONE;
    l_run = 0.f;
    ev_row = PA_E_NONE;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[dt][i] = 0.f;
    for (int at_step = 4 * first; at_step < 4 * z; at_step += at_step % 4 == 3 ? 4 * GROUPS - 3 : 1) {
        const int blk = 4 * span.template real<WIN>(at_step >> 2) + (at_step & 3);
        if (blk * KVP_BLOCK >= seg_end) break;
        const int page = table[min(blk >> bl, max_pages - 1)];
        if ((unsigned)page >= (unsigned)c.n_pages) continue;
        const size_t at = (((size_t)page * c.n_kv + h) << bl) + (blk & ((1 << bl) - 1));
        const int ek = c.k_exp[at], ev = c.v_exp[at], n = end - blk * KVP_BLOCK;  // places that the row sees
        const uint32_t bits = WIN ? pa_seen(blk * KVP_BLOCK, low, end, sinks) : 0;
        auto sees = [&](int t) { return WIN ? (bits >> t & 1) != 0 : t < n; };
        const uint8_t* kr = c.k + at * (KVP_BLOCK * HD) + 8 * half;
        const uint8_t* vr = c.v + at * (KVP_BLOCK * HD) + 4 * half * KVP_BLOCK;
        float w[KVP_BLOCK], top = -INFINITY;  // of the block
        const float kf = kvp_scale(ek) * c2;
#pragma unroll
        for (int t = 0; t < KVP_BLOCK; ++t) {
            float s = 0.f;
#pragma unroll
            for (int i = 0; i < KS; ++i) {
                const uint2 b = *reinterpret_cast<const uint2*>(kr + t * HD + 16 * i);
                union {
                    half8_t v;
                    pa_h2 h[4];
                } k, x;
                k.v = pa_half8(b.x, b.y);
#pragma unroll
                for (int p = 0; p < PARTS; ++p) {
                    x.v = qb[p][i];
#pragma unroll
                    for (int j = 0; j < 4; ++j) s = __builtin_amdgcn_fdot2(k.h[j], x.h[j], s, false);
                }
            }
            const pa_u2 u = __builtin_amdgcn_permlane32_swap(__float_as_uint(s), __float_as_uint(s), false, false);
            w[t] = sees(t) ? (__uint_as_float(u[0]) + __uint_as_float(u[1])) * kf : -INFINITY;
            top = fmaxf(top, w[t]);
        }
        const float mx = fmaxf(m_run, top);
        const int evm = (int)fmaxf(fmaxf(pa_weight(m_run, ev_row, mx), pa_weight(top, ev, mx)), (float)PA_E_NONE);
        const float both = pa_joined(m_run, ev_row, mx, evm), d = ev == KVP_E_NAN ? NAN : (float)(ev - evm + PA_Q_LOG2);
        l_run *= __builtin_amdgcn_exp2f(m_run - mx);
#pragma unroll
        for (int t = 0; t < KVP_BLOCK; ++t) {
            const float x = w[t] - mx;
            l_run += __builtin_amdgcn_exp2f(x + (float)PA_Q_LOG2);
            w[t] = sees(t) ? __builtin_amdgcn_exp2f(x + d) : 0.f;
        }
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const uint4 b = ldg_g16(vr + (32 * dt + 8 * (i / 4) + i % 4) * KVP_BLOCK);
                const half8_t v0 = pa_half8(b.x, b.y), v1 = pa_half8(b.z, b.w);
                float x = o[dt][i] * both;
#pragma unroll
                for (int t = 0; t < 8; ++t) x = fmaf((float)v0[t], w[t], fmaf((float)v1[t], w[8 + t], x));
                o[dt][i] = x;
            }
        m_run = mx;
        ev_row = evm;
    }
    if (half) l_run = 0.f;  // (both halves hold the whole sum)
}

// grid (row blocks * n_kv, nsp), the last row blocks (which see most) first, whatever their head: with the heads one after
// the other some started long ones late (four ragged fp32 prompts 65 -> 53 us).  nsp > 1 with two groups only.
template <typename T, int HD, int GROUPS, int WAVES, bool WIN>
__global__ __launch_bounds__(64 * GROUPS * WAVES, GROUPS * WAVES == 4 && HD == 64 ? 3 : 2) void attn_pages_prompt_kernel(
    KvPages c, KvRows r, PaPrompt pp, const T* q, T* out, int n_q, float scale, PaWindow win) {
    constexpr int PARTS = sizeof(T) == 4 ? 2 : 1;  // fp16 parts of q
    constexpr int ROWS = 32 * WAVES;  // of a group
    constexpr int KS = HD / 16, DT = HD / 32;              // 16-dim steps of a score, 32-dim tiles
    constexpr int NP = 8 * HD / (64 * WAVES);              // 16-byte pieces of K and V a thread stages (1: waves 0..3 K, 4..7 V)
    // A lane's operand is 16 bytes of one token (K) or dim (V); those of neighbouring tokens or dims lie side by side, so
    // that reads touch every bank once (with a token's two pieces side by side they took twice as long).
    constexpr int KROW = PA_TILE * 8 + 8;  // halves of 8 dims of K, 64 tokens; rows of neighbouring dims 16 bytes apart in banks
    struct alignas(16) Tile {
        _Float16 k[2 * KS * KROW];     // [dims 8 half .. of 16][16-dim step][token][8 dims]
        _Float16 v[4 * 2 * HD * 8];    // [block][its 8 tokens][dim][8 tokens]
    };
    union Shared {
        Tile tiles[GROUPS][2];         // [group][buffer]
        float o[GROUPS][GROUPS == 2 ? DT / 2 * 16 : 1][64 * WAVES];  // what a group leaves to the other
    };
    __shared__ Shared S;
    __shared__ float m_sh[GROUPS][ROWS], l_sh[GROUPS][ROWS];
    __shared__ int ev_sh[GROUPS][ROWS];
    const int tid = threadIdx.x & (64 * WAVES - 1), lane = threadIdx.x & 63;
    const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) & (WAVES - 1);
    const int grp = GROUPS == 2 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 8) : 0;
    const int row = lane & 31, half = lane >> 5;
    const int G = n_q / c.n_kv, cap = kvp_capacity(c, r), bl = c.page_log2 - 4;
    const int slot = (gridDim.x - 1 - blockIdx.x) / c.n_kv, h = blockIdx.x % c.n_kv;
    const PaRowBlock R = pa_row_block<ROWS>(r, G, slot);
    if (R.b < 0) return;
    const KvSeq s = R.s;
    const PaSpan span = pa_steps<ROWS, WIN>(R, G, cap, win);
    const int steps = span.n, share = pa_share_of(steps, pp.nsp);
    const int a = blockIdx.y * share, z = min(steps, a + share), pieces = steps ? (steps + share - 1) / share : 1;
    if (a >= z && !(steps == 0 && blockIdx.y == 0)) return;
    const int* table = r.page_table + (size_t)R.b * r.max_pages;

    // ---- this lane's row ----
    const int r0 = R.rb * ROWS + wv * 32, rows = s.n * G;
    const int ri = min(r0 + row, rows - 1), qi = ri / G, qh = h * G + ri - qi * G;
    T* dst = out + ((size_t)(s.first + qi) * n_q + qh) * HD;
    if (steps == 0) {  // a sequence that does not run
        if (r0 + row < rows && grp == 0)
            for (int d = half * (HD / 2); d < (half + 1) * (HD / 2); ++d) st_act<T>(dst + d, 0.f);
        return;
    }
    const int end = r0 + row < rows ? kvp_len(s.pos + qi, cap) : 0;
    const int seg_end = kvp_len(s.pos + min((R.rb * ROWS + ROWS - 1) / G, s.n - 1), cap);  // of the row block
    const int shortest = r0 + 31 < rows ? kvp_len(s.pos + r0 / G, cap) : 0;  // of the wave
    const int low = WIN ? max(s.pos + qi + 1 - win.window, 0) : 0;
    const int lowest = WIN ? max(s.pos + min(r0 + 31, rows - 1) / G + 1 - win.window, 0) : 0;  // of the wave's last row

    // Staging: registers, then LDS.  Lane j & 3 knows block j's page and exponents; a wave's pieces lie in one block.
    uint4 stage[NP];
    // u: its part of K or V, the block and the first piece of it (of HD) that the wave's lanes take
    auto is_v = [&](int u) { return NP >= 2 ? u >= NP / 2 : wv >= WAVES / 2; };
    auto first = [&](int u) { return (NP >= 2 ? u % (NP / 2) * WAVES + wv : wv % (WAVES / 2)) * 64; };
    // (No branches here and in put, which stand in one run with the products; a page number is not looked at until
    // the step after the one in which it is asked for.)
    int ek, ev, page;
    bool got;  // block j of the step in the registers is of use
    auto find = [&](int i) {
        const int step = span.template real<WIN>(i);
        page = table[min((4 * step + (lane & 3)) >> bl, r.max_pages - 1)];
    };
    auto load = [&](int i0) {
        const int step = span.template real<WIN>(i0);
        const int blk = 4 * step + (lane & 3);
        const bool used = (i0 < z) & (blk * KVP_BLOCK < seg_end) & ((unsigned)page < (unsigned)c.n_pages);
        const size_t i = (((size_t)(used ? page : 0) * c.n_kv + h) << bl) + (blk & ((1 << bl) - 1));
        ek = c.k_exp[i];
        ev = c.v_exp[i];
#pragma unroll
        for (int u = 0; u < NP; ++u) {
            const int j = first(u) / HD, p = __builtin_amdgcn_readlane(used ? page : 0, j);
            const size_t at = (((size_t)p * c.n_kv + h) << bl) + ((4 * step + j) & ((1 << bl) - 1));
            stage[u] = ldg_g16((is_v(u) ? c.v : c.k) + at * (KVP_BLOCK * HD) + (first(u) % HD + lane) * 16);
        }
        got = used;
        find(i0 + GROUPS);
    };
    find(a + grp);
    // q is asked for while the page number is on its way.  The wave's 32 rows by lanes in 128-byte pieces, which change
    // places in LDS (a row a lane touches a line each: the first tile was there 1.2 us later), in the second buffer, which
    // nothing is put into before the first barrier; where that is too small, a row a lane.
    constexpr bool TURN_Q = sizeof(Tile) >= (size_t)WAVES * 4096;
    constexpr int QP = HD * (int)sizeof(T) / 128;  // pieces of a row
    typedef typename std::conditional<PARTS == 1, half8_t, floatx8_t>::type q8_t;
    q8_t q_raw[KS];
    uint4 q_piece[QP][4];
    if constexpr (TURN_Q) {
        const uint32_t inv = 0xFFFFFFFFu / (uint32_t)G + 1;  // ri / G = ri inv >> 32 for ri < 2^28, 1 < G <= 16
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int i = min(r0 + 8 * k + (lane >> 3), rows - 1), n = G == 1 ? i : (int)__umulhi((uint32_t)i, inv);
            const uint8_t* at = reinterpret_cast<const uint8_t*>(q + ((size_t)(s.first + n) * n_q + h * G + i - n * G) * HD) +
                                (lane & 7) * 16;
#pragma unroll
            for (int p = 0; p < QP; ++p) q_piece[p][k] = ldg_g16(at + 128 * p);
        }
    } else {
        const T* qp = q + ((size_t)(s.first + qi) * n_q + qh) * HD + 8 * half;
#pragma unroll
        for (int i = 0; i < KS; ++i) q_raw[i] = *reinterpret_cast<const q8_t*>(qp + 16 * i);
    }
    __builtin_amdgcn_sched_barrier(0);
    load(a + grp);
    if constexpr (TURN_Q) {
        uint4* to = reinterpret_cast<uint4*>(&S.tiles[grp][1]) + wv * 256;
        auto order = [] {  // of the wave's own LDS accesses
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        };
#pragma unroll
        for (int p = 0; p < QP; ++p) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int rr = 8 * k + (lane >> 3);
                to[rr * 8 + ((lane & 7) ^ (rr >> 1 & 7))] = q_piece[p][k];
            }
            order();
#pragma unroll
            for (int i = 0; i < KS / QP; ++i) {
                union {
                    uint4 u[sizeof(q8_t) / 16];
                    q8_t v;
                } x;
#pragma unroll
                for (int e = 0; e < (int)sizeof(q8_t) / 16; ++e)
                    x.u[e] = to[row * 8 + (((2 * i + half) * (int)sizeof(q8_t) / 16 + e) ^ (row >> 1 & 7))];
                q_raw[p * (KS / QP) + i] = x.v;
            }
            order();
        }
    }

    half8_t qb[PARTS][KS];
    float q_unit = 1.f;
    if constexpr (PARTS == 1) {
#pragma unroll
        for (int i = 0; i < KS; ++i) qb[0][i] = q_raw[i];
    } else {  // scaled by a power of two so that the second part keeps its bits too
        float amax = 0.f;
#pragma unroll
        for (int i = 0; i < KS; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) amax = fmaxf(amax, fabsf(q_raw[i][j]));
        amax = fmaxf(amax, __shfl_xor(amax, 32, 64));
        const int e = min(max((int)(__float_as_uint(amax) >> 23) - 127, -110), 126);  // 2^e <= amax
        const float up = __uint_as_float((uint32_t)(127 + 13 - e) << 23);
        q_unit = __uint_as_float((uint32_t)(127 - 13 + e) << 23);
#pragma unroll
        for (int i = 0; i < KS; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float y = q_raw[i][j] * up;
                qb[0][i][j] = (_Float16)y;
                qb[1][i][j] = (_Float16)(y - (float)qb[0][i][j]);
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
    int k_ref = KVP_E_MIN, v_ref = KVP_E_MIN;           // of the step staged last: its largest, the largest so far
    int next_odd = 0;                                   // its blocks without a page, and with NaN in V
    int apart = 0;                                      // some blocks' scales lie too far apart for all this
    int v_low = 1000;                                   // lane j & 3: the least V exponent of its blocks so far, zeros aside
    int by_k = 0, by_v = 0;                             // lane j & 3: block j's factors, fp16
    auto scales = [&] {
        const int my_k = got ? ek : -1000, my_v = got ? ev : -1000;  // -1000: times 0
        auto max4 = [](int x) {                                      // of the four blocks
            x = max(x, __builtin_amdgcn_update_dpp(0, x, 0xB1, 0xF, 0xF, false));
            return __builtin_amdgcn_readfirstlane(max(x, __builtin_amdgcn_update_dpp(0, x, 0x4E, 0xF, 0xF, false)));
        };
        k_ref = max(max4(my_k), KVP_E_MIN);
        v_ref = max(max4(my_v), v_ref);
        v_low = my_v > KVP_E_MIN ? min(v_low, my_v) : v_low;
        next_odd = (int)(__ballot(!got) & 15) | (int)(__ballot(my_v == KVP_E_NAN) & 15) << 4;
        apart |= ((my_k > KVP_E_MIN) & (my_k < k_ref - PA_APART)) | (v_low < v_ref - PA_APART_V);
        // (NaN in V is dealt with where its rows are: 0 times it would reach rows that do not see it)
        by_k = my_k == KVP_E_NAN ? 0x7E00 : (int)__builtin_bit_cast(unsigned short, (_Float16)pa_pow2(my_k - k_ref));
        by_v = my_v == KVP_E_NAN ? 0 : (int)__builtin_bit_cast(unsigned short, (_Float16)pa_pow2(my_v - v_ref));
    };
    auto put = [&](Tile& D, int u) {
        const int j = first(u) / HD, piece = first(u) % HD + lane;
        const int by16 = __builtin_amdgcn_readlane(is_v(u) ? by_v : by_k, j);
        const _Float16 by = __builtin_bit_cast(_Float16, (unsigned short)by16);
        // K piece: token piece / KS of the block, dims 16 (piece % KS) ..; V piece: dim `piece`
        _Float16* to = is_v(u) ? D.v + (2 * j * HD + piece) * 8
                               : D.k + (piece % KS) * KROW + (16 * j + piece / KS) * 8;
        *reinterpret_cast<half8_t*>(to) = pa_half8(stage[u].x, stage[u].y, by);
        *reinterpret_cast<half8_t*>(to + (is_v(u) ? HD * 8 : KS * KROW)) = pa_half8(stage[u].z, stage[u].w, by);
    };

    // K row of 32-token tile tt: token with bits 2 and 3 of the lane's row swapped
    const int kt = (row & 0x13) | (row & 4) << 1 | (row & 8) >> 1;
    // `ends`: some of the wave's rows do not see all of the step, or a block of it has no page or NaN in V
    auto work = [&](const Tile& D, Tile& next, int i0, int step, bool ends) {
        const int cur_k = k_ref, cur_v = v_ref, cur_odd = next_odd;
        // Scores: under every four products the next four operands are read and a part of the next step's bytes is turned.
        constexpr int RUN = 4, RUNS = 2 * KS / RUN;
        floatx16_t sc[2];
        half8_t kb[2][RUN];
        auto read_k = [&](int u) {  // tile u / KS, 16-dim step u % KS
            return *reinterpret_cast<const half8_t*>(D.k + (half * KS + u % KS) * KROW + (32 * (u / KS) + kt) * 8);
        };
#pragma unroll
        for (int u = 0; u < RUN; ++u) kb[0][u] = read_k(u);
        scales();
#pragma unroll
        for (int tt = 0; tt < 2; ++tt)
#pragma unroll
            for (int j = 0; j < 16; ++j) sc[tt][j] = 0.f;
#pragma unroll
        for (int n = 0; n < RUNS; ++n) {
            __builtin_amdgcn_sched_barrier(0);
            if (n + 1 < RUNS)
#pragma unroll
                for (int u = 0; u < RUN; ++u) kb[n + 1 & 1][u] = read_k((n + 1) * RUN + u);
#pragma unroll
            for (int u = n * RUN; u < (n + 1) * RUN; ++u)
#pragma unroll
                for (int p = 0; p < PARTS; ++p)
                    sc[u / KS] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kb[n & 1][u % RUN], qb[p][u % KS], sc[u / KS], 0, 0, 0);
#pragma unroll
            for (int u = n * NP / RUNS; u < (n + 1) * NP / RUNS; ++u) put(next, u);
            __builtin_amdgcn_sched_group_barrier(0x100, RUN, 0);
#pragma unroll
            for (int i = 0; i < RUN * PARTS; ++i) {
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x002, 6 / PARTS, 0);
            }
        }
        __builtin_amdgcn_sched_barrier(0);
        load(i0 + 2 * GROUPS);
        // lane: its row's scores of tokens 32 tt + 16 (j / 8) + 8 half + j % 8
        const int live = end - step * PA_TILE - 8 * half;
        if (ends) {
#pragma unroll
            for (int kb = 0; kb < 4; ++kb) {
                const int n = cur_odd >> kb & 1 ? 0 : live - 16 * kb;
                uint32_t bits = 0;
                if constexpr (WIN) bits = cur_odd >> kb & 1 ? 0 : pa_seen(step * PA_TILE + 16 * kb + 8 * half, low, end, win.sinks);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int i = 8 * (kb & 1) + j;
                    if constexpr (WIN) {  // (the bit as a mask: two operations a score)
                        const uint32_t m = (uint32_t)__builtin_amdgcn_sbfe((int)bits, j, 1);
                        sc[kb >> 1][i] = __uint_as_float((m & __float_as_uint(sc[kb >> 1][i])) | (~m & 0xFF800000u));
                    } else {
                        sc[kb >> 1][i] = j < n ? sc[kb >> 1][i] : -INFINITY;
                    }
                }
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
        const float kf = fmaxf(kvp_scale(cur_k) * c2, 1e-38f);  // (not 0: masked scores are -Inf)
        mx = fmaxf(m_run, mx * kf);
        if (__any(mx > m_run + (float)PA_LAG) || cur_v > o_ref) {
            const float corr = __builtin_amdgcn_exp2f(m_run - mx);
            l_run *= corr;
            const float both = corr * pa_pow2(o_ref - cur_v);
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) o[dt] *= both;
            m_run = mx;
            o_ref = cur_v;
            // (products enter the exponent unrounded, their maximum rounded: beyond 2^20 that is too far apart)
            apart |= (fabsf(mx) > 1048576.f) & (mx > PA_NONE);
        }
        if (cur_odd >> 4) {  // NaN in V: the sums of the rows that see a token of its block
#pragma unroll
            for (int kb = 0; kb < 4; ++kb)
                if ((cur_odd >> (4 + kb) & 1) && (WIN ? pa_seen(step * PA_TILE + 16 * kb, low, end, win.sinks) != 0
                                                      : end - step * PA_TILE > 16 * kb)) {
#pragma unroll
                    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                        for (int j = 0; j < 16; ++j) o[dt][j] = NAN;
                }
        }
        // Sums: a block's probabilities are formed, and the one's V behind it read, under its products.
        const float shift = (float)PA_Q_LOG2 - m_run;
        const pa_h2 ones = {(_Float16)1.f, (_Float16)1.f};
        float l_odd = 0.f;
        float minus = -1.f;  // (a value that the compiler does not know: p - h as one mixed operation instead of two)
        asm("" : "+v"(minus));
        union Probs {
            half8_t v;
            pa_h2 h[4];
        } pf[2][PA_P_PARTS];
        half8_t vb[2][DT];
        auto probs = [&](int kb) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {  // the sum of the probabilities as the products have them
                const int j = 8 * (kb & 1) + 2 * i;
                const float p0 = __builtin_amdgcn_exp2f(fmaf(sc[kb >> 1][j], kf, shift));
                const float p1 = __builtin_amdgcn_exp2f(fmaf(sc[kb >> 1][j + 1], kf, shift));
                Probs(&f)[PA_P_PARTS] = pf[kb & 1];
                f[0].h[i] = __builtin_convertvector(pa_f2{p0, p1}, pa_h2);
                const pa_h2 h = f[0].h[i];
                f[1].h[i] = __builtin_convertvector(pa_f2{fmaf((float)h[0], minus, p0), fmaf((float)h[1], minus, p1)}, pa_h2);
                if constexpr (WIN) {
                    l_run += p0;
                    l_odd += p1;
                } else {
                    l_run = __builtin_amdgcn_fdot2(f[0].h[i], ones, l_run, false);
                    l_run = __builtin_amdgcn_fdot2(f[1].h[i], ones, l_run, false);
                }
            }
        };
        auto read_v = [&](int kb) {
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
                vb[kb & 1][dt] = *reinterpret_cast<const half8_t*>(D.v + ((2 * kb + half) * HD + 32 * dt + row) * 8);
        };
        read_v(0);
        probs(0);
#pragma unroll
        for (int kb = 0; kb < 4; ++kb) {
            __builtin_amdgcn_sched_barrier(0);
            if (kb < 3) read_v(kb + 1);
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                for (int p = 0; p < PA_P_PARTS; ++p)
                    o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vb[kb & 1][dt], pf[kb & 1][p].v, o[dt], 0, 0, 0);
            if (kb < 3) {
                probs(kb + 1);
                __builtin_amdgcn_sched_group_barrier(0x100, DT, 0);
#pragma unroll
                for (int i = 0; i < DT * PA_P_PARTS; ++i) {
                    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                    __builtin_amdgcn_sched_group_barrier(0x402, 40 / (DT * PA_P_PARTS) + 1, 0);
                }
            }
        }
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (WIN) l_run += l_odd;
    };

    scales();
#pragma unroll
    for (int u = 0; u < NP; ++u) put(S.tiles[grp][0], u);
    load(a + grp + GROUPS);
    __syncthreads();
    int buf = 0;
    // (A group without a last step, and a wave whose rows end before the block's, go along with everything masked.)
    for (int step = a + grp; step < z + grp; step += GROUPS) {
        const int at = span.template real<WIN>(step) * PA_TILE;
        const bool ends = at + PA_TILE > shortest || (WIN && at < lowest && at + PA_TILE > win.sinks);
        work(S.tiles[grp][buf], S.tiles[grp][buf ^ 1], step, at / PA_TILE, ends || next_odd != 0);
        __syncthreads();
        buf ^= 1;
    }

    int ev_row = o_ref;  // of this lane's row
    if (__any(apart))
        pa_apart<T, HD, GROUPS, WIN>(c, table, r.max_pages, h, a + grp, z, span, seg_end, low, end, win.sinks, half, qb, c2, m_run,
                                     l_run, ev_row, o);

    // ---- results ----
    {
        const pa_u2 w = __builtin_amdgcn_permlane32_swap(__float_as_uint(l_run), __float_as_uint(l_run), false, false);
        l_run = __uint_as_float(w[0]) + __uint_as_float(w[1]);
    }
    if (l_run == 0.f) ev_row = PA_E_NONE;  // (o_ref is of all tokens of its steps, whether the row sees one or not)
    if constexpr (GROUPS == 1) {
        if (r0 + row < rows) pa_store<T, DT>(dst + 4 * half, o, l_run, ev_row);
    } else {  // each group leaves half of the dims to the other
        if (half == 0) {
            m_sh[grp][wv * 32 + row] = m_run;
            l_sh[grp][wv * 32 + row] = l_run;
            ev_sh[grp][wv * 32 + row] = ev_row;
        }
        floatx16_t mine[DT / 2];
#pragma unroll
        for (int i = 0; i < DT / 2; ++i) {
            mine[i] = grp ? o[DT / 2 + i] : o[i];
            const floatx16_t other = grp ? o[i] : o[DT / 2 + i];
#pragma unroll
            for (int j = 0; j < 16; ++j) S.o[grp][16 * i + j][tid] = other[j];
        }
        __syncthreads();
        const float m2 = m_sh[grp ^ 1][wv * 32 + row], M = fmaxf(m_run, m2);
        const int e2 = ev_sh[grp ^ 1][wv * 32 + row];
        const int EV = (int)fmaxf(fmaxf(pa_weight(m_run, ev_row, M), pa_weight(m2, e2, M)), (float)PA_E_NONE);
        const float f1 = __builtin_amdgcn_exp2f(m_run - M), f2 = __builtin_amdgcn_exp2f(m2 - M);
        const float L = l_run * f1 + l_sh[grp ^ 1][wv * 32 + row] * f2;
        const float g1 = pa_joined(m_run, ev_row, M, EV), g2 = pa_joined(m2, e2, M, EV);
#pragma unroll
        for (int i = 0; i < DT / 2; ++i)
#pragma unroll
            for (int j = 0; j < 16; ++j) mine[i][j] = mine[i][j] * g1 + S.o[grp ^ 1][16 * i + j][tid] * g2;
        const int d0 = grp * (HD / 2) + 4 * half;  // first dim of mine
        if (pieces > 1) {
            const size_t rec = ((size_t)slot * c.n_kv + h) * pp.nsp + blockIdx.y;
            if (r0 + row >= rows) return;
            floatx4_t* po = reinterpret_cast<floatx4_t*>(pp.o + rec * ROWS * HD) + grp * (HD / 16) * 256 + tid;
#pragma unroll
            for (int i = 0; i < DT / 2; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    po[(4 * i + j) * 256] = floatx4_t{mine[i][4 * j], mine[i][4 * j + 1], mine[i][4 * j + 2], mine[i][4 * j + 3]};
            if (half == 0 && grp == 0) {
                pp.ml[(rec * ROWS + wv * 32 + row) * 2] = M;
                pp.ml[(rec * ROWS + wv * 32 + row) * 2 + 1] = L;
                pp.ev[rec * ROWS + wv * 32 + row] = EV;
            }
        } else if (r0 + row < rows) {
            pa_store<T, DT / 2>(dst + d0, mine, L, EV);
        }
    }
}

// Joins the shares of the row blocks: grid (row blocks, n_kv, HD / 8).  A block takes 32 rows and 32 dims, a wave 8 of
// them, as the records have them (1024 bytes on end a load); results change places in LDS: 64 or 128 bytes of a row together.
template <typename T, int HD, bool WIN>
__global__ __launch_bounds__(256) void attn_pages_prompt_combine_kernel(KvPages c, KvRows r, PaPrompt pp,
                                                                        T* __restrict__ out, int n_q, PaWindow win) {
    constexpr int ROWS = 128;
    const int slot = blockIdx.x, h = blockIdx.y, G = n_q / c.n_kv;
    const PaRowBlock R = pa_row_block<ROWS>(r, G, slot);
    if (R.b < 0) return;
    const int lane = threadIdx.x & 63, tile = blockIdx.z & 3, part = (blockIdx.z & ~3) + (threadIdx.x >> 6);
    const int rr = 32 * tile + (lane & 31), rows = R.s.n * G;
    __shared__ __align__(16) float o_sh[32][32 + 4];
    const int steps = pa_steps<ROWS, WIN>(R, G, kvp_capacity(c, r), win).n, share = pa_share_of(steps, pp.nsp);
    if (steps <= share || R.rb * ROWS + 32 * tile >= rows) return;
    const int pieces = (steps + share - 1) / share;
    const size_t rec0 = ((size_t)slot * c.n_kv + h) * pp.nsp;
    float M = PA_NONE, L = 0.f;
    int EV = PA_E_NONE;
    floatx4_t O = {0.f, 0.f, 0.f, 0.f};
    constexpr int AT_ONCE = 8;
    for (int i0 = 0; i0 < pieces; i0 += AT_ONCE) {  // requested together (past the last one: the last again)
        floatx4_t o[AT_ONCE];
        float2 ml[AT_ONCE];
        int ev[AT_ONCE];
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i) {
            const size_t rec = (rec0 + min(i0 + i, pieces - 1)) * ROWS + rr;
            o[i] = reinterpret_cast<const floatx4_t*>(pp.o + (rec - rr) * HD)[part * 256 + 64 * tile + lane];
            ml[i] = *reinterpret_cast<const float2*>(pp.ml + rec * 2);
            ev[i] = pp.ev[rec];
        }
        float m = M;
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i) m = fmaxf(m, ml[i].x);
        float x = fmaxf(pa_weight(M, EV, m), (float)PA_E_NONE);
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i) x = fmaxf(x, pa_weight(ml[i].x, ev[i], m));
        L *= __builtin_amdgcn_exp2f(M - m);
        O *= pa_joined(M, EV, m, (int)x);
        M = m;
        EV = (int)x;
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i) {
            const bool in = i0 + i < pieces;
            L = fmaf(ml[i].y, in ? __builtin_amdgcn_exp2f(ml[i].x - M) : 0.f, L);
            O += o[i] * (in ? pa_joined(ml[i].x, ev[i], M, EV) : 0.f);
        }
    }
    floatx4_t x;
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = L == 0.f ? 0.f : ldexpf(O[e] / L, EV);
    *reinterpret_cast<floatx4_t*>(&o_sh[lane & 31][8 * (threadIdx.x >> 6) + 4 * (lane >> 5)]) = x;
    __syncthreads();
    const int at = threadIdx.x >> 3, d = threadIdx.x % 8 * 4, ri = R.rb * ROWS + 32 * tile + at;
    if (ri >= rows) return;
    T* dst = out + ((size_t)(R.s.first + ri / G) * n_q + h * G + ri % G) * HD + (blockIdx.z >> 2) * 32 + d;
#pragma unroll
    for (int e = 0; e < 4; ++e) st_act<T>(dst + e, o_sh[at][d + e]);
}

// ---------------------------------------------------------------------------
// Host launchers
// ---------------------------------------------------------------------------
namespace vte {

static long long pa_up(long long x) { return (x + 15) / 16 * 16; }

// Tiles that `rows` rows of one sequence, one after the other, see at most, with the window of `w` (window 0: none).
static long long most_tiles(const KvPages& c, const KvRows& r, long long rows, const PaWindow& w) {
    const long long all = (((long long)r.max_pages << c.page_log2) + PA_TILE - 1) / PA_TILE;
    if (w.window == 0) return all;
    return std::min(all, (w.window + rows + PA_TILE - 2) / PA_TILE + 1 + ((long long)w.sinks + PA_TILE - 1) / PA_TILE);
}
// Whether the window is shorter than the table, so that row blocks see about as many tokens each.
static bool limited(const KvPages& c, const KvRows& r, const PaWindow& w) {
    return w.window != 0 && 2LL * w.window < (long long)r.max_pages << c.page_log2;
}
// Blocks of the few-rows form: two per CU (their registers allow no more), and
// no more than the table's capacity, or the window, has shares of four tiles.
static PaPlan rows_plan(const KvPages& c, const KvRows& r, int hd, int G, const PaWindow& w, void* scratch, long long* bytes) {
    const long long segments = (long long)r.batch * c.n_kv;
    const long long tiles = segments * most_tiles(c, r, r.max_rows, w);
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
    n += pa_up(recs * p.ncol * 4);
    p.seg = reinterpret_cast<int2*>(at + n);
    n += pa_up(segments * 8);
    *bytes = n;
    return p;
}
// The many-rows form: rows of a block, row blocks at most (each sequence may end one early), and shares of each, as many
// as fill the CUs.
// Rows of a block: 256 (one group) from 9/4 blocks a CU on, else 128 (two groups).  256 / 128, us, fp16, four sequences of
// 2048 new tokens, heads of 128: 1.5 blocks a CU 120 / 103, 1.77 134 / 122, 2 151 / 128, 2.27 146 / 146, 2.5 156 / 161, 3
// 175 / 195, 4 222 / 248; fp32 1.77 153 / 141, 2.27 175 / 178, 3 215 / 240; ragged prompts of 100 to 900 tokens 1.75 75 / 79,
// 2.45 95 / 103.
// Shares: of four steps at least, or of two while there are no more than 16; no more than 64.  Three new tokens, 16 query
// heads, 16 / 32 / 64 / 128 shares, us: after 8192 tokens 23.0 / 19.8 / 21.8 / 22.0, after 32768 57 / 37 / 30 / 34; after
// 2048 8 / 16 shares 16.0 / 14.4.
struct PromptForm {
    int groups;  // 0: one of four waves
    long long rbs;
    PaPrompt p;
    long long bytes;
};
static PromptForm prompt_form(const KvPages& c, const KvRows& r, int hd, int G, const PaWindow& w, void* scratch) {
    PromptForm f;
    auto blocks = [&](int rows) { return ((long long)r.rows * G + rows - 1) / rows + r.batch - 1; };
    f.groups = blocks(256) * c.n_kv * 4 >= 9 * device_cus() ? 1 : 2;
    // Short windows: row blocks see about as many tokens each, and their starts and ends, some two steps' time, weigh on
    // them.  With heads of 64 blocks of four waves, three of which share a CU, so that one's start lies under another's
    // steps; with heads of 128 the form that takes the least: whole rounds of eight waves, or of four, two blocks a CU, which
    // follow each other without rounds but whose steps take 8 % longer.  us by the rule above / wide / of four waves: four
    // ragged prompts of up to 1500 tokens, window 300, heads of 64 fp32 55.1 / 48.4 / 39.8, fp16 47.6 / 40.7 / 34.3, of 128
    // 37.7 / 29.4 / 29.9; eight of 300 to 1000, window 128 28.8 / 28.6 / 22.6; four of 2048, window 256 50.0 / 50.0 / 43.2;
    // 4000 tokens, window 2000 103.3 / 90.2 / 98.2; two of 2400, window 1000 53.6 wide, 55.8 of four.
    if (limited(c, r, w) && blocks(128) * c.n_kv >= device_cus()) {  // (else shares: two groups)
        const long long cus = device_cus();
        auto steps = [&](int rows) { return most_tiles(c, r, std::min(r.max_rows, rows / G + 2), w); };
        auto rounds = [&](int rows) { return (blocks(rows) * c.n_kv + cus - 1) / cus; };
        const long long wide = rounds(256) * (200 + 100 * steps(256)), two = rounds(128) * (200 + 50 * steps(128));
        const long long four = std::max(2 * cus, blocks(128) * c.n_kv) * (200 + 108 * steps(128)) / (2 * cus);
        f.groups = hd == 64 || four < std::min(wide, two) ? 0 : wide <= two ? 1 : 2;
    }
    f.rbs = blocks(f.groups == 1 ? 256 : 128);
    const long long steps = most_tiles(c, r, std::min(r.max_rows, 128 / G + 2), w);
    const long long most = std::max(std::min(16LL, steps / 2), std::min<long long>(PA_SHARES, steps / 4));
    f.p.nsp = (int)std::max(1LL, std::min(most, device_cus() / (f.rbs * c.n_kv)));
    const long long recs = f.p.nsp == 1 ? 0 : f.rbs * c.n_kv * f.p.nsp;
    uint8_t* at = static_cast<uint8_t*>(scratch);
    long long n = 16;
    f.p.o = reinterpret_cast<float*>(at + n);
    n += pa_up(recs * 128 * hd * 4);
    f.p.ml = reinterpret_cast<float*>(at + n);
    n += pa_up(recs * 128 * 8);
    f.p.ev = reinterpret_cast<int*>(at + n);
    n += pa_up(recs * 128 * 4);
    f.bytes = n;
    return f;
}
// One tile's columns hold them all.  (Few-rows / many-rows form, us: one sequence of 2049 tokens 11.8 / 16.9, 16 ragged ones
// of up to 8192 18.1 / 34.5, eight of up to 65536 37.0 / 105.)
static bool rows_form(const KvRows& r, int G) { return r.max_rows * G <= 16; }

static long long scratch_bytes(const KvPages& c, const KvRows& r, int hd, int n_q, const PaWindow& w) {
    const int G = n_q / c.n_kv;
    if (!rows_form(r, G)) return prompt_form(c, r, hd, G, w, nullptr).bytes;
    long long n;
    rows_plan(c, r, hd, G, w, nullptr, &n);
    return n;
}
long long attn_pages_scratch_bytes(const KvPages& c, const KvRows& r, int hd, int n_q) {
    return scratch_bytes(c, r, hd, n_q, PaWindow{0, 0});
}
long long attn_pages_window_scratch_bytes(const KvPages& c, const KvRows& r, int hd, int n_q, int window, int sinks) {
    return scratch_bytes(c, r, hd, n_q, PaWindow{window, sinks});
}

template <typename T, int HD, bool WIN>
static hipError_t attn_hd(const KvPages& c, const KvRows& r, const void* q, void* out, int n_q, float scale,
                          const PaWindow& w, void* scratch, hipStream_t st) {
    const int G = n_q / c.n_kv;
    long long bytes;
    if (rows_form(r, G)) {
        const PaPlan p = rows_plan(c, r, HD, G, w, scratch, &bytes);
        hipLaunchKernelGGL((attn_pages_rows_kernel<T, HD, WIN>), dim3(p.blocks), dim3(256), 0, st, c, r, p, (const T*)q,
                           (T*)out, n_q, scale, w);
        hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
        hipLaunchKernelGGL((attn_pages_combine_kernel<T, HD, WIN>), dim3(r.batch * c.n_kv, p.ncol), dim3(256), 0, st, c, r,
                           p, (T*)out, n_q, w);
        return hipGetLastError();
    }
    const PromptForm f = prompt_form(c, r, HD, G, w, scratch);
    auto kernel = f.groups == 1 ? attn_pages_prompt_kernel<T, HD, 1, 8, WIN> : attn_pages_prompt_kernel<T, HD, 2, 4, WIN>;
    int threads = 512;
    if constexpr (WIN) {
        if (f.groups == 0) {
            kernel = attn_pages_prompt_kernel<T, HD, 1, 4, WIN>;
            threads = 256;
        }
    }
    hipLaunchKernelGGL(kernel, dim3((unsigned)(f.rbs * c.n_kv), f.p.nsp), dim3(threads), 0, st, c, r, f.p, (const T*)q, (T*)out,
                       n_q, scale, w);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || f.p.nsp == 1) return e;
    hipLaunchKernelGGL((attn_pages_prompt_combine_kernel<T, HD, WIN>), dim3((unsigned)f.rbs, c.n_kv, HD / 8),
                       dim3(256), 0, st, c, r, f.p, (T*)out, n_q, w);
    return hipGetLastError();
}
template <bool WIN>
static hipError_t attn_any(const KvPages& c, const KvRows& r, int hd, bool f16, const void* q, void* out, int n_q, float scale,
                           const PaWindow& w, void* scratch, hipStream_t st) {
#define PA_ATTN(T, HD) attn_hd<T, HD, WIN>(c, r, q, out, n_q, scale, w, scratch, st)
    if (hd == 128) return f16 ? PA_ATTN(__half, 128) : PA_ATTN(float, 128);
    return f16 ? PA_ATTN(__half, 64) : PA_ATTN(float, 64);
#undef PA_ATTN
}
hipError_t attn_pages(const KvPages& c, const KvRows& r, int hd, bool f16, const void* q, void* out, int n_q,
                      float scale, void* scratch, hipStream_t st) {
    return attn_any<false>(c, r, hd, f16, q, out, n_q, scale, PaWindow{0, 0}, scratch, st);
}
hipError_t attn_pages_window(const KvPages& c, const KvRows& r, int hd, bool f16, const void* q, void* out, int n_q,
                             float scale, int window, int sinks, void* scratch, hipStream_t st) {
    return attn_any<true>(c, r, hd, f16, q, out, n_q, scale, PaWindow{window, sinks}, scratch, st);
}

}  // namespace vte
