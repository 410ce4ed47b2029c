// The pages of a paged KV cache as a pool that sequences share: copies, pages given back, room for new tokens, forks
// and compaction, gfx950.  No counterpart in the reference, whose sequences own a fixed range each
// (vte/compiler/qwen_mapper.py:300-351).
//
// refs[p] is the number of users of page p (table entries, and whatever else the program counts); 0: free.  One table and
// one refs array serve the pools of all layers: only copies touch bytes.  New pages are always the lowest free ones, in
// the order of the call's list, so what a call does depends on its inputs alone and not on which block came first; users
// are counted by integer atomics, whose order does not matter.  Entries are exchanged, not written, and what stood there
// loses a user; new pages of one entry (of a sequence listed twice) are compared, and the lowest stays.  (A fork's lists may
// not have a child twice, or as a parent too: whose pages such a child shows, and whether a begun page is copied before or
// after it was filled, would go by the threads' order.  Users are counted right all the same.)
#include <algorithm>
#include "kv_pages.h"

#define KVM_LAYERS 64    // of a copy launch: 2 KB of arguments
#define KVM_CHUNK 1024   // pages a block counts
#define KVM_PIECE 1024   // 16-byte words that a block copies
#define KVM_FEW 8192     // pages that every block of a compaction counts itself
#define KVM_BLOCKS 128   // of a CU, at most, where the number of pairs is not known

struct KvLayers {
    uint8_t *k[KVM_LAYERS], *v[KVM_LAYERS];
    int8_t *k_exp[KVM_LAYERS], *v_exp[KVM_LAYERS];
};

__device__ __forceinline__ bool kvm_is_page(const KvTables& t, int p) { return (unsigned)p < (unsigned)t.n_pages; }
// One user less (not below none, whatever the count was).
__device__ __forceinline__ void kvm_release(const KvTables& t, int p) {
    if (!kvm_is_page(t, p)) return;
    if (atomicSub(&t.refs[p], 1) <= 0) atomicAdd(&t.refs[p], 1);
}
// Entry j of a row becomes p, whose user it already counts as.
__device__ __forceinline__ void kvm_set(const KvTables& t, int row, int j, int p) {
    kvm_release(t, atomicExch(&t.table[(size_t)row * t.max_pages + j], p));
}
// Entry j of a row, which is no page (above all of them without a sign), becomes p, whose user it already counts as, or
// keeps the lower page that it was given meanwhile.  Whether a page is free again by that.
__device__ __forceinline__ bool kvm_set_lowest(const KvTables& t, int row, int j, int p) {
    const unsigned old = atomicMin(reinterpret_cast<unsigned*>(&t.table[(size_t)row * t.max_pages + j]), (unsigned)p);
    kvm_release(t, (int)max(old, (unsigned)p));
    return kvm_is_page(t, (int)max(old, (unsigned)p));
}

// ---------------------------------------------------------------------------
// Copies: pages src[i] -> dst[i] of every layer, i < n; pairs of which one is no page are skipped.  grid (pieces, layers,
// pairs, or as many of them as there are blocks for): a block copies KVM_PIECE words of K then V, the first piece takes
// the exponents along.
//
// Stores pass the caches by, whose lines they would fill for nobody; loads too (ONCE) where the pools are larger than the
// memory-side cache, so that the pages are not in it.  us of two inputs in turn with neither past the caches, stores, both:
// 470 MB read and written by a compaction 112.0, 104.4, 101.9 (98.3 of more inputs); one of a smaller pool, a graph, 10.2,
// 10.0, 11.5; 117 MB of forks, whose pages are in the cache, 30.5, 29.8, 36.6.
// ---------------------------------------------------------------------------
template <bool ONCE>
__device__ __forceinline__ uint4 kvm_load(const uint8_t* p) {
    if constexpr (!ONCE) return ldg_g16(p);
    const vte_u32x4 v = __builtin_nontemporal_load((vte_g_u32x4*)p);
    return make_uint4(v.x, v.y, v.z, v.w);
}
template <bool ONCE>
__device__ __forceinline__ void kvm_copy(const KvLayers& L, int layer_words, int exps, int n_pages, const int* src,
                                         const int* dst, int n) {
    const int words = 2 * layer_words, piece = blockIdx.x, l = blockIdx.y;  // 16-byte words of a page, K and V
    auto at = [&](int page, int w) {
        return w < layer_words ? L.k[l] + ((size_t)page * layer_words + w) * 16
                               : L.v[l] + ((size_t)page * layer_words + w - layer_words) * 16;
    };
    for (int i = blockIdx.z; i < n; i += gridDim.z) {
        const int a = src[i], b = dst[i];
        if ((unsigned)a >= (unsigned)n_pages || (unsigned)b >= (unsigned)n_pages) continue;
        uint4 x[KVM_PIECE / 256];
#pragma unroll
        for (int u = 0; u < KVM_PIECE / 256; ++u) {
            const int w = piece * KVM_PIECE + u * 256 + threadIdx.x;
            if (w < words) x[u] = kvm_load<ONCE>(at(a, w));
        }
#pragma unroll
        for (int u = 0; u < KVM_PIECE / 256; ++u) {
            const int w = piece * KVM_PIECE + u * 256 + threadIdx.x;
            if (w < words)
                __builtin_nontemporal_store(vte_u32x4{x[u].x, x[u].y, x[u].z, x[u].w}, reinterpret_cast<vte_u32x4*>(at(b, w)));
        }
        if (piece == 0)
            for (int e = threadIdx.x; e < exps; e += 256) {
                L.k_exp[l][(size_t)b * exps + e] = L.k_exp[l][(size_t)a * exps + e];
                L.v_exp[l][(size_t)b * exps + e] = L.v_exp[l][(size_t)a * exps + e];
            }
    }
}
__global__ __launch_bounds__(256) void kv_copy_kernel(KvLayers L, int layer_words, int exps, int n_pages,
                                                      const int* __restrict__ src, const int* __restrict__ dst, int n) {
    kvm_copy<false>(L, layer_words, exps, n_pages, src, dst, n);
}

// ---------------------------------------------------------------------------
// Pages given back: entries of whole pages of tokens keep .. end[i] - behind - 1.  grid (entries, sequences); a chain of
// loads and atomics, 2.6 to 3 us.
// ---------------------------------------------------------------------------
__global__ __launch_bounds__(256) void kv_free_kernel(KvTables t, const int* __restrict__ seqs, int keep,
                                                      const int* __restrict__ end, int behind) {
    const int row = seqs != nullptr ? seqs[blockIdx.y] : (int)blockIdx.y;
    if ((unsigned)row >= (unsigned)t.batch) return;
    const int j = blockIdx.x * 256 + threadIdx.x;
    const int low = (int)(((long long)keep + (1 << t.page_log2) - 1) >> t.page_log2);
    int high = t.max_pages;
    if (end != nullptr) high = min(high, end[blockIdx.y] < 0 ? 0 : max(end[blockIdx.y] - behind, 0) >> t.page_log2);
    if (j < low || j >= high) return;
    if (t.table[(size_t)row * t.max_pages + j] != -1) kvm_set(t, row, j, -1);
}

// ---------------------------------------------------------------------------
// New pages, by one block of 1024 threads, so that they are the lowest free ones in the slots' order without a wait between
// blocks.  `want(slot)` says whether a slot of 0 .. slots - 1 needs one (1), is to have none (KVM_LEFT) or has one (0),
// `give(slot, page)`, called by the same thread right after, takes it (page -1: there are no more).  The result: slots that got
// none, and those that were to have none (counted in one sum with the others, which holds 1024 of both).
//
// Pages are looked at 16384 at a time, the next ones asked for meanwhile, and free ones put into a ring in LDS, 4096 pages'
// at a time while slots need them.  Bound by latency: a chain of five loads and atomics, 2.9 us where no page is needed (a
// graph), 3.1 traced of eight sequences, 4.6 of 64; a reserve and a free where the last 70 of 4096, 65536 or 2^20 pages are
// free 6.8, 14 to 17 and 82 us (4096 pages at a time and none ahead: 6.9, 30 and 410).  (refs of pages that were not looked
// at yet do not change in a search: what it takes or gives back lies before them.)
// ---------------------------------------------------------------------------
#define KVM_RING 8192
#define KVM_LOOK 16384
#define KVM_LEFT (1 << 16)
struct KvmNone {
    int missing, left;
};
template <class Want, class Give>
__device__ __forceinline__ KvmNone kvm_new_pages(const KvTables& t, int slots, Want want, Give give) {
    __shared__ int ring[KVM_RING];
    __shared__ int sums[16];
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    auto scan = [&](int v, int& total) {  // the sum before this thread's, and of all
        int incl = v;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int o = __shfl_up(incl, d, 64);
            incl += lane >= d ? o : 0;
        }
        __syncthreads();
        if (lane == 63) sums[wv] = incl;
        __syncthreads();
        int before = 0;
        total = 0;
#pragma unroll
        for (int w = 0; w < 16; ++w) {
            before += w < wv ? sums[w] : 0;
            total += sums[w];
        }
        return before + incl - v;
    };
    uint4 ahead[4];
    auto ask = [&](int base) {  // for this thread's four pages of every 4096 from base on
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int p = base + 4096 * g + 4 * tid;
            ahead[g] = make_uint4(1, 1, 1, 1);
            if (p + 4 <= t.n_pages) {
                ahead[g] = ldg_g16(t.refs + p);
            } else if (p < t.n_pages) {
                ahead[g].x = t.refs[p];
                if (p + 1 < t.n_pages) ahead[g].y = t.refs[p + 1];
                if (p + 2 < t.n_pages) ahead[g].z = t.refs[p + 2];
            }
        }
    };
    uint32_t free_bits = 0;  // of the pages at hand: bit 4 g + u
    auto look = [&] {
        free_bits = 0;
#pragma unroll
        for (int g = 0; g < 4; ++g)
            free_bits |= (uint32_t)((int)ahead[g].x <= 0) << (4 * g) | (uint32_t)((int)ahead[g].y <= 0) << (4 * g + 1) |
                         (uint32_t)((int)ahead[g].z <= 0) << (4 * g + 2) | (uint32_t)((int)ahead[g].w <= 0) << (4 * g + 3);
    };
    ask(0);  // (while it is not known yet whether a slot needs one)
    KvmNone none = {0, 0};
    int head = 0, have = 0, next = 0;  // of the ring; the first page not looked at
    for (int s0 = 0; s0 < slots; s0 += 1024) {
        const int w = s0 + tid < slots ? want(s0 + tid) : 0;
        int n;
        const int rank = scan(w, n) & (KVM_LEFT - 1);
        none.left += n / KVM_LEFT;
        n &= KVM_LEFT - 1;
        while (have < n && next < t.n_pages) {
            const int group = next / 4096 % (KVM_LOOK / 4096);
            if (group == 0) {
                look();
                if (next + KVM_LOOK < t.n_pages) ask(next + KVM_LOOK);
                if (next > 0 && !__syncthreads_or(free_bits != 0)) {  // (the lowest pages: with the scan)
                    next += KVM_LOOK;
                    continue;
                }
            }
            const uint32_t mine = free_bits >> (4 * group) & 15;
            int found;
            int at = head + have + scan(__popc(mine), found);
#pragma unroll
            for (int u = 0; u < 4; ++u)
                if (mine >> u & 1) ring[at++ & (KVM_RING - 1)] = next + 4 * tid + u;
            have += found;
            next += 4096;
        }
        __syncthreads();
        if (w == 1) {
            const int page = rank < have ? ring[(head + rank) & (KVM_RING - 1)] : -1;
            if (page >= 0) {
                atomicExch(&t.refs[page], 1);
                __threadfence_block();  // (before the entry that shows it to others, which may release it)
            }
            give(s0 + tid, page);
        }
        const int got = min(n, have);
        head += got;
        have -= got;
        none.missing += n - got;
        __syncthreads();
    }
    return none;
}

// Entries of tokens start[i] .. start[i] + count - 1 (below stop[i]) of each sequence; `per` slots a sequence.  `follow`: the
// tokens follow others, which are in the cache or were dropped; an entry that begins before start[i] and is no page stays
// so, because a page given now would show what it held as the tokens before.
__global__ __launch_bounds__(1024) void kv_reserve_kernel(KvTables t, int n, const int* __restrict__ seqs,
                                                          const int* __restrict__ start, const int* __restrict__ stop,
                                                          int count, int per, bool follow, int* missing) {
    int row = 0, j = 0;   // of the slot at hand
    bool inside = false;  // its entry begins before start[i]
    auto entry = [&](int slot) {
        const int i = slot / per;
        row = seqs != nullptr ? seqs[i] : i;
        if ((unsigned)row >= (unsigned)t.batch || start[i] < 0) return false;
        long long end = min((long long)start[i] + count, (long long)t.max_pages << t.page_log2);
        if (stop != nullptr) end = min(end, (long long)stop[i]);
        const long long at = (start[i] >> t.page_log2) + (long long)(slot - i * per);
        j = (int)at;
        inside = at << t.page_log2 < start[i];
        return at << t.page_log2 < end && end > start[i];
    };
    auto page_at_entry = [&] {  // (not from the cache of this CU: it may have been given a page by an earlier slot)
        return kvm_is_page(t, __hip_atomic_load(&t.table[(size_t)row * t.max_pages + j], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
    };
    bool back = false;  // a page that an entry was given twice is free again
    auto want = [&](int slot) { return !entry(slot) || page_at_entry() ? 0 : follow && inside ? KVM_LEFT : 1; };
    auto give = [&](int, int page) {
        if (page >= 0 && kvm_set_lowest(t, row, j, page)) back = true;
    };
    KvmNone none = kvm_new_pages(t, n * per, want, give);
    if (none.missing + none.left == 0) {
        if (missing != nullptr && threadIdx.x == 0) *missing = 0;
        return;
    }
    // Pages that came back go to the entries that got none.  (A search of its own: with the first one inside the loop every
    // call took 0.6 us more.)
    while (none.missing != 0) {
        __threadfence();  // users as they are now: what was counted here is in memory,
        if (!__syncthreads_or(back)) break;
        __threadfence();  // and nothing older is left in the cache of this CU
        back = false;
        none = kvm_new_pages(t, n * per, want, give);
    }
    // Entries as they are now: one that the list asks for twice may have got a page by the other slot.
    __shared__ int without;
    if (threadIdx.x == 0) without = 0;
    __syncthreads();
    for (int slot = threadIdx.x; slot < n * per; slot += 1024)
        if (entry(slot) && !page_at_entry()) atomicAdd(&without, 1);
    __syncthreads();
    if (missing != nullptr && threadIdx.x == 0) *missing = without;
}

// ---------------------------------------------------------------------------
// Forks.  First the whole pages of a parent's first tokens are shared with the child, whose own go (grid (entries,
// children)); then one block finds a page for each child whose last page is begun, and lists what is to be copied.
// Up to an entry a thread of the one block, it does both: a launch less (a fork of 1020 entries between a free and a
// reserve, a graph 14.9 against 15.2 us, calls 19.8 against 22.7; of 2108 entries the graph is slower, 17.4 against 16.3).
// A child that is its own parent stays as it is.
// ---------------------------------------------------------------------------
struct KvFork {
    const int *parents, *children, *lengths;
    int n;
};
__device__ __forceinline__ bool kvm_fork(const KvTables& t, const KvFork& f, int i, int& parent, int& child, int& length) {
    parent = f.parents[i];
    child = f.children[i];
    length = f.lengths[i];
    return (unsigned)parent < (unsigned)t.batch && (unsigned)child < (unsigned)t.batch && parent != child && length >= 0;
}
__device__ __forceinline__ void kvm_fork_entry(const KvTables& t, int parent, int child, int length, int j) {
    int p = -1;
    if (j < length >> t.page_log2) {
        p = t.table[(size_t)parent * t.max_pages + j];
        if (kvm_is_page(t, p)) atomicAdd(&t.refs[p], 1);
        else p = -1;
    }
    kvm_set(t, child, j, p);
}
__global__ __launch_bounds__(256) void kv_fork_kernel(KvTables t, KvFork f) {
    const int j = blockIdx.x * 256 + threadIdx.x;
    int parent, child, length;
    if (kvm_fork(t, f, blockIdx.y, parent, child, length) && j < t.max_pages) kvm_fork_entry(t, parent, child, length, j);
}
// `all`: the entries that kv_fork_kernel takes, too.
__global__ __launch_bounds__(1024) void kv_fork_last_kernel(KvTables t, KvFork f, bool all, int* src, int* dst, int* missing) {
    if (all) {
        for (int e = threadIdx.x; e < f.n * t.max_pages; e += 1024) {
            const int i = e / t.max_pages;
            int parent, child, length;
            if (kvm_fork(t, f, i, parent, child, length)) kvm_fork_entry(t, parent, child, length, e - i * t.max_pages);
        }
    }
    for (int i = threadIdx.x; i < f.n; i += 1024) src[i] = dst[i] = -1;
    __builtin_amdgcn_s_waitcnt(0);  // (atomics that return nothing, too: the counts are read next)
    __syncthreads();
    int child = 0, j = 0, page = -1;  // of the slot at hand
    const KvmNone none = kvm_new_pages(
        t, f.n,
        [&](int i) {
            int parent, length;
            if (!kvm_fork(t, f, i, parent, child, length)) return 0;
            j = length >> t.page_log2;
            if ((length & ((1 << t.page_log2) - 1)) == 0 || j >= t.max_pages) return 0;
            page = t.table[(size_t)parent * t.max_pages + j];
            return kvm_is_page(t, page) ? 1 : 0;
        },
        [&](int i, int to) {
            if (to < 0) return;
            src[i] = page;
            dst[i] = to;
            kvm_set(t, child, j, to);
        });
    if (missing != nullptr && threadIdx.x == 0) *missing = none.missing;
}

// ---------------------------------------------------------------------------
// Compaction: with U used pages, the k-th used page from U on moves to the k-th free one below U.  Counts per chunk (of
// up to KVM_FEW pages every block counts them all itself, a launch less, a graph's us: 1000 pages 10.4 against 11.9, 8192
// 13.8 against 14.8, 16384 17.9 against 16.4); then every block knows U and what lies before its chunk, lists its pages'
// places and writes where each page goes, those that move as -2 - k until the copies' launch, which knows the lists.
// ---------------------------------------------------------------------------
struct KvMoves {
    int *counts, *src, *dst, *moves;  // used pages of each chunk; pairs; how many
};
__global__ __launch_bounds__(256) void kv_count_kernel(KvTables t, int* __restrict__ counts) {
    __shared__ int sums[4];
    int n = 0;
    for (int u = 0; u < KVM_CHUNK / 256; ++u) {
        const int p = blockIdx.x * KVM_CHUNK + u * 256 + threadIdx.x;
        n += __popcll(__ballot(p < t.n_pages && t.refs[p] > 0));
    }
    if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = n;
    __syncthreads();
    if (threadIdx.x == 0) counts[blockIdx.x] = sums[0] + sums[1] + sums[2] + sums[3];
}
template <bool COUNTED>
__global__ __launch_bounds__(256) void kv_place_kernel(KvTables t, KvMoves m, int chunks, int* __restrict__ where,
                                                       int* __restrict__ used) {
    __shared__ int sums[3][4];
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6, chunk0 = blockIdx.x * KVM_CHUNK;
    auto all = [&](int row, int v) {  // the block's sum
#pragma unroll
        for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d, 64);
        if (lane == 0) sums[row][wv] = v;
        __syncthreads();
        return sums[row][0] + sums[row][1] + sums[row][2] + sums[row][3];
    };
    int v = 0, first = 0;  // used pages: all of them, and those before the chunk
    if constexpr (COUNTED) {
        for (int c = tid; c < chunks; c += 256) {
            v += m.counts[c];
            first += c < (int)blockIdx.x ? m.counts[c] : 0;
        }
    } else {
#pragma unroll 8
        for (int p = tid; p < t.n_pages; p += 256) {
            const int n = t.refs[p] > 0;
            v += n;
            first += p < chunk0 ? n : 0;
        }
    }
    const int U = all(0, v);
    int before = all(1, first);
    v = 0;
    int p0 = 0;
    if constexpr (COUNTED) {
        const int cut = U / KVM_CHUNK;  // (U is in chunk `cut`, which may be one behind the last)
        for (int c = tid; c < cut; c += 256) v += m.counts[c];
        p0 = cut * KVM_CHUNK;
    }
#pragma unroll 8
    for (int p = p0 + tid; p < U; p += 256) v += t.refs[p] > 0;
    const int below = all(2, v);  // used pages below U
    if (blockIdx.x == 0 && tid == 0) {
        *used = U;
        *m.moves = U - below;
    }
    __shared__ int row_sums[4][4];
    uint64_t bits[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        const int p = chunk0 + u * 256 + tid;
        bits[u] = __ballot(p < t.n_pages && t.refs[p] > 0);
        if (lane == 0) row_sums[u][wv] = __popcll(bits[u]);
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        const int p = chunk0 + u * 256 + tid;
        int n = before + __popcll(bits[u] & ((1ull << lane) - 1));  // used pages before p
        for (int w = 0; w < 4; ++w) {
            n += w < wv ? row_sums[u][w] : 0;
            before += row_sums[u][w];
        }
        if (p >= t.n_pages) continue;
        const bool mine = bits[u] >> lane & 1;
        if (mine && p >= U) {
            m.src[n - below] = p;
            where[p] = -2 - (n - below);
        } else {
            if (!mine && p < U) m.dst[p - n] = p;
            where[p] = mine ? p : -1;
        }
    }
}
// (first: the launch that also rewrites tables, counts and `where`)
template <bool ONCE>
__global__ __launch_bounds__(256) void kv_move_kernel(KvLayers L, int layer_words, int exps, KvTables t, KvMoves m, int* where,
                                                      bool first) {
    const int n = *m.moves;
    if (first) {
        const long long step = (long long)gridDim.x * gridDim.y * gridDim.z * 256;
        const long long at = (blockIdx.x + (long long)gridDim.x * (blockIdx.y + gridDim.y * blockIdx.z)) * 256 + threadIdx.x;
        for (long long e = at; e < (long long)t.batch * t.max_pages; e += step) {
            const int p = t.table[e];
            if (!kvm_is_page(t, p)) continue;
            const int w = where[p];  // (-2 - k, or already the place that stands for)
            t.table[e] = w <= -2 ? m.dst[-2 - w] : w;
        }
        for (long long k = at; k < n; k += step) {
            const int a = m.src[k], b = m.dst[k];
            where[a] = b;
            t.refs[b] = t.refs[a];
            t.refs[a] = 0;
        }
    }
    kvm_copy<ONCE>(L, layer_words, exps, t.n_pages, m.src, m.dst, n);
}

// ---------------------------------------------------------------------------
// Host launchers
// ---------------------------------------------------------------------------
namespace vte {

static KvLayers layers_of(const KvPages* layers, int n) {
    KvLayers L = {};
    for (int i = 0; i < n; ++i) {
        L.k[i] = layers[i].k;
        L.v[i] = layers[i].v;
        L.k_exp[i] = layers[i].k_exp;
        L.v_exp[i] = layers[i].v_exp;
    }
    return L;
}
struct CopyShape {
    int words, exps, pieces;
};
static CopyShape copy_shape(const KvPages& c, int hd) {
    CopyShape s;
    s.words = (int)((((long long)c.n_kv << c.page_log2) * hd) / 16);
    s.exps = c.n_kv << (c.page_log2 - 4);
    s.pieces = (2 * s.words + KVM_PIECE - 1) / KVM_PIECE;
    return s;
}
// One block for each piece of n pairs, KVM_BLOCKS a CU at most; at least `least` in all.
static dim3 copy_grid(const CopyShape& s, int n_layers, long long n, long long least) {
    const long long each = (long long)s.pieces * n_layers;
    const long long z = std::max(std::min(n, (KVM_BLOCKS * device_cus() + each - 1) / each), (least + each - 1) / each);
    return dim3(s.pieces, n_layers, (unsigned)std::min(std::max(z, 1LL), 65535LL));
}

hipError_t kv_pages_copy(const KvPages* layers, int n_layers, int hd, const int* src, const int* dst, int n, hipStream_t st) {
    const CopyShape s = copy_shape(layers[0], hd);
    for (int l = 0; l < n_layers; l += KVM_LAYERS) {
        const int m = std::min(KVM_LAYERS, n_layers - l);
        hipLaunchKernelGGL(kv_copy_kernel, copy_grid(s, m, n, 1), dim3(256), 0, st, layers_of(layers + l, m), s.words, s.exps,
                           layers[0].n_pages, src, dst, n);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}
hipError_t kv_pages_free(const KvTables& t, int n, const int* seqs, int keep, const int* end, int behind, hipStream_t st) {
    hipLaunchKernelGGL(kv_free_kernel, dim3((t.max_pages + 255) / 256, n), dim3(256), 0, st, t, seqs, keep, end, behind);
    return hipGetLastError();
}
// Slots of a sequence: pages that `count` tokens touch at most.
int kv_pages_reserve_slots(const KvTables& t, int count) {
    return (int)std::min<long long>(t.max_pages, (((long long)count - 1) >> t.page_log2) + 2);
}
hipError_t kv_pages_reserve(const KvTables& t, int n, const int* seqs, const int* start, const int* stop, int count,
                            bool follow, int* missing, hipStream_t st) {
    hipLaunchKernelGGL(kv_reserve_kernel, dim3(1), dim3(1024), 0, st, t, n, seqs, start, stop, count,
                       kv_pages_reserve_slots(t, count), follow, missing);
    return hipGetLastError();
}
long long kv_pages_fork_scratch_bytes(int n) { return 8LL * n; }
hipError_t kv_pages_fork(const KvPages* layers, int n_layers, int hd, const KvTables& t, int n, const int* parents,
                         const int* children, const int* lengths, int* missing, void* scratch, hipStream_t st) {
    const KvFork f{parents, children, lengths, n};
    int* src = static_cast<int*>(scratch);
    const bool all = (long long)n * t.max_pages <= 1024;
    hipError_t e = hipSuccess;
    if (!all) {
        hipLaunchKernelGGL(kv_fork_kernel, dim3((t.max_pages + 255) / 256, n), dim3(256), 0, st, t, f);
        e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    hipLaunchKernelGGL(kv_fork_last_kernel, dim3(1), dim3(1024), 0, st, t, f, all, src, src + n, missing);
    e = hipGetLastError();
    return e != hipSuccess ? e : kv_pages_copy(layers, n_layers, hd, src, src + n, n, st);
}
static int chunks_of(const KvTables& t) { return (t.n_pages + KVM_CHUNK - 1) / KVM_CHUNK; }
long long kv_pages_compact_scratch_bytes(const KvTables& t) { return 4LL * (4 + chunks_of(t) + 2LL * t.n_pages); }
hipError_t kv_pages_compact(const KvPages* layers, int n_layers, int hd, const KvTables& t, int* where, int* used, void* scratch,
                            hipStream_t st) {
    KvMoves m;
    m.moves = static_cast<int*>(scratch);
    m.counts = m.moves + 4;
    m.src = m.counts + chunks_of(t);
    m.dst = m.src + t.n_pages;
    hipError_t e = hipSuccess;
    if (t.n_pages <= KVM_FEW) {
        hipLaunchKernelGGL(kv_place_kernel<false>, dim3(chunks_of(t)), dim3(256), 0, st, t, m, chunks_of(t), where, used);
    } else {
        hipLaunchKernelGGL(kv_count_kernel, dim3(chunks_of(t)), dim3(256), 0, st, t, m.counts);
        e = hipGetLastError();
        if (e != hipSuccess) return e;
        hipLaunchKernelGGL(kv_place_kernel<true>, dim3(chunks_of(t)), dim3(256), 0, st, t, m, chunks_of(t), where, used);
    }
    e = hipGetLastError();
    const CopyShape s = copy_shape(layers[0], hd);
    for (int l = 0; l < n_layers && e == hipSuccess; l += KVM_LAYERS) {
        const int n = std::min(KVM_LAYERS, n_layers - l);
        const long long entries = std::min<long long>((long long)t.batch * t.max_pages / 256 + 1, 4 * device_cus());
        // (256 MB: the memory-side cache)
        const bool once = 32LL * s.words * t.n_pages * n > (256LL << 20);
        hipLaunchKernelGGL(once ? kv_move_kernel<true> : kv_move_kernel<false>, copy_grid(s, n, t.n_pages / 2, l == 0 ? entries : 1), dim3(256), 0, st,
                           layers_of(layers + l, n), s.words, s.exps, t, m, where, l == 0);
        e = hipGetLastError();
    }
    return e;
}

}  // namespace vte
