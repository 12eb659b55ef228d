// How attention of a few rows a sequence over a paged cache is cut into units of work, for the kernels of attn_rows.cu and
// attn_rows_tcgen05.cu.
//
// The query heads that share a kv head are rows of one problem: packed row r of a sequence is token r / G, head r % G of the
// group (G = H / KV). A tile is `tile_rows` packed rows, a chunk `cp` pages of the sequence's keys, a unit one chunk of one tile
// (and, in the grid's second dimension, one kv head). Every CTA works the units out from the step's description on the device,
// so a captured launch serves whatever lengths its replays bring: cp is such that all units together are about `target`, and
// the grid is sized for the most units that the step's rows can make (units() on the host). A sequence of many pages has many
// chunks, a short one a single unit, whatever the other sequences are.
#pragma once
#include "layout.cuh"

struct RowsArgs {
    int T, B, H, KV, HD, G;
    int ldq, ldo;
    int tile_rows;                    // packed rows a tile
    int min_pages;                    // pages a chunk at least
    int target;                       // units to aim at, over all kv heads; 0: a tile's keys are never cut
    int causal;                       // 1: token i sees rows <= past + i; 0: the mask words
    int words;                        // mask words a token
    float scale_log2;                 // score scale * log2(e)
};

// Most units (of one kv head) that a step can make: tiles * ceil(pages / cp) <= tiles * pages / cp + tiles.
static inline long long row_units_max(const RowsArgs& a) {
    const long long tiles = ceil_div_ll((long long)a.T * a.G, a.tile_rows) + a.B;
    return tiles + (a.target > 0 ? ceil_div(a.target, a.KV) : 0);
}

struct SeqShape {
    int q_begin, n_q, kvl, tiles, pages;
};

// A sequence's numbers. Bounds that cannot be (rows outside the step, fewer keys than rows) count as a sequence without rows
// and are reported.
__device__ __forceinline__ SeqShape seq_shape(const int* __restrict__ cu_q, const int* __restrict__ kv_len, int b, const RowsArgs& a,
                                              int* status) {
    SeqShape s;
    s.q_begin = cu_q[b];
    const int end = cu_q[b + 1];
    s.n_q = end - s.q_begin;
    s.kvl = kv_len[b];
    if (s.n_q <= 0 || s.q_begin < 0 || end > a.T || s.kvl < s.n_q) {
        if (s.n_q != 0) atomicOr(status, MYNAH_ST_PAGE_RANGE);
        s.n_q = 0;
    }
    s.tiles = (int)(((long long)s.n_q * a.G + a.tile_rows - 1) / a.tile_rows);
    s.pages = s.n_q > 0 ? (s.kvl + PAGE_TOKENS - 1) / PAGE_TOKENS : 0;
    return s;
}

struct RowUnit {
    int b, tile, chunk;
    int unit0;                        // the first unit of the sequence; unit0 + tile * seq_chunks + chunk is this one
    int seq_chunks;                   // units a tile of this sequence has room for
    int cp;                           // pages a chunk
    SeqShape s;

    __device__ __forceinline__ int past() const { return s.kvl - s.n_q; }
    __device__ __forceinline__ int rows(const RowsArgs& a) const { return min(a.tile_rows, s.n_q * a.G - tile * a.tile_rows); }
    // pages that some row of the tile may see: all, or up to the tile's last token
    __device__ __forceinline__ int tile_pages(const RowsArgs& a) const {
        if (!a.causal) return s.pages;
        const int last = (min(s.n_q * a.G, (tile + 1) * a.tile_rows) - 1) / a.G;
        return (past() + last) / PAGE_TOKENS + 1;
    }
};

__device__ __forceinline__ long long warp_sum_ll(long long v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Finds unit number `flat` (the units of a sequence lie together, its last tile first, so that the longest work of a causal step
// starts first); false when the step has fewer. Warp 0 does the sums, 32 sequences at a time; every thread of the CTA must call
// this (it synchronises the CTA).
__device__ __forceinline__ bool find_row_unit(const int* __restrict__ cu_q, const int* __restrict__ kv_len, const RowsArgs& a, int flat,
                                              RowUnit& u, int* status) {
    __shared__ int found_s[4];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (warp == 0) {
        int cp = 1 << 28;
        if (a.target > 0) {
            long long work = 0;
            for (int b0 = 0; b0 < a.B; b0 += 32) {
                const int b = b0 + lane;
                if (b < a.B) {
                    const SeqShape s = seq_shape(cu_q, kv_len, b, a, status);
                    work += (long long)s.tiles * s.pages;
                }
            }
            work = warp_sum_ll(work);
            cp = (int)max((long long)a.min_pages, (work * a.KV + a.target - 1) / a.target);
        }
        int fb = -1, base = 0, first = 0;
        for (int b0 = 0; b0 < a.B && fb < 0; b0 += 32) {
            const int b = b0 + lane;
            int n = 0;
            if (b < a.B) {
                const SeqShape s = seq_shape(cu_q, kv_len, b, a, status);
                n = s.tiles * ((s.pages + cp - 1) / cp);
            }
            int incl = n;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= o) incl += v;
            }
            const int excl = incl - n;
            const unsigned hit = __ballot_sync(0xffffffffu, n > 0 && flat >= base + excl && flat < base + incl);
            if (hit != 0u) {
                const int src = __ffs(hit) - 1;
                fb = b0 + src;
                first = base + __shfl_sync(0xffffffffu, excl, src);
            }
            base += __shfl_sync(0xffffffffu, incl, 31);
        }
        if (lane == 0) {
            found_s[0] = fb;
            found_s[1] = first;
            found_s[2] = cp;
        }
    }
    __syncthreads();
    u.b = found_s[0];
    if (u.b < 0) return false;
    u.unit0 = found_s[1];
    u.cp = found_s[2];
    u.s = seq_shape(cu_q, kv_len, u.b, a, status);
    u.seq_chunks = (u.s.pages + u.cp - 1) / u.cp;
    const int at = flat - u.unit0;
    u.tile = u.s.tiles - 1 - at / u.seq_chunks;
    u.chunk = at % u.seq_chunks;
    return true;
}

// What a unit's CTA leaves for the merge, per sequence: where its units begin, their pages a chunk.
struct RowInfo {
    int unit0, cp;
};

// Which of the 64 keys from key0 (a multiple of 64) on token `tok` of a sequence sees: bit e for key key0 + e. Held rows (below
// past) are seen by all; of the step's own rows, those up to the token's own (causal), or those whose bits are set in the
// token's mask words. Keys at and behind kvl are never seen, whatever the words say.
__device__ __forceinline__ unsigned long long visible64(int key0, int kvl, int past, int tok, int causal,
                                                        const long long* __restrict__ words, int n_words) {
    const int n = kvl - key0;
    if (n <= 0) return 0ull;
    const unsigned long long all = ~0ull, lim = n >= 64 ? all : (1ull << n) - 1ull;
    if (causal) {
        const int c = past + tok + 1 - key0;
        if (c <= 0) return 0ull;
        return lim & (c >= 64 ? all : (1ull << c) - 1ull);
    }
    const int off = key0 - past;
    if (off <= -64) return lim;
    auto w = [&](int i) { return i < n_words ? (unsigned long long)words[i] : 0ull; };
    if (off < 0) return lim & (((1ull << -off) - 1ull) | (w(0) << -off));
    const int i = off >> 6, s = off & 63;
    unsigned long long v = w(i) >> s;
    if (s != 0) v |= w(i + 1) << (64 - s);
    return lim & v;
}
