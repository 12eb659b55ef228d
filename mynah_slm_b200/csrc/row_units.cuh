// How attention of a few rows a sequence over a paged cache is shared out among CTAs, for the kernels of attn_rows.cu and
// attn_rows_tcgen05.cu.
//
// The query heads that share a kv head are rows of one problem: packed row r of a sequence is token r / G, head r % G of the
// group (G = H / KV). A tile is `tile_rows` packed rows; an item is one tile against all keys it may see, for one kv head; its
// length is the number of those keys' pages. All items of the step lie one behind the other (by sequence, kv head, tile) on a
// line, and CTA c takes the `range` pages from c * range on, whatever items they belong to: every CTA has the same number of
// pages, however ragged the batch. A piece of an item that a CTA has on its own is a segment. An item that one CTA has whole is
// finished there; of the others every CTA leaves its segment's maximum, sum and unnormalised output in scratch (at most two a
// CTA: one that began before its range, one that goes on behind it), and a second launch joins them: an item that is cut is cut
// at the start of some range, so there is one CTA (and its helpers) of that launch for every range, which finds there what the
// range's own CTA wrote down of its start.
//
// Everything is worked out on the device from the step's description, so a captured launch serves whatever lengths its replays
// bring. Where sequences have several tiles, `group` CTAs side by side take the same pages for `group` tiles (an item is then
// that many tiles), so that a page comes from memory once and from L2 for the others: 16 trees of 64 tokens with four heads a kv
// head (two tiles each) behind 8,191 rows read 1.05 GB one tile after the other, 0.54 GB together. Against chunks of equal pages per sequence, whose last chunks are short and whose number is no multiple of what the
// device holds, equal ranges took 8 trees of 24 tokens behind 2,050 rows from 41 to TREE8 us and 16 of 64 behind 8,191 from 216
// to TREE16 (with the smaller key tiles that came with them).
#pragma once
#include "layout.cuh"

struct RowsArgs {
    int T, B, H, KV, HD, G;
    int ldq, ldo;
    int tile_rows;                    // packed rows a tile
    int two;                          // 1: the tcgen05 kernel's tile is two of its own
    int min_range;                    // pages a CTA at least
    int ctas;                         // ranges that the line is cut into; the launch has ctas * group CTAs
    int group;                        // tiles an item, each a CTA's
    int causal;                       // 1: token i sees rows <= past + i; 0: the mask words
    int words;                        // mask words a token
    float scale_log2;                 // score scale * log2(e)
};

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
    s.tiles = (s.n_q * a.G + a.tile_rows - 1) / a.tile_rows;
    s.pages = s.n_q > 0 ? (s.kvl + PAGE_TOKENS - 1) / PAGE_TOKENS : 0;
    return s;
}

// Pages that some row of a tile may see: all, or up to the tile's last token.
__device__ __forceinline__ int tile_pages(const SeqShape& s, int tile, const RowsArgs& a) {
    if (!a.causal) return s.pages;
    const int last = (min(s.n_q * a.G, (tile + 1) * a.tile_rows) - 1) / a.G;
    return (s.kvl - s.n_q + last) / PAGE_TOKENS + 1;
}

__device__ __forceinline__ int seq_items(const SeqShape& s, const RowsArgs& a) { return (s.tiles + a.group - 1) / a.group; }
// Pages of an item: of its last tile, which sees the most.
__device__ __forceinline__ int item_pages(const SeqShape& s, int item, const RowsArgs& a) {
    return tile_pages(s, min(s.tiles, (item + 1) * a.group) - 1, a);
}
// Pages of the sequence's items together, for one kv head.
__device__ __forceinline__ long long seq_pages(const SeqShape& s, const RowsArgs& a) {
    const int items = seq_items(s, a);
    if (!a.causal || items <= 1) return (long long)items * s.pages;
    long long n = 0;
    for (int i = 0; i < items; i++) n += item_pages(s, i, a);
    return n;
}

// Where a CTA is on the line, and the segment it is at: pages [pg0, pg1) of one tile of item (b, g, item).
struct RowWalk {
    int b, g, item, tile, pg0, pg1;
    int from, to;                     // the item's pages in this range
    int pages;                        // that the tile may see
    long long left;                   // pages of the range that are left, this segment's among them
    SeqShape s;

    __device__ __forceinline__ int past() const { return s.kvl - s.n_q; }
    __device__ __forceinline__ int rows(const RowsArgs& a) const { return min(a.tile_rows, s.n_q * a.G - tile * a.tile_rows); }
    __device__ __forceinline__ bool whole() const { return pg0 == 0 && pg1 == pages; }
    // which of a CTA's two places in scratch a segment of a cut item takes
    __device__ __forceinline__ int place() const { return from > 0 ? 0 : 1; }
    // Whether this CTA has a part of the item at `from`: its tile exists and sees a page of the range.
    __device__ __forceinline__ bool set(const RowsArgs& a) {
        to = (int)min((long long)item_pages(s, item, a), from + left);
        tile = a.group == 1 ? item : item * a.group + (int)blockIdx.x % a.group;
        if (tile >= s.tiles) return false;
        pages = tile_pages(s, tile, a);
        pg0 = from;
        pg1 = min(to, pages);
        return pg0 < pg1;
    }
    // The next segment of the range; false when there is none.
    __device__ __forceinline__ bool next(const int* __restrict__ cu_q, const int* __restrict__ kv_len, const RowsArgs& a, int* status) {
        do {
            left -= to - from;
            if (left <= 0) return false;
            from = 0;
            if (++item == seq_items(s, a)) {
                item = 0;
                if (++g == a.KV) {
                    g = 0;
                    do {
                        if (++b >= a.B) return false;
                        s = seq_shape(cu_q, kv_len, b, a, status);
                    } while (s.n_q == 0);
                }
            }
        } while (!set(a));
        return true;
    }
};

// Where a range begins: what the joining launch goes by. from > 0: inside item (b, g, item).
struct RowStart {
    int b, g, item, from;             // b < 0: behind the end of the line
};

__device__ __forceinline__ long long warp_sum_ll(long long v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ long long warp_scan_ll(long long v, int lane) {      // sum over the lanes up to this one
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long x = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += x;
    }
    return v;
}
// Quotients of numbers that hardly ever need 64 bits.
__device__ __forceinline__ long long div_ll(long long x, long long y) {
    return ((x | y) >> 32) == 0 ? (long long)((uint32_t)x / (uint32_t)y) : x / y;
}

// The start of this CTA's range, for one whole warp, into `at` (b < 0: nothing to do) and, for the joining launch, starts[range];
// starts[ctas].from is the length of a range.
__device__ __forceinline__ void find_range(const int* __restrict__ cu_q, const int* __restrict__ kv_len, const RowsArgs& a, RowWalk* at,
                                           RowStart* starts, int* status) {
    const int lane = threadIdx.x & 31, cta = blockIdx.x / a.group;
    const bool writes = a.group == 1 || blockIdx.x % a.group == 0;
    long long total = 0, own = 0;
    SeqShape s;
    for (int b0 = 0; b0 < a.B; b0 += 32) {
        own = 0;
        if (b0 + lane < a.B) {
            s = seq_shape(cu_q, kv_len, b0 + lane, a, status);
            own = seq_pages(s, a) * a.KV;
        }
        total += warp_sum_ll(own);
    }
    const long long range = max((long long)a.min_range, div_ll(total + a.ctas - 1, a.ctas));
    const long long from = range * cta;
    if (lane == 0) {
        at->b = -1;
        if (writes && from >= total) starts[cta] = RowStart{-1, 0, 0, 0};
        if (blockIdx.x == 0) starts[a.ctas] = RowStart{0, 0, 0, (int)min(range, 0x7fffffffll)};
    }
    __syncwarp();
    if (from >= total) return;
    long long base = 0;
    for (int b0 = 0; b0 < a.B; b0 += 32) {
        if (a.B > 32) {                                        // (of up to 32 sequences every lane still has its own)
            own = 0;
            if (b0 + lane < a.B) {
                s = seq_shape(cu_q, kv_len, b0 + lane, a, status);
                own = seq_pages(s, a) * a.KV;
            }
        }
        const long long incl = warp_scan_ll(own, lane), excl = incl - own;
        if (own > 0 && from >= base + excl && from < base + incl) {
            RowWalk w;
            w.b = b0 + lane;
            w.s = s;
            const long long each = div_ll(own, a.KV);
            long long x = from - base - excl;
            w.g = (int)div_ll(x, each);
            x -= w.g * each;
            if (a.causal) {
                w.item = 0;
                for (int p; x >= (p = item_pages(s, w.item, a)); w.item++) x -= p;
            } else {
                w.item = (int)div_ll(x, s.pages);
                x -= (long long)w.item * s.pages;
            }
            w.from = (int)x;
            w.left = range;
            if (writes) starts[cta] = RowStart{w.b, w.g, w.item, w.from};
            if (w.set(a) || w.next(cu_q, kv_len, a, status)) *at = w;
        }
        base += __shfl_sync(0xffffffffu, incl, 31);
        if (from < base) break;
    }
    __syncwarp();
}

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
