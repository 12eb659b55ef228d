// How attention of a few rows a sequence over a paged cache is shared out among CTAs, for the kernels of attn_rows.cu and
// attn_rows_tcgen05.cu.
//
// The query heads that share a kv head are rows of one problem: packed row r of a sequence is token r / G, head r % G of the
// group (G = H / KV). A tile is `tile_rows` packed rows; an item is one tile against all keys it may see, for one kv head; its
// length is the number of those keys' pages. What a CTA takes of an item is a segment. There are two ways:
//
//   pieces  every item is cut into pieces of equal numbers of pages, of `each` at most, a CTA a piece. `each` is the least that
//           leaves no more pieces than CTAs. One segment a CTA, but items that do not divide well leave CTAs idle.
//   line    all items lie one behind the other (by sequence, kv head, item), and CTA c takes the `range` pages from c * range on:
//           every CTA has the same number of pages, however ragged the batch, but a range that reaches from one item into the
//           next is two segments, and most items are cut.
//
// The line is taken where `each` exceeds `range` by more than a segment and a join cost (LINE_COST pages). 8 trees of 24 tokens
// behind 2,050 rows, 16 heads: PIECES8; a decode step of 64 sequences of 3,000 rows, 32 heads: LINE64. An item that one CTA has
// whole is finished there; of the others every CTA leaves its segment's maximum, sum and unnormalised output in scratch (at
// most two a CTA: one whose item began before, one whose item goes on), and a second launch joins them: there is one CTA (and
// its helpers) of that launch for every CTA of the first, which finds there what that one wrote down of its start.
//
// Everything is worked out on the device from the step's description, so a captured launch serves whatever lengths its replays
// bring. Where sequences have several tiles, `group` CTAs side by side take the same pages for `group` tiles (an item is then
// that many tiles), so that a page comes from memory once and from L2 for the others: 16 trees of 64 tokens with four heads a kv
// head (two tiles each) behind 8,191 rows read 1.05 GB one tile after the other, 0.54 GB together.
#pragma once
#include "layout.cuh"

struct RowsArgs {
    int T, B, H, KV, HD, G;
    int ldq, ldo;
    int tile_rows;                    // packed rows a tile
    int most_rows;                    // of one tile that the step's longest sequence fills
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
    int list0, list1;                 // its page list: entries [list0, list1), the first one for logical page `first`
    int first;
};

// A sequence's numbers. Bounds that cannot be (rows outside the step, fewer keys than rows) count as a sequence without rows
// and are reported.
__device__ __forceinline__ SeqShape seq_shape(const int* __restrict__ cu_q, const int* __restrict__ kv_len, const PageTable& pt, int b,
                                              const RowsArgs& a, int* status) {
    SeqShape s;
    s.q_begin = cu_q[b];
    const int end = cu_q[b + 1];
    s.list0 = pt.indptr[b];
    s.list1 = pt.indptr[b + 1];
    s.first = pt.base[b];
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

// The physical page of a sequence's logical page, or -1.
__device__ __forceinline__ int page_at(const PageTable& pt, const SeqShape& s, int page) {
    const int at = s.list0 + page - s.first;
    if (at < s.list0 || at >= s.list1) return -1;
    const int id = pt.ids[at];
    return id >= 0 && id < pt.n_pages ? id : -1;
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
    long long left;                   // pages that are left of what this CTA takes, this segment's among them
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
    __device__ __forceinline__ bool next(const int* __restrict__ cu_q, const int* __restrict__ kv_len, const PageTable& pt, const RowsArgs& a,
                                         int* status) {
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
                        s = seq_shape(cu_q, kv_len, pt, b, a, status);
                    } while (s.n_q == 0);
                }
            }
        } while (!set(a));
        return true;
    }
};

// Where a CTA begins: what the joining launch goes by. from > 0: inside item (b, g, item), of which a CTA has `each` pages.
struct RowStart {
    int b, g, item, from;             // b < 0: nothing
    int each, pad[3];
};
constexpr int LINE_COST = 16;

__device__ __forceinline__ long long warp_sum_ll(long long v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
// The same where no lane has more than 2^26, which is all but always.
__device__ __forceinline__ long long warp_sum_small(long long v) {
    if (__all_sync(0xffffffffu, v < (1ll << 26))) return (long long)__reduce_add_sync(0xffffffffu, (unsigned)v);
    return warp_sum_ll(v);
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

// Pieces of one kv head's items of a sequence.
__device__ __forceinline__ int seq_pieces(const SeqShape& s, int each, const RowsArgs& a) {
    const int items = seq_items(s, a);
    if (!a.causal || items <= 1) return items * ((s.pages + each - 1) / each);
    int n = 0;
    for (int i = 0; i < items; i++) n += (item_pages(s, i, a) + each - 1) / each;
    return n;
}

// The start of this CTA, for one whole warp, into `at` (b < 0: nothing to do) and, for the joining launch, starts[CTA].
__device__ __forceinline__ void find_start(const int* __restrict__ cu_q, const int* __restrict__ kv_len, const PageTable& pt,
                                           const RowsArgs& a, RowWalk* at, RowStart* starts, int* status) {
    const int lane = threadIdx.x & 31, cta = blockIdx.x / a.group;
    const bool writes = a.group == 1 || blockIdx.x % a.group == 0;
    long long total = 0, own = 0;
    SeqShape s;
    s.tiles = s.pages = 0;
    for (int b0 = 0; b0 < a.B; b0 += 32) {
        own = 0;
        if (b0 + lane < a.B) {
            s = seq_shape(cu_q, kv_len, pt, b0 + lane, a, status);
            own = seq_pages(s, a) * a.KV;
        }
        total += warp_sum_small(own);
    }
    const long long range = max((long long)a.min_range, div_ll(total + a.ctas - 1, a.ctas));
    // Pieces, for up to 32 sequences: the least `each` of range .. range + LINE_COST that makes no more pieces than there are CTAs.
    int each = 0;
    if (a.B <= 32 && range < (1 << 20)) {
        int lo = (int)range, hi = (int)range + LINE_COST + 1;
        while (lo < hi) {                                      // hi: fits, or is beyond what pays
            const int mid = (lo + hi) / 2;
            const bool fits = warp_sum_small(s.tiles > 0 ? (long long)seq_pieces(s, mid, a) * a.KV : 0) <= a.ctas;
            if (fits) hi = mid; else lo = mid + 1;
        }
        if (lo <= (int)range + LINE_COST) each = lo;
    }
    if (lane == 0) at->b = -1;
    __syncwarp();
    long long base = 0, pieces = 0;
    if (each > 0) {
        pieces = s.tiles > 0 ? (long long)seq_pieces(s, each, a) * a.KV : 0;
        total = warp_sum_small(pieces);
    }
    const long long from = each > 0 ? cta : range * cta;       // in pieces, or in pages
    if (from >= total) {
        if (lane == 0 && writes) starts[cta].b = -1;
        return;
    }
    for (int b0 = 0; b0 < a.B; b0 += 32) {
        if (a.B > 32) {                                        // (of up to 32 sequences every lane still has its own)
            own = 0;
            if (b0 + lane < a.B) {
                s = seq_shape(cu_q, kv_len, pt, b0 + lane, a, status);
                own = seq_pages(s, a) * a.KV;
            }
        }
        const long long mine = each > 0 ? pieces : own, incl = warp_scan_ll(mine, lane), excl = incl - mine;
        if (mine > 0 && from >= base + excl && from < base + incl) {
            RowWalk w;
            w.b = b0 + lane;
            w.s = s;
            const long long head = div_ll(mine, a.KV);         // one kv head's
            long long x = from - base - excl;
            w.g = (int)div_ll(x, head);
            x -= w.g * head;
            w.item = 0;
            if (each > 0) {
                int p = item_pages(s, 0, a), n = (p + each - 1) / each;
                if (!a.causal) {
                    w.item = (int)x / n;
                    x -= (long long)w.item * n;
                } else {
                    while (x >= n) {
                        x -= n;
                        p = item_pages(s, ++w.item, a);
                        n = (p + each - 1) / each;
                    }
                }
                w.left = (p + n - 1) / n;                      // pieces of one size
                w.from = (int)(x * w.left);
            } else {
                w.left = range;
                if (!a.causal) {
                    w.item = (int)div_ll(x, s.pages);
                    x -= (long long)w.item * s.pages;
                } else {
                    for (int p; x >= (p = item_pages(s, w.item, a)); w.item++) x -= p;
                }
                w.from = (int)x;
            }
            if (writes) starts[cta] = RowStart{w.b, w.g, w.item, w.from, (int)min(w.left, 0x7fffffffll)};
            // (a piece is one segment: what is left of it when the item ends is nobody's)
            const bool has = w.set(a);
            if (each > 0) w.left = w.to - w.from;
            if (has || w.next(cu_q, kv_len, pt, a, status)) *at = w;
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
