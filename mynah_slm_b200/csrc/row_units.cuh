// How attention of a few rows a sequence over a paged cache is shared out among CTAs, for the kernels of attn_rows.cu and
// attn_rows_tcgen05.cu.
//
// The query heads that share a kv head are rows of one problem: packed row r of a sequence is token r / G, head r % G of the
// group (G = H / KV). A tile is `tile_rows` packed rows; an item is one tile against all keys it may see, for one kv head; its
// length is the number of those keys' pages. What a CTA takes of an item in one go is a segment. An item that is one segment is
// finished where it is; of the others every segment leaves its maximum, sum and unnormalised output in scratch, and a second launch
// joins them.
//
// On the tensor cores items are cut by the whole step, in one of three ways:
//
//   items   a CTA an item, the longest of every sequence first, nothing is cut: steps with enough tiles for that (prompts).
//
//   pieces  every item is cut into pieces of equal numbers of pages, of `each` at most, a CTA a piece. The longest item has as
//           many pieces as all items can have with a CTA for each. One segment a CTA, but shorter items and numbers that do not
//           divide well leave CTAs idle.
//   line    all items lie one behind the other (by sequence, kv head, item), and CTA c takes the `range` pages from c * range on:
//           every CTA has the same number of pages, however ragged the batch, but a range that reaches from one item into the
//           next is two segments, and most items are cut.
//
// The line is taken where `each` exceeds `range` by more than a segment and a join cost (LINE_COST pages), and for more sequences
// than a warp has lanes. Pieces against line: 8 trees of 24 tokens behind up to 2,050 rows, 16 heads (9 pages each, a range of 8)
// 29.7 us against 33.9; 16 trees of 8, one behind 800 rows, 15 behind 500 (7 and 4) 22.5 against 22.7; behind 1,600 and 500 rows
// (13 and 4) 26.7 against 24.1, behind 8,000 and 500 (63 and 7) 73.9 against 30.9; 24 trees of 8 behind 1,600 rows (26 and 17)
// 43.5 both, behind 9,000 (141 and 92) 165 against 149. A CTA has at most two segments of cut items (one whose item began before, one
// whose item goes on), each with a place of its own in scratch, and writes down where it begins for the launch that joins.
//
// On the general kernel (OWN) items are cut by their own sequence alone (own_cut): in 32 bits what a sequence gets, and which rows of it
// a bounded cache keeps, has the same bits whatever else is in the step. Up to OWN_PIECES pieces for all rows of a sequence
// together, of equal numbers of pages, lie on a line as above, and CTA c takes those that begin in its range. A row's bits do not
// depend on the tile it is in either: what a page, a rescaling or a join does to a row does not involve the rows beside it, and
// pages that a row does not see add exact zeros. It costs segments, joins and some balance, in fp32 against the step's cut: 3 trees of
// 19 behind up to 1,021 rows the same, 8 of 40 behind up to 4,000, 16 heads of 128 on 4, 490 us -> 551, 64 of 60 behind up to 500 645
// -> 791; with sums, 64 tokens behind up to 4,000 rows, 32 heads of 128 on 8, 1,480 -> 1,536, 2,048 tokens, 16 heads of 64 on 8, 717 ->
// 781, 2 pieces of 150 behind 333 the same, 3 of 420 behind up to 800, 8 heads of 64 on 4, 145 -> 170. Half as many pieces take
// one piece of 300 behind 2,000 rows from 93 to 165, at least two pages a piece the 3 trees of 19 from 25 to 35. On the tensor cores, where pages are so much quicker than
// the ends of segments, the same cut made 64 tokens 169 us -> 226, 262, 337 (pieces of at least eight, four, two pages) and 600
// tokens behind up to 500 rows 331 -> 482, 647, 703; there the step's cut stays.
//
// Everything is worked out on the device from the step's description (in few instructions: a CTA's first trip through any code
// waits for that code, about 0.3 us for every 128 bytes of it, which is most of what a small call takes), so a captured launch
// serves whatever lengths its replays bring. Where sequences have several tiles, `group` CTAs side by side take the same pages for
// `group` tiles (an item is then that many tiles), so that a page comes from memory once and from L2 for the others: 16 trees of
// 64 tokens with four heads a kv head (two tiles each) behind 8,191 rows read 1.05 GB one tile after the other, 0.54 GB together.
#pragma once
#include "layout.cuh"

// Quotient of x < 2^31 and a divisor that the host knows: multiply and shift.
struct FastDiv {
    uint32_t by, mul;
    int shift;
    static FastDiv of(int d) {
        int s = 0;
        while ((1ll << s) < d) s++;                                // 2^s >= d: (2^(31 + s) / d rounded up) fits 32 bits and is exact below 2^31
        return FastDiv{(uint32_t)d, (uint32_t)(((1ull << (31 + s)) + d - 1) / d), 31 + s};
    }
    __device__ __forceinline__ int div(int x) const { return (int)(((unsigned long long)(uint32_t)x * mul) >> shift); }
    __device__ __forceinline__ int mod(int x) const { return x - div(x) * (int)by; }
};

struct RowsArgs {
    int T, B, H, KV, HD, G;
    int most_q;                       // rows of a sequence at most: a longer one is refused
    int ldq, ldo;
    int tile_rows;                    // packed rows a tile
    int most_rows;                    // of one tile that the step's longest sequence fills
    int whole_items;                  // 1: a CTA an item
    int two;                          // 1: the tcgen05 kernel's tile is two of its own
    int min_range;                    // pages a CTA, or a piece, at least
    int ctas;                         // ranges that the line is cut into, or pieces; the launch has ctas * group CTAs
    int group;                        // tiles an item, each a CTA's
    int causal;                       // 1: token i sees rows <= past + i; 0: the mask words (the kernels have an instance for each)
    int own;                          // 1: items are cut by their own sequence alone
    long long cut_rows;               // own: rows of scratch that there are for cut items
    int words;                        // mask words a token
    float scale_log2;                 // score scale * log2(e)
    int q_aligned;                    // 1: q's and the output's rows are whole 16-byte pieces
    FastDiv by_G, by_tile, by_group, by_KV, by_ctas, by_quads;
    void finish() {                   // once the numbers above stand
        by_G = FastDiv::of(G), by_tile = FastDiv::of(tile_rows), by_group = FastDiv::of(group), by_KV = FastDiv::of(KV), by_ctas = FastDiv::of(ctas);
        by_quads = FastDiv::of(HD >= 4 ? HD / 4 : 1);
    }
};
constexpr int LINE_COST = 6;
constexpr int OWN_PIECES = 256;       // pieces of a sequence's rows at most (OWN): about one for every place that CTAs have on the device
constexpr int OWN_ROWS = 64;          // rows that count as one there, whatever the tiles are
// Most page visits of a step (pages of every tile's keys, over the kv heads) that the numbers below are made for: a prompt of a
// million tokens and 32 heads. A step of more is refused through the status word.
constexpr long long MAX_VISITS = 1ll << 30;

// Quotient of two numbers of the device's, 0 <= x < 2^31, y > 0. Below 2^22 the fp32 quotient is off by less than one.
__device__ __forceinline__ int quotient(int x, int y) {
    if (x >= 1 << 22) return x / y;
    const int q = (int)__fdividef((float)x, (float)y), r = x - q * y;
    return q + (r >= y ? 1 : 0) - (r < 0 ? 1 : 0);
}

struct SeqShape {
    int q_begin, n_q, kvl, tiles, pages;
    int list0, list1;                 // its page list: entries [list0, list1), the first one for logical page `first`
    int first;
};

// A sequence's numbers. Bounds that cannot be (rows outside the step, fewer keys than rows, more rows than the call was made for)
// count as a sequence without rows and are reported.
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
    if (s.n_q <= 0 || s.q_begin < 0 || end > a.T || s.kvl < s.n_q || s.n_q > a.most_q) {
        if (s.n_q != 0) atomicOr(status, MYNAH_ST_PAGE_RANGE);
        s.n_q = 0;
    }
    s.tiles = a.by_tile.div(s.n_q * a.G + a.tile_rows - 1);
    s.pages = s.n_q > 0 ? (int)(((unsigned)s.kvl + PAGE_TOKENS - 1) / PAGE_TOKENS) : 0;
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
template <bool CAUSAL> __device__ __forceinline__ int tile_pages(const SeqShape& s, int tile, const RowsArgs& a) {
    if (!CAUSAL) return s.pages;
    const int last = a.by_G.div(min(s.n_q * a.G, (tile + 1) * a.tile_rows) - 1);
    return (s.kvl - s.n_q + last) / PAGE_TOKENS + 1;
}

__device__ __forceinline__ int seq_items(const SeqShape& s, const RowsArgs& a) { return a.by_group.div(s.tiles + a.group - 1); }
// Pages of an item: of its last tile, which sees the most.
template <bool CAUSAL> __device__ __forceinline__ int item_pages(const SeqShape& s, int item, const RowsArgs& a) {
    return tile_pages<CAUSAL>(s, min(s.tiles, (item + 1) * a.group) - 1, a);
}
// Pages of the sequence's items together, for one kv head.
template <bool CAUSAL> __device__ __forceinline__ long long seq_pages(const SeqShape& s, const RowsArgs& a) {
    const int items = seq_items(s, a);
    if (!CAUSAL || items <= 1) return (long long)items * s.pages;
    long long n = 0;
#pragma unroll 1
    for (int i = 0; i < items; i++) n += item_pages<CAUSAL>(s, i, a);
    return n;
}

// How the items of a sequence of causal rows are cut: into up to n pieces of `each` pages. By the sequence's own numbers and the
// model's alone, and not by its tiles, whose size goes by the step. (The pages that its list has bound what its scratch takes.)
struct OwnCut {
    int n, each;
};
__device__ __forceinline__ OwnCut own_cut(const SeqShape& s, const RowsArgs& a) {
    if (s.n_q == 0) return OwnCut{1, 1};
    const int tiles = min(OWN_PIECES, (s.n_q * a.G + OWN_ROWS - 1) / OWN_ROWS) * a.KV;
    const int listed = max(1, min(s.pages, s.list1 - s.list0));
    const int n = min(max(1, quotient(OWN_PIECES, tiles)), quotient(listed + a.min_range - 1, a.min_range));
    const int each = quotient(s.pages + n - 1, n);
    return OwnCut{quotient(s.pages + each - 1, each), each};
}
// Rows of scratch that the sequence's cut items take: row (g * n + piece) * (rows of the sequence) + its packed row, behind those of
// the sequences before it.
__device__ __forceinline__ int own_rows(const SeqShape& s, const OwnCut& c, const RowsArgs& a) { return c.n > 1 ? a.KV * c.n * s.n_q * a.G : 0; }

// Where a CTA is, and the segment it is at: pages [pg0, pg1) of one tile of item (b, g, item).
template <bool CAUSAL, bool OWN> struct RowWalk {
    int b, g, item, tile, pg0, pg1;
    int from, to;                     // the item's pages in this range (OWN: of this piece)
    int pages;                        // that the tile may see
    int left;                         // pages that are left of what this CTA takes, this segment's among them
    SeqShape s;
    OwnCut cut;                       // (OWN)
    long long rows0;                  // (OWN) rows of scratch before the sequence's

    __device__ __forceinline__ int past() const { return s.kvl - s.n_q; }
    __device__ __forceinline__ int rows(const RowsArgs& a) const { return min(a.tile_rows, s.n_q * a.G - tile * a.tile_rows); }
    __device__ __forceinline__ bool whole() const { return pg0 == 0 && pg1 == pages; }
    // The row of scratch that the tile's first row takes in a segment of a cut item (not OWN: one of the CTA's two places).
    __device__ __forceinline__ long long scratch_row(const RowsArgs& a) const {
        if (OWN) return rows0 + (long long)(g * cut.n + quotient(pg0, cut.each)) * (s.n_q * a.G) + tile * a.tile_rows;
        return ((long long)blockIdx.x * 2 + (from > 0 ? 0 : 1)) * a.tile_rows;
    }
    // Whether this CTA has a part of the item at `from`: its tile exists and sees a page of the range.
    __device__ __forceinline__ bool set(const RowsArgs& a) {
        to = min(item_pages<CAUSAL>(s, item, a), from + (OWN ? cut.each : left));
        tile = item * a.group + a.by_group.mod(blockIdx.x);
        if (tile >= s.tiles) return false;
        pages = tile_pages<CAUSAL>(s, tile, a);
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
            if (OWN && to < item_pages<CAUSAL>(s, item, a)) {
                from = to;                                         // the item's next piece
                continue;
            }
            from = 0;
            if (++item == seq_items(s, a)) {
                item = 0;
                if (++g == a.KV) {
                    g = 0;
                    if (OWN) rows0 += own_rows(s, cut, a);
                    do {
                        if (++b >= a.B) return false;
                        s = seq_shape(cu_q, kv_len, pt, b, a, status);
                    } while (s.n_q == 0);
                    if (OWN) cut = own_cut(s, a);
                }
            }
        } while (!set(a));
        return true;
    }
};

// Where a CTA begins: what the joining launch goes by (not OWN). from > 0: inside item (b, g, item), of which a CTA has `each` pages.
struct RowStart {
    int b, g, item, from;             // b < 0: nothing
    int each, pad[3];
};

__device__ __forceinline__ long long warp_sum_ll(long long v) {
#pragma unroll 1
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ int warp_scan(int v, int lane) {        // sum over the lanes up to this one
#pragma unroll 1
    for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += x;
    }
    return v;
}

// The start of this CTA, for one whole warp, into `at` (b < 0: nothing to do) and, for the joining launch, starts[CTA].
template <bool CAUSAL, bool OWN>
__device__ __forceinline__ void find_start(const int* __restrict__ cu_q, const int* __restrict__ kv_len, const PageTable& pt,
                                           const RowsArgs& a, RowWalk<CAUSAL, OWN>* at, RowStart* starts, int* status) {
    const int lane = threadIdx.x & 31, cta = a.by_group.div(blockIdx.x);
    const bool writes = !OWN && a.by_group.mod(blockIdx.x) == 0, whole_items = CAUSAL && !OWN && a.whole_items;
    long long all = 0, own = 0;
    int items = 0, longest = 0;
    bool alike = true;                                             // every item of a sequence has its pages
    SeqShape s;
    s.n_q = s.tiles = s.pages = 0;
#pragma unroll 1
    for (int b0 = 0; b0 < a.B; b0 += 32) {
        own = 0;
        if (b0 + lane < a.B) {
            s = seq_shape(cu_q, kv_len, pt, b0 + lane, a, status);
            items = seq_items(s, a);
            own = (whole_items ? items : seq_pages<CAUSAL>(s, a)) * a.KV;
            alike = !CAUSAL || items <= 1;
            longest = s.pages;
        }
        all += own;
    }
    all = __all_sync(0xffffffffu, all < (1ll << 26)) ? (long long)__reduce_add_sync(0xffffffffu, (unsigned)all) : warp_sum_ll(all);
    if (lane == 0) at->b = -1;
    if (all > MAX_VISITS) {
        if (lane == 0) atomicOr(status, MYNAH_ST_SPLIT_RANGE);
        all = 0;
    }
    int total = (int)all;
    const int range = max(a.min_range, a.by_ctas.div(total + a.ctas - 1));
    // Pieces, for up to 32 sequences whose items are alike, where they pay.
    int each = 0, n = 0;                                           // n: pieces of one of this lane's items
    if (!OWN && !whole_items && a.B <= 32 && __all_sync(0xffffffffu, alike)) {
        const int lots = (int)__reduce_add_sync(0xffffffffu, (unsigned)items) * a.KV;
        if (lots > 0 && lots <= a.ctas) {
            longest = (int)__reduce_max_sync(0xffffffffu, (unsigned)longest);
            const int most = quotient(a.ctas, lots);
            each = max(a.min_range, quotient(longest + most - 1, most));
            if (each > range + LINE_COST) {
                each = 0;
            } else {
                n = quotient(s.pages + each - 1, each);
                own = (long long)(items * n) * a.KV;
                total = (int)__reduce_add_sync(0xffffffffu, (unsigned)own);
            }
        }
    }
    const long long from64 = each > 0 || whole_items ? cta : (long long)range * cta;         // in pieces, in items, or in pages
    __syncwarp();
    if (from64 >= total) {
        if (lane == 0 && writes) starts[cta].b = -1;
        return;
    }
    const int from = (int)from64;
    int base = 0;
    long long rows0 = 0;
#pragma unroll 1
    for (int b0 = 0; b0 < a.B; b0 += 32) {
        if (a.B > 32) {                                            // (of up to 32 sequences every lane still has its own)
            own = 0;
            s.n_q = 0;
            if (b0 + lane < a.B) {
                s = seq_shape(cu_q, kv_len, pt, b0 + lane, a, status);
                own = (whole_items ? seq_items(s, a) : seq_pages<CAUSAL>(s, a)) * a.KV;
            }
        }
        const int mine = (int)own, incl = a.B == 1 ? mine : warp_scan(mine, lane);
        OwnCut cut{1, 1};
        int held = 0, held_incl = 0;
        if (OWN) {
            cut = own_cut(s, a);
            held = own_rows(s, cut, a);
            held_incl = a.B == 1 ? held : warp_scan(held, lane);
        }
        int x = from - base - (incl - mine);                       // within this lane's sequence
        if (x >= 0 && x < mine) {
            RowWalk<CAUSAL, OWN> w;
            w.b = b0 + lane;
            w.s = s;
            const int head = a.by_KV.div(mine);                    // one kv head's
            w.g = quotient(x, head);
            x -= w.g * head;
            w.item = 0;
            int p = 0;                                             // pages of the item
            if (whole_items) {
                x = from - base - (incl - mine);
                w.item = head - 1 - a.by_KV.div(x);                // (the last tile sees the most)
                w.g = a.by_KV.mod(x);
            } else if (!CAUSAL) {
                p = s.pages;
                const int one = each > 0 ? n : p;                  // of one item
                w.item = quotient(x, one);
                x -= w.item * one;
            } else if (each == 0) {
                p = item_pages<CAUSAL>(s, 0, a);
#pragma unroll 1
                while (x >= p) {
                    x -= p;
                    p = item_pages<CAUSAL>(s, ++w.item, a);
                }
            }
            bool has;
            if (OWN) {
                w.cut = cut;
                w.rows0 = rows0 + held_incl - held;
                w.from = min(p, quotient(x + cut.each - 1, cut.each) * cut.each);       // the first piece that begins here or later
                w.left = range - (w.from - x);
                w.to = w.from;
                has = w.from < p && w.left > 0 && w.set(a);
            } else {
                w.left = whole_items ? s.pages : each > 0 ? quotient(s.pages + n - 1, n) : range;      // pieces of one size
                w.from = whole_items ? 0 : each > 0 ? x * w.left : x;
                if (writes) starts[cta] = RowStart{w.b, w.g, w.item, w.from, w.left};
                has = w.set(a);
                // (a piece is one segment: what is left of it when the item ends is nobody's)
                if (each > 0 || whole_items) w.left = w.to - w.from;
            }
            if (has || w.next(cu_q, kv_len, pt, a, status)) *at = w;
        }
        base += __shfl_sync(0xffffffffu, incl, 31);
        if (OWN) rows0 += __shfl_sync(0xffffffffu, held_incl, 31);
        if (from < base) break;
    }
    __syncwarp();
}

// Tile number `flat` of the step's, sequence by sequence, and the rows of scratch before its sequence's, for one whole warp: the
// sequence, or -1 (OWN).
__device__ __forceinline__ int find_tile(const int* __restrict__ cu_q, const int* __restrict__ kv_len, const PageTable& pt, const RowsArgs& a, int flat,
                                         int& tile, long long& rows0, int* status) {
    const int lane = threadIdx.x & 31;
    int base = 0;
    rows0 = 0;
#pragma unroll 1
    for (int b0 = 0; b0 < a.B; b0 += 32) {
        int tiles = 0, held = 0;
        if (b0 + lane < a.B) {
            const SeqShape s = seq_shape(cu_q, kv_len, pt, b0 + lane, a, status);
            tiles = s.tiles;
            held = own_rows(s, own_cut(s, a), a);
        }
        const int incl = warp_scan(tiles, lane), held_incl = warp_scan(held, lane);
        const unsigned hit = __ballot_sync(0xffffffffu, flat >= base + incl - tiles && flat < base + incl);
        if (hit != 0u) {
            const int src = __ffs(hit) - 1;
            tile = flat - base - __shfl_sync(0xffffffffu, incl - tiles, src);
            rows0 += __shfl_sync(0xffffffffu, held_incl - held, src);
            return b0 + src;
        }
        base += __shfl_sync(0xffffffffu, incl, 31);
        rows0 += __shfl_sync(0xffffffffu, held_incl, 31);
    }
    return -1;
}
// Which of the 64 keys from key0 (a multiple of 64) on token `tok` of a sequence sees: bit e for key key0 + e. Held rows (below
// past) are seen by all; of the step's own rows, those up to the token's own (causal), or those whose bits are set in the
// token's mask words. Keys at and behind kvl are never seen, whatever the words say.
template <bool CAUSAL>
__device__ __forceinline__ unsigned long long visible64(int key0, int kvl, int past, int tok, const long long* __restrict__ words, int n_words) {
    const int n = kvl - key0;
    if (n <= 0) return 0ull;
    const unsigned long long all = ~0ull, lim = n >= 64 ? all : (1ull << n) - 1ull;
    if (CAUSAL) {
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
