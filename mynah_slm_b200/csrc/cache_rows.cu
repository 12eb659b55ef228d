// Rows of the paged cache that stay and rows that go: the eviction of the rows that gathered the least attention, and the
// acceptance of a drafted tree's path. Both end in moving rows of K and V to lower rows of the same sequence, for all layers
// that share the page lists, in one launch.
#include "attn_rows.cuh"

namespace {

// ------------------------------------------------------------------ choosing

constexpr int CH_THREADS = 512, CH_WARPS = CH_THREADS / 32;
constexpr int CH_BITS = 11, CH_BINS = 1 << CH_BITS;       // of a word that one pass settles (the last pass: the ten that are left)

// A sum's order as an unsigned word: greater sums have greater words, both zeros the same one, a NaN the greatest.
__device__ __forceinline__ uint32_t order_of(float x) {
    if (x != x) return 0xffffffffu;
    const uint32_t u = __float_as_uint(x + 0.0f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

struct EvictArgs {
    int E, B, KV, n_pages, keep, recent, first, cached;   // cached: rows whose words fit the shared memory that was asked for
};

// One CTA for one (layer, sequence, kv head): the rows that stay, ascending. Of n > keep rows the first `first` and the last
// `recent` stay anyway; of those between them the `need` = keep - first - recent with the greatest sums. The need-th greatest
// word is found in three passes, 11, 11 and 10 bits (a histogram of the words that still agree with it in the bits above, the bin
// that holds it, and so on); then every warp takes a run of rows, counts those above it and those equal to it, and, once it
// knows the counts of the runs before, writes its own: those above, and the first of the equal ones. The words are read from
// memory once where they fit shared memory. Bound by its chain of barriers and passes, so up to four CTAs an SM (32 registers a thread;
// four where the page lists of the step have up to about 190 entries together, three to 265, two beyond: see the launch): 448 choices of 2,048 of 4,100 rows 27.5 us, against 35 with two (64 registers), which are 5% faster for rows beyond shared
// memory (48 choices of 8,192 of 20,000: 96 and 101 us); with 256 threads 30 and 167.
__global__ void __launch_bounds__(CH_THREADS, 4)
evict_choose_kernel(const float* __restrict__ mass, PageTable pt, const int* __restrict__ kv_len, EvictArgs a, int* __restrict__ kept,
                    int* __restrict__ new_len, int* __restrict__ status) {
    extern __shared__ uint32_t words_s[];
    __shared__ int hist[CH_BINS];
    __shared__ int warp_s[CH_WARPS], equal_s[CH_WARPS];
    __shared__ int found[2];
    const int unit = blockIdx.x, g = unit % a.KV, b = unit / a.KV % a.B, e = unit / a.KV / a.B;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int n = max(0, kv_len[b]);
    int* out = kept + (size_t)unit * a.keep;
    if (e == 0 && g == 0 && tid == 0) new_len[b] = min(n, a.keep);
    if (n <= a.keep) {
        for (int i = tid; i < a.keep; i += CH_THREADS) out[i] = i < n ? i : -1;
        return;
    }
    const float* m = mass + ((size_t)e * a.n_pages * a.KV + g) * PAGE_TOKENS;
    const int lo = a.first, hi = n - a.recent, need = a.keep - a.first - a.recent;
    const bool cached = hi - lo <= a.cached;
    const int list0 = pt.indptr[b] - pt.base[b], list_lo = pt.indptr[b], list_hi = pt.indptr[b + 1];
    bool bad = false;
    auto word_at = [&](int r) {
        const int at = list0 + r / PAGE_TOKENS;
        int page = at >= list_lo && at < list_hi ? pt.ids[at] : -1;
        if (page < 0 || page >= a.n_pages) {
            bad = true;
            return 0u;
        }
        return order_of(m[(size_t)page * a.KV * PAGE_TOKENS + r % PAGE_TOKENS]);
    };
    auto word = [&](int r) { return cached ? words_s[r - lo] : word_at(r); };
    for (int i = tid; i < CH_BINS; i += CH_THREADS) hist[i] = 0;
    if (cached && need > 0) {
#pragma unroll 8
        for (int r = lo + tid; r < hi; r += CH_THREADS) words_s[r - lo] = word_at(r);
    }
    uint32_t prefix = 0;
    int left = need;                                       // the left-th greatest among the words with this prefix is sought
    for (int pass = 0; pass < 3 && need > 0; pass++) {
        const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
        const uint32_t above = pass == 0 ? 0u : pass == 1 ? 0xffe00000u : 0xfffffc00u, mask = pass == 2 ? 1023u : 2047u;
        __syncthreads();                                   // (words and empty bins)
#pragma unroll 4
        for (int r = lo + tid; r < hi; r += CH_THREADS) {
            const uint32_t w = word(r);
            if ((w & above) == prefix) atomicAdd(&hist[(w >> shift) & mask], 1);
        }
        __syncthreads();
        // bins from the greatest down, four a thread
        int own[4], sum = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            own[i] = hist[CH_BINS - 1 - (tid * 4 + i)];
            sum += own[i];
        }
        int incl = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += v;
        }
        if (lane == 31) warp_s[warp] = incl;
        __syncthreads();
        int before = incl - sum;
        for (int i = 0; i < warp; i++) before += warp_s[i];
        if (before < left && before + sum >= left) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                if (before < left && before + own[i] >= left) {
                    found[0] = CH_BINS - 1 - (tid * 4 + i);
                    found[1] = left - before;
                    break;
                }
                before += own[i];
            }
        }
#pragma unroll
        for (int i = 0; i < 4; i++) hist[CH_BINS - 1 - (tid * 4 + i)] = 0;
        __syncthreads();
        prefix |= (uint32_t)found[0] << shift;
        left = found[1];
    }
    // `left` of the words equal to `prefix` stay, the first ones. A row's place: those above before it, the equal ones before it
    // up to `left`, and the rows that stay anyway.
    const int run = (n + CH_THREADS - 1) / CH_THREADS * 32, r_begin = warp * run, r_end = min(n, r_begin + run);
    auto kind = [&](int r, bool& sure, bool& equal) {
        sure = equal = false;
        if (r >= r_end) return;
        if (r < lo || r >= hi) {
            sure = true;
        } else if (need > 0) {
            const uint32_t w = word(r);
            sure = w > prefix;
            equal = w == prefix;
        }
    };
    int n_sure = 0, n_equal = 0;
    for (int r0 = r_begin; r0 < r_end; r0 += 32) {
        bool sure, equal;
        kind(r0 + lane, sure, equal);
        n_sure += __popc(__ballot_sync(0xffffffffu, sure));
        n_equal += __popc(__ballot_sync(0xffffffffu, equal));
    }
    __syncthreads();                                       // (warp_s is read above)
    if (lane == 0) {
        warp_s[warp] = n_sure;
        equal_s[warp] = n_equal;
    }
    __syncthreads();
    int sure0 = 0, equal0 = 0;
    for (int i = 0; i < warp; i++) {
        sure0 += warp_s[i];
        equal0 += equal_s[i];
    }
    for (int r0 = r_begin; r0 < r_end; r0 += 32) {
        bool sure, equal;
        kind(r0 + lane, sure, equal);
        const unsigned bs = __ballot_sync(0xffffffffu, sure), be = __ballot_sync(0xffffffffu, equal), under = (1u << lane) - 1u;
        const int eb = equal0 + __popc(be & under);
        if (sure || (equal && eb < left)) out[sure0 + __popc(bs & under) + min(eb, left)] = r0 + lane;
        sure0 += __popc(bs);
        equal0 += __popc(be);
    }
    if (bad) atomicOr(status, MYNAH_ST_PAGE_RANGE);
}

// -------------------------------------------------------------------- moving

constexpr int MV_THREADS = 256, MV_UNROLL = 4;
constexpr int MV_BATCH = 512;                             // rows whose places are worked out together

struct MoveArgs {
    int B, KV, n_pages, keep;
    int same;                         // 1: the rows go to lower rows of the same pages
    int k_pieces, v_pieces;           // 16-byte pieces a row
    int k_slices, v_slices;           // slices of up to LANES pieces, each a CTA's
};

// Rows kept[i] -> i of one (layer, sequence, kv head), one slice of up to LANES * 16 bytes of every row of K or of V, or the sums.
// i <= kept[i], ascending. In the same pages a row is read before it is written over: a step's rows are all in registers, the
// next step's already asked for, when the barrier lets the step's writes go; and a row that is written in a step is a source of
// that step or of an earlier one. Places are worked out 512 rows ahead, so that the copies wait for one read, not for the
// choice, the page list and the row one behind the other. LANES: 16 (whole rows of 256 bytes: 28 layers of 2 sequences, 2,048 rows
// of 8 heads of 128, 160 us of both launches' 191, against 329 with 4), or 4 where that would leave too few CTAs (one layer of one
// sequence, 512 rows of 700: both launches 12.3 against 14.4 us).
template <int LANES>
__global__ void __launch_bounds__(MV_THREADS)
evict_move_kernel(uint4* __restrict__ k, uint4* __restrict__ v, float* __restrict__ mass, PageTable from, PageTable to,
                  const int* __restrict__ kv_len, const int* __restrict__ kept, MoveArgs a, int* __restrict__ status) {
    constexpr int EACH_ROW = MV_THREADS / LANES, MV_ROWS = EACH_ROW * MV_UNROLL;       // rows at once, rows a step
    static_assert(MV_BATCH % MV_ROWS == 0, "a batch is whole steps");
    __shared__ int src_s[2][MV_BATCH], dst_s[2][MV_BATCH];         // rows of the layer's storage, -1: none
    const int unit = blockIdx.x, g = unit % a.KV, b = unit / a.KV % a.B, e = unit / a.KV / a.B;
    const int held = max(0, kv_len[b]);
    const int n = min(held, a.keep);
    if (n == 0 || (a.same && held <= a.keep)) return;      // nothing moves
    const int* src = kept + (size_t)unit * a.keep;
    const size_t row0 = (size_t)e * a.n_pages * a.KV * PAGE_TOKENS;        // the layer's first row
    bool bad = false;
    // a row of the layer's storage, or -1 (the launch is refused where these do not fit 31 bits)
    auto row_of = [&](const PageTable& pt, int r) {
        const int page = page_of(pt, b, r);
        if (page < 0) {
            bad = true;
            return -1;
        }
        return (page * a.KV + g) * PAGE_TOKENS + r % PAGE_TOKENS;
    };
    auto places = [&](int i0, int buf) {
#pragma unroll
        for (int j = 0; j < MV_BATCH / MV_THREADS; j++) {
            const int i = i0 + j * MV_THREADS + threadIdx.x;
            src_s[buf][j * MV_THREADS + threadIdx.x] = i < n ? row_of(from, src[i]) : -1;
            dst_s[buf][j * MV_THREADS + threadIdx.x] = i < n ? row_of(to, i) : -1;
        }
    };
    const int sl = blockIdx.y;
    if (sl == a.k_slices + a.v_slices) {                   // the sums, a row a thread
        float* t = mass + row0;
        constexpr int EACH = MV_BATCH / MV_THREADS;
        places(0, 0);
        for (int i0 = 0, buf = 0; i0 < n; i0 += MV_BATCH, buf ^= 1) {
            float x[EACH];
#pragma unroll
            for (int j = 0; j < EACH; j++) {               // (a thread reads the places that it wrote itself)
                const int s = src_s[buf][j * MV_THREADS + threadIdx.x];
                x[j] = s >= 0 ? t[s] : 0.f;
            }
            places(i0 + MV_BATCH, buf ^ 1);
            __syncthreads();
#pragma unroll
            for (int j = 0; j < EACH; j++) {
                const int d = dst_s[buf][j * MV_THREADS + threadIdx.x];
                if (d >= 0 && src_s[buf][j * MV_THREADS + threadIdx.x] >= 0) t[d] = x[j];
            }
        }
    } else {
        const bool is_k = sl < a.k_slices;
        const int pieces = is_k ? a.k_pieces : a.v_pieces, at = (is_k ? sl : sl - a.k_slices) * LANES + threadIdx.x % LANES;
        uint4* t = (is_k ? k : v) + row0 * pieces + at;
        const bool on = at < pieces;
        const int row = threadIdx.x / LANES;
        uint4 x[MV_UNROLL], y[MV_UNROLL];
        auto load = [&](int i0, uint4 (&w)[MV_UNROLL]) {   // the step from row i0 on
            const int* s = src_s[(i0 / MV_BATCH) & 1] + i0 % MV_BATCH;
#pragma unroll
            for (int j = 0; j < MV_UNROLL; j++) {
                const int r = s[j * EACH_ROW + row];
                if (r >= 0 && on) w[j] = t[(size_t)r * pieces];
            }
        };
        places(0, 0);
        __syncthreads();
        load(0, x);
        for (int i0 = 0; i0 < n; i0 += MV_ROWS) {
            // the next step's rows; in a batch's last step its successor's places first
            if (i0 % MV_BATCH == MV_BATCH - MV_ROWS) {
                places(i0 + MV_ROWS, ((i0 + MV_ROWS) / MV_BATCH) & 1);
                __syncthreads();
            }
            if (i0 + MV_ROWS < n) load(i0 + MV_ROWS, y);
            __syncthreads();
            const int* d = dst_s[(i0 / MV_BATCH) & 1] + i0 % MV_BATCH;
            const int* s = src_s[(i0 / MV_BATCH) & 1] + i0 % MV_BATCH;
#pragma unroll
            for (int j = 0; j < MV_UNROLL; j++) {
                const int q = j * EACH_ROW + row, r = d[q];
                if (r >= 0 && s[q] >= 0 && on) t[(size_t)r * pieces] = x[j];
                x[j] = y[j];
            }
        }
    }
    if (bad) atomicOr(status, MYNAH_ST_PAGE_RANGE);
}

// ---------------------------------------------------------------- acceptance

constexpr int CM_THREADS = 256, CM_UNROLL = 8;

struct CommitArgs {
    int E, B, T, KV, n_pages, max_q;
    int k_pieces, v_pieces;
};

// The accepted path of one sequence's tree, found by every CTA that moves rows of the sequence, then the moves: row past +
// path[i] -> past + i, a warp a (layer, kv head). A row's child that goes on is its lowest one whose token is what was chosen
// behind the row; the walk from row 0 over such children is one thread's, its steps are reads of shared memory.
__global__ void __launch_bounds__(CM_THREADS)
tree_commit_kernel(const int* __restrict__ tokens, const int* __restrict__ parents, const int* __restrict__ chosen,
                   const int* __restrict__ cu_q, const int* __restrict__ kv_len, PageTable pt, uint4* __restrict__ k, uint4* __restrict__ v,
                   int* __restrict__ path, int* __restrict__ count, int* __restrict__ next, CommitArgs a, int* __restrict__ status) {
    extern __shared__ int tree_s[];
    int* child = tree_s;                                   // [max_q] the child that goes on
    int* walk = tree_s + a.max_q;                          // [max_q]
    __shared__ int len_s;
    const int b = blockIdx.y, q0 = cu_q[b], end = cu_q[b + 1], n = end - q0, held = kv_len[b];
    if (n <= 0 || q0 < 0 || end > a.T || n > a.max_q || held < n) {
        if (blockIdx.x == 0 && threadIdx.x == 0) {
            count[b] = 0;
            next[b] = -1;
            if (n != 0) atomicOr(status, MYNAH_ST_PAGE_RANGE);
        }
        return;
    }
    for (int c = threadIdx.x; c < n; c += CM_THREADS) child[c] = n;
    __syncthreads();
    for (int c = 1 + (int)threadIdx.x; c < n; c += CM_THREADS) {
        const int p = parents[q0 + c];
        if (p >= 0 && p < c && tokens[q0 + c] == chosen[q0 + p]) atomicMin(&child[p], c);
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        int len = 1, at = 0;
        walk[0] = 0;
        while ((at = child[at]) < n) walk[len++] = at;     // (a row has one parent, before it: no row comes twice)
        len_s = len;
    }
    __syncthreads();
    const int len = len_s, past = held - n;
    if (blockIdx.x == 0) {
        for (int i = threadIdx.x; i < n; i += CM_THREADS) path[q0 + i] = i < len ? walk[i] : -1;
        if (threadIdx.x == 0) {
            count[b] = len;
            next[b] = chosen[q0 + walk[len - 1]];
        }
    }
    const int lane = threadIdx.x & 31, warps = CM_THREADS / 32 * gridDim.x;
    for (int unit = blockIdx.x * (CM_THREADS / 32) + (threadIdx.x >> 5); unit < a.E * a.KV; unit += warps) {
        const int e = unit / a.KV, g = unit % a.KV;
        const size_t page0 = (size_t)e * a.n_pages * a.KV + g;
        for (int kv = 0; kv < 2; kv++) {
            uint4* t = kv ? v : k;
            const int pieces = kv ? a.v_pieces : a.k_pieces, total = len * pieces;
            // pieces of the path's rows in order: those of a batch are in registers before any of it is written, and what a
            // batch writes is a source of no later batch (path[i] >= i, ascending)
            for (int i0 = pieces; i0 < total; i0 += 32 * CM_UNROLL) {      // (row 0 of the path is row 0)
                uint4 x[CM_UNROLL];
                long long d[CM_UNROLL];
#pragma unroll
                for (int j = 0; j < CM_UNROLL; j++) {
                    const int i = i0 + j * 32 + lane;
                    d[j] = -1;
                    if (i >= total) continue;
                    const int r = i / pieces, c = i % pieces, w = walk[r];
                    if (w == r) continue;
                    const int ps = page_of(pt, b, past + w), pd = page_of(pt, b, past + r);
                    if (ps < 0 || pd < 0) {
                        atomicOr(status, MYNAH_ST_PAGE_RANGE);
                        continue;
                    }
                    d[j] = ((long long)(page0 + (size_t)pd * a.KV) * PAGE_TOKENS + (past + r) % PAGE_TOKENS) * pieces + c;
                    x[j] = t[((long long)(page0 + (size_t)ps * a.KV) * PAGE_TOKENS + (past + w) % PAGE_TOKENS) * pieces + c];
                }
                __syncwarp();
#pragma unroll
                for (int j = 0; j < CM_UNROLL; j++)
                    if (d[j] >= 0) t[d[j]] = x[j];
                __syncwarp();
            }
        }
    }
}

bool row_ok(int bytes) { return bytes > 0 && bytes % 16 == 0; }

}  // namespace

// k [E, n_pages, KV, 64, k_bytes], v likewise, mass [E, n_pages, KV, 64]; kept [E, B, KV, keep], new_len [B]. `same`: the out
// page lists are the page lists. n_ids: entries of page_ids.
struct CacheEvictCall {
    void *k, *v;
    float* mass;
    int E, B, KV, n_pages, k_bytes, v_bytes;
    const int *kv_len, *page_indptr, *page_ids, *page_base;
    int n_ids;
    const int *out_indptr, *out_ids, *out_base;
    int same, keep, recent, first;
    int *kept, *new_len, *status;
    cudaStream_t stream;
};
static_assert(sizeof(CacheEvictCall) == 160, "as packed by the caller");
MYNAH_API int mynah_cache_evict(const CacheEvictCall* call) {
    const auto& [k, v, mass, E, B, KV, n_pages, k_bytes, v_bytes, kv_len, page_indptr, page_ids, page_base, n_ids, out_indptr, out_ids, out_base,
                 same, keep, recent, first, kept, new_len, status, stream] = *call;
    if (E <= 0 || B <= 0) return 0;
    MYNAH_REQUIRE(KV > 0 && n_pages >= 0, "cache_evict: %d kv heads, %d pages", KV, n_pages);
    MYNAH_REQUIRE(row_ok(k_bytes) && row_ok(v_bytes), "cache_evict: rows of %d and %d bytes are not whole 16-byte pieces", k_bytes, v_bytes);
    MYNAH_REQUIRE(((uintptr_t)k & 15) == 0 && ((uintptr_t)v & 15) == 0, "cache_evict: the cache must be 16-byte aligned");
    MYNAH_REQUIRE(keep > 0 && recent >= 0 && first >= 0 && (long long)recent + first <= keep, "cache_evict: keep %d, recent %d and first %d do not go together", keep, recent, first);
    MYNAH_REQUIRE((long long)E * B * KV < (1ll << 31) && (long long)n_pages * KV * PAGE_TOKENS < (1ll << 31), "cache_evict: launch too large");
    MYNAH_REQUIRE(status != nullptr && kept != nullptr && new_len != nullptr && mass != nullptr, "cache_evict: outputs, sums and a status word are required");
    const PageTable from{page_indptr, page_ids, page_base, n_pages}, to{out_indptr, out_ids, out_base, n_pages};
    // Words of up to 96 KB a CTA are kept in shared memory; longer rows are read again from L2. The host knows the entries of all page lists
    // together, not the longest sequence's: many sequences get more than they use, and fewer CTAs an SM for it.
    const long long most = (long long)n_ids * PAGE_TOKENS;
    const int cached = (int)(most < 24576 ? most : 24576);
    const EvictArgs ea{E, B, KV, n_pages, keep, recent, first, cached};
    static std::atomic<unsigned long long> opted{0};
    const cudaError_t err = shared_memory_once(evict_choose_kernel, 24576 * 4, opted);
    if (err != cudaSuccess) return mynah_fail("cache_evict: %s", cudaGetErrorString(err));
    evict_choose_kernel<<<(unsigned)(E * B * KV), CH_THREADS, (size_t)cached * 4, stream>>>(mass, from, kv_len, ea, kept, new_len, status);
    if (mynah_check_launch("evict_choose")) return -1;
    const int kp = k_bytes / 16, vp = v_bytes / 16;
    const int lanes = (long long)E * B * KV * (ceil_div(kp, 16) + ceil_div(vp, 16)) >= 2ll * mynah_sm_count() ? 16 : 4;
    const MoveArgs ma{B, KV, n_pages, keep, same, kp, vp, ceil_div(kp, lanes), ceil_div(vp, lanes)};
    const dim3 grid((unsigned)(E * B * KV), ma.k_slices + ma.v_slices + 1);
    if (lanes == 16) evict_move_kernel<16><<<grid, MV_THREADS, 0, stream>>>((uint4*)k, (uint4*)v, mass, from, to, kv_len, kept, ma, status);
    else evict_move_kernel<4><<<grid, MV_THREADS, 0, stream>>>((uint4*)k, (uint4*)v, mass, from, to, kv_len, kept, ma, status);
    return mynah_check_launch("evict_move");
}

// tokens, parents, chosen [T]; k [E, n_pages, KV, 64, k_bytes], v likewise. path [T] (-1 behind a path's end), count [B], next [B].
struct TreeCommitCall {
    const int *tokens, *parents, *chosen;
    int T, B, max_q_len;
    const int *cu_q, *kv_len, *page_indptr, *page_ids, *page_base;
    int n_pages;
    void *k, *v;
    int E, KV, k_bytes, v_bytes;
    int *path, *count, *next, *status;
    cudaStream_t stream;
};
static_assert(sizeof(TreeCommitCall) == 160, "as packed by the caller");
MYNAH_API int mynah_tree_commit(const TreeCommitCall* call) {
    const auto& [tokens, parents, chosen, T, B, max_q_len, cu_q, kv_len, page_indptr, page_ids, page_base, n_pages, k, v, E, KV, k_bytes, v_bytes,
                 path, count, next, status, stream] = *call;
    if (B <= 0) return 0;
    MYNAH_REQUIRE(E >= 0 && KV > 0, "tree_commit: %d layers, %d kv heads", E, KV);
    MYNAH_REQUIRE(row_ok(k_bytes) && row_ok(v_bytes), "tree_commit: rows of %d and %d bytes are not whole 16-byte pieces", k_bytes, v_bytes);
    MYNAH_REQUIRE(((uintptr_t)k & 15) == 0 && ((uintptr_t)v & 15) == 0, "tree_commit: the cache must be 16-byte aligned");
    MYNAH_REQUIRE(max_q_len >= 0 && max_q_len <= 4096 && B <= 65535, "tree_commit: %d sequences of up to %d rows are too many", B, max_q_len);
    MYNAH_REQUIRE(status != nullptr, "tree_commit: a status word is required");
    const CommitArgs a{E, B, T, KV, n_pages, max_q_len, k_bytes / 16, v_bytes / 16};
    int x = ceil_div(E * KV, CM_THREADS / 32);
    const int most = ceil_div(4 * mynah_sm_count(), B);
    x = x < 1 ? 1 : (x > most ? most : x);
    tree_commit_kernel<<<dim3(x, B), CM_THREADS, 2 * (size_t)(max_q_len > 0 ? max_q_len : 1) * sizeof(int), stream>>>(
        tokens, parents, chosen, cu_q, kv_len, PageTable{page_indptr, page_ids, page_base, n_pages}, (uint4*)k, (uint4*)v, path, count, next, a, status);
    return mynah_check_launch("tree_commit");
}
