// Attention of a few rows a sequence over the paged cache, with any mask among the step's own rows: the tokens of a drafted
// tree (every token sees what was held before the step and its ancestors), or causal rows.
//
//   visible(i, r) = r < past, or bit (r - past) of token i's mask words (causal: r <= past + i), and r < kv_len
//   s_ihr = scale * q_ih . k_gr,   w = softmax over the visible r,   out_ih = sum_r w_ihr v_gr      (g = h / (H / KV))
//
// with past = kv_len - n_q. A token that sees nothing gives zeros. The query heads of a kv head are rows of one problem, so a
// page is read once for all of them; the keys are shared out among the CTAs, each with its own running maximum and sum, and a
// second launch joins what was cut (row_units.cuh has the rules).
//
// This file holds the general kernel (fp32, and bfloat16 heads that the tensor-core kernel does not take), the joining, and
// the entry points.
#include "attn_rows.cuh"

#include <limits.h>
#include <math.h>

namespace {

constexpr int KT = 32;               // keys a tile of the general kernel
constexpr int MAX_HEAD = 256;
constexpr size_t MOST_SHARED = 226 * 1024;        // (heads of 256 and 64 rows in fp32 take 209 KB)

__device__ __forceinline__ float max_or_nan(float a, float b) {
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}

__device__ __forceinline__ void copy16_async(void* dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// Row pitch of a staged K or V tile: 16 bytes of padding, so that eight lanes' 16-byte reads of eight rows meet no bank twice.
template <typename T> __host__ __device__ constexpr int pitch_of(int HD) { return HD + 16 / (int)sizeof(T); }

// TY x TX threads; thread (ty, tx) has the packed rows ty + TY * i (i < 4) of the tile, for the scores the keys tx + TX * j of
// KT, for the output the columns 4 * tx + 4 * TX * c. fp32 throughout, products and sums as written (FFMA). The row's maximum
// and sum are kept by every thread of the row. An unseen key has the weight 0; in a tile that holds unseen keys and a value
// that is not finite (a stale row, an infinity) it is stored as -1, and such keys are left out of the output by a select:
// what lies in an unseen row of V cannot reach a result, while a seen one does what arithmetic does (the select everywhere in
// masked tiles, and the queries read one by one: 30.5 us against 26.7 for 3 trees of 19 in fp32 behind 1,021 rows). K and V come KT
// keys at a time by asynchronous copies, two tiles in flight.
// 16-row tiles (TY = 4, TX = 32) are for the few rows of decode steps and small trees, 64-row tiles (TY = TX = 16) for the rest.
template <typename T, int TY, int TX, int NC, bool CAUSAL>
__global__ void __launch_bounds__(TY * TX, 2)
attn_rows_kernel(const T* __restrict__ q, T* __restrict__ out, const T* __restrict__ k_cache, const T* __restrict__ v_cache,
                 const int* __restrict__ cu_q, const int* __restrict__ kv_len, PageTable pt, const long long* __restrict__ masks,
                 RowsArgs a, RowsScratch sc, int* __restrict__ status) {
    constexpr int R = 4 * TY, KJ = KT / TX, THREADS = TY * TX;
    extern __shared__ __align__(16) unsigned char smem_rows[];
    const int HD = a.HD, kp = pitch_of<T>(HD), qp = HD + 4;
    float* q_s = reinterpret_cast<float*>(smem_rows);              // [R][qp]
    float* p_s = q_s + R * qp;                                     // [R][KT + 4]
    T* k_s = reinterpret_cast<T*>(p_s + R * (KT + 4));             // [2][KT][kp]
    T* v_s = k_s + 2 * KT * kp;                                    // [2][KT][kp]
    __shared__ RowWalk<CAUSAL, true> walk_s;

    if (threadIdx.x < 32) find_start(cu_q, kv_len, pt, a, &walk_s, sc.starts, status);
    __syncthreads();
    RowWalk<CAUSAL, true> u = walk_s;
    if (u.b < 0) return;
    const int ty = threadIdx.x / TX, tx = threadIdx.x % TX;
    // the 16-byte pieces of a K or V tile that this thread copies: the first one, and how far on the next is
    const int per_row = HD * (int)sizeof(T) / 16, copy_r = threadIdx.x / per_row, copy_c = threadIdx.x % per_row;
    const int rows_on = THREADS / per_row, pieces_on = THREADS % per_row;
    do {
    const int g = u.g, n_rows = u.rows(a), past = u.past(), row0 = u.tile * a.tile_rows;
    const int pg0 = u.pg0, pg1 = u.pg1;
    __syncthreads();                                               // (the segment before is done with shared memory)
    // every page of the segment must be there: one that lacks a page counts as keys that nobody sees
    bool lacks = false;
    for (int p = pg0 + (int)threadIdx.x; p < pg1; p += THREADS) lacks |= page_at(pt, u.s, p) < 0;
    // the tile's queries, four values a thread (one by one where rows are not aligned); rows that are not there are zero
    const int quads = HD >> 2;
#pragma unroll 4
    for (int i = threadIdx.x; i < R * quads; i += THREADS) {
        const int r = a.by_quads.div(i), d = (i - r * quads) * 4, pr = row0 + r, tok = a.by_G.div(pr);
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
        if (r < n_rows) {
            const T* at = q + (size_t)(u.s.q_begin + tok) * a.ldq + (size_t)(g * a.G + pr - tok * a.G) * HD + d;
            x = a.q_aligned ? four_of(at) : four_apart(at);
        }
        *reinterpret_cast<float4*>(q_s + r * qp + d) = x;
    }
    // The answer comes out of the barrier, the same for every thread: a flag in shared memory that the next segment clears could be
    // read behind that by a late warp, which would go on into the pages alone.
    const bool bad = __syncthreads_or(lacks);
    if (bad && threadIdx.x == 0) atomicOr(status, MYNAH_ST_PAGE_RANGE);

    const int first_tok = a.by_G.div(row0);
    const int t0 = bad ? 0 : pg0 * (PAGE_TOKENS / KT), t1 = bad ? 0 : min(pg1 * (PAGE_TOKENS / KT), (u.s.kvl + KT - 1) / KT);
    auto bring = [&](int t, int st) {
        const int page = page_at(pt, u.s, t / (PAGE_TOKENS / KT));
        const size_t base = (((size_t)page * a.KV + g) * PAGE_TOKENS + (t * KT) % PAGE_TOKENS) * HD;
#pragma unroll 2
        for (int r = copy_r, c = copy_c; r < KT;) {
            copy16_async(reinterpret_cast<unsigned char*>(k_s + (st * KT + r) * kp) + c * 16, reinterpret_cast<const unsigned char*>(k_cache + base + (size_t)r * HD) + c * 16);
            copy16_async(reinterpret_cast<unsigned char*>(v_s + (st * KT + r) * kp) + c * 16, reinterpret_cast<const unsigned char*>(v_cache + base + (size_t)r * HD) + c * 16);
            r += rows_on;
            if ((c += pieces_on) >= per_row) c -= per_row, r++;
        }
        copies_commit();
    };

    float m[4], l[4], acc[4][NC][4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        m[i] = -INFINITY;
        l[i] = 0.f;
#pragma unroll
        for (int c = 0; c < NC; c++)
#pragma unroll
            for (int e = 0; e < 4; e++) acc[i][c][e] = 0.f;
    }
    if (t0 < t1) bring(t0, 0);
    for (int t = t0; t < t1; t++) {
        const int st = (t - t0) & 1;
        if (t + 1 < t1) {
            bring(t + 1, st ^ 1);
            copies_wait<1>();
        } else {
            copies_wait<0>();
        }
        const T* ks = k_s + st * KT * kp;
        const T* vs = v_s + st * KT * kp;
        const int key0 = t * KT;
        // is there a key in the tile that some row of the tile must not see?
        const bool need_mask = key0 + KT > u.s.kvl || (CAUSAL ? key0 + KT - 1 > past + first_tok : key0 + KT > past);
        __syncthreads();
        bool odd = false;                                          // and then a value that is not finite (or a stale row)?
        if (need_mask) {
            for (int i = threadIdx.x; i < KT * quads; i += THREADS) {
                const int r = a.by_quads.div(i);
                const float4 x = four_of(vs + r * kp + (i - r * quads) * 4);
                odd |= !(fabsf(x.x) <= 3e38f && fabsf(x.y) <= 3e38f && fabsf(x.z) <= 3e38f && fabsf(x.w) <= 3e38f);
            }
            odd = __syncthreads_or(odd);
        }
        float s[4][KJ];
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int j = 0; j < KJ; j++) s[i][j] = 0.f;
#pragma unroll 4
        for (int d = 0; d < HD; d += 4) {
            float4 qv[4], kv[KJ];
#pragma unroll
            for (int i = 0; i < 4; i++) qv[i] = four_of(q_s + (ty + TY * i) * qp + d);
#pragma unroll
            for (int j = 0; j < KJ; j++) kv[j] = four_of(ks + (tx + TX * j) * kp + d);
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int j = 0; j < KJ; j++) {
                    s[i][j] = fmaf(qv[i].x, kv[j].x, s[i][j]);
                    s[i][j] = fmaf(qv[i].y, kv[j].y, s[i][j]);
                    s[i][j] = fmaf(qv[i].z, kv[j].z, s[i][j]);
                    s[i][j] = fmaf(qv[i].w, kv[j].w, s[i][j]);
                }
        }
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int r = ty + TY * i, pr = row0 + r, tok = a.by_G.div(pr);
            uint32_t seen = 0xffffffffu;
            if (need_mask) {
                const unsigned long long vis = r < n_rows ? visible64<CAUSAL>(key0 & ~63, u.s.kvl, past, tok, masks + (size_t)(u.s.q_begin + tok) * a.words, a.words) : 0ull;
                seen = (uint32_t)(vis >> (key0 & 63));
            }
            float mx = -INFINITY;
#pragma unroll
            for (int j = 0; j < KJ; j++) {
                s[i][j] = (seen >> (tx + TX * j)) & 1u ? s[i][j] * a.scale_log2 : -INFINITY;
                mx = fmaxf(mx, s[i][j]);
            }
#pragma unroll
            for (int o = TX / 2; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
            const float m_new = fmaxf(m[i], mx);
            const float m_use = m_new == -INFINITY ? 0.f : m_new;
            const float alpha = exp2f(m[i] - m_use);               // 0 before the first seen key
            m[i] = m_new;
            float sum = 0.f;
#pragma unroll
            for (int j = 0; j < KJ; j++) {
                const bool in = (seen >> (tx + TX * j)) & 1u;
                const float p = exp2f(s[i][j] - m_use);
                if (in) sum += p;
                p_s[r * (KT + 4) + tx + TX * j] = in ? p : odd ? -1.f : 0.f;
            }
#pragma unroll
            for (int o = TX / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            l[i] = l[i] * alpha + sum;
#pragma unroll
            for (int c = 0; c < NC; c++)
#pragma unroll
                for (int e = 0; e < 4; e++) acc[i][c][e] *= alpha;
        }
        __syncwarp();                                              // a row's weights are written and read within one warp
#pragma unroll 2
        for (int kk = 0; kk < KT; kk += 4) {
            float p[4][4];
#pragma unroll
            for (int i = 0; i < 4; i++) *reinterpret_cast<float4*>(p[i]) = *reinterpret_cast<const float4*>(p_s + (ty + TY * i) * (KT + 4) + kk);
#pragma unroll
            for (int e4 = 0; e4 < 4; e4++) {
#pragma unroll
                for (int c = 0; c < NC; c++) {
                    const int col = 4 * tx + 4 * TX * c;
                    if (col >= HD) continue;
                    const float4 x = four_of(vs + (kk + e4) * kp + col);
                    if (odd) {
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            const float w = p[i][e4];
                            acc[i][c][0] = w < 0.f ? acc[i][c][0] : fmaf(w, x.x, acc[i][c][0]);
                            acc[i][c][1] = w < 0.f ? acc[i][c][1] : fmaf(w, x.y, acc[i][c][1]);
                            acc[i][c][2] = w < 0.f ? acc[i][c][2] : fmaf(w, x.z, acc[i][c][2]);
                            acc[i][c][3] = w < 0.f ? acc[i][c][3] : fmaf(w, x.w, acc[i][c][3]);
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            acc[i][c][0] = fmaf(p[i][e4], x.x, acc[i][c][0]);
                            acc[i][c][1] = fmaf(p[i][e4], x.y, acc[i][c][1]);
                            acc[i][c][2] = fmaf(p[i][e4], x.z, acc[i][c][2]);
                            acc[i][c][3] = fmaf(p[i][e4], x.w, acc[i][c][3]);
                        }
                    }
                }
            }
        }
        __syncthreads();                                           // the stage and the weights are free again
    }

    const bool whole = u.whole();
    const long long to = whole ? 0 : u.scratch_row(a);
    // (lists that hold more pages than the call said would take more scratch than there is)
    const bool fits = whole || to + n_rows <= a.cut_rows;
    if (!fits && threadIdx.x == 0) atomicOr(status, MYNAH_ST_PAGE_RANGE);
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int r = ty + TY * i;
        if (r >= n_rows) continue;
        const int pr = row0 + r, tok = a.by_G.div(pr), h = g * a.G + pr - tok * a.G;
        if (whole) {
            const float inv = l[i] > 0.f ? 1.f / l[i] : (l[i] == 0.f ? 0.f : l[i]);    // a NaN stays one
            T* o = out + (size_t)(u.s.q_begin + tok) * a.ldo + (size_t)h * HD;
#pragma unroll
            for (int c = 0; c < NC; c++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int col = 4 * tx + 4 * TX * c + e;
                    if (col < HD) o[col] = from_f32<T>(acc[i][c][e] * inv);
                }
            if (CAUSAL && tx == 0) sc.lse[((size_t)g * a.T + u.s.q_begin) * a.G + pr] = l[i] == 0.f ? -INFINITY : m[i] + log2f(l[i]);
        } else if (fits) {
            float* o = sc.o + (to + r) * HD;
#pragma unroll
            for (int c = 0; c < NC; c++) {
                const int col = 4 * tx + 4 * TX * c;
                if (col < HD) *reinterpret_cast<float4*>(o + col) = make_float4(acc[i][c][0], acc[i][c][1], acc[i][c][2], acc[i][c][3]);
            }
            if (tx == 0) sc.ml[to + r] = make_float2(m[i], l[i]);
        }
    }
    } while (u.next(cu_q, kv_len, pt, a, status));
    griddep_launch_late();
}

// Four values of a row. Whether rows are aligned is the host's to say, and each way is an instance of its own: in one that looked at the
// address and had both, a row in fp32 that was not aligned met a 16-byte store.
template <bool ALIGNED> __device__ __forceinline__ void store4(float* o, float a, float b, float c, float d) {
    if (ALIGNED) *reinterpret_cast<float4*>(o) = make_float4(a, b, c, d);
    else o[0] = a, o[1] = b, o[2] = c, o[3] = d;
}
template <bool ALIGNED> __device__ __forceinline__ void store4(bf16* o, float a, float b, float c, float d) {
    if (ALIGNED) {
        const __nv_bfloat162 x = __floats2bfloat162_rn(a, b), y = __floats2bfloat162_rn(c, d);
        *reinterpret_cast<uint2*>(o) = make_uint2(*reinterpret_cast<const uint32_t*>(&x), *reinterpret_cast<const uint32_t*>(&y));
    } else {
        o[0] = from_f32<bf16>(a), o[1] = from_f32<bf16>(b), o[2] = from_f32<bf16>(c), o[3] = from_f32<bf16>(d);
    }
}

// Joins the segments of a cut item, running over them with the maximum so far as the softmax does over keys. CTA c's helpers
// (blockIdx.x = c - 1) take the item that CTA c begins inside of, if the item's first pages are CTA c - 1's (each cut item has one
// such CTA). OWN: a CTA for every tile and kv head that the step's rows can make, which leaves where the tile was not cut. A warp
// a row. Bound by its start behind the attention and three dependent reads (where the CTA begins or which tile it
// has, the sequence's numbers, then the segments' maxima and rows together, from L2).
constexpr int JOIN_WARPS = 8, JOIN_HELPERS = 16;                   // warps of a CTA; CTAs that share an item's rows at most
constexpr int JOIN_AHEAD = 4;                                      // segments asked for at once

// Sums of the weights from the scores that the attention has kept (steps of up to 8 rows a kv head, so one tile and one item a
// sequence and kv head): CTA number `cta` of those that add, for one sequence and kv head a run of its pages, a thread a key. The
// rows' log-sums come from the segments' maxima and sums, as the joining CTAs have them, so neither waits for the other and no
// launch is needed for it (one of its own behind the join: one token of 16 heads behind 1,535 rows 18.5 us, so 16.4; 64 tokens
// behind up to 4,000 rows 172 both). Bound by the scores' and the sums' bytes.
constexpr int SUM_PAGES = JOIN_WARPS * 32 / PAGE_TOKENS;           // at once
__device__ __forceinline__ void sum_scores(int cta, const int* __restrict__ cu_q, const int* __restrict__ kv_len, const PageTable& pt, const RowsArgs& a,
                                           const RowsScratch& sc, int* status) {
    __shared__ RowStart cut_s;                                     // b: the CTA that begins inside the item first, or -1
    __shared__ float lse_s[JOIN_WARPS];
    const int chunk = cta % sc.sum_chunks, bg = cta / sc.sum_chunks, g = a.by_KV.mod(bg), b = a.by_KV.div(bg);
    if (threadIdx.x == 0) cut_s.b = -1;
    const SeqShape s = seq_shape(cu_q, kv_len, pt, b, a, status);
    __syncthreads();
    if (s.n_q == 0) return;
    if (!a.whole_items) {
        for (int c = threadIdx.x; c < a.ctas; c += JOIN_WARPS * 32) {
            const RowStart at = sc.starts[c];
            if (at.b == b && at.g == g && at.from > 0 && at.from <= at.each) {
                cut_s.from = at.from;
                cut_s.each = at.each;
                cut_s.b = c;
            }
        }
    }
    __syncthreads();
    const int row = threadIdx.x >> 5, lane = threadIdx.x & 31, rows = min(s.n_q * a.G, sc.score_rows), past = s.kvl - s.n_q;
    if (row < rows) {
        float lse;
        if (cut_s.b < 0 || s.pages <= cut_s.from) {                // one CTA had it whole
            lse = sc.lse[((size_t)g * a.T + s.q_begin) * a.G + row];
        } else {
            const int n = 2 + quotient(s.pages - cut_s.from - 1, cut_s.each);
            float m = -INFINITY, l = 0.f;
            for (int c = lane; c < n; c += 32) {
                const float2 ml = sc.ml[((long long)(cut_s.b - 1 + c) * 2 + (c == 0 ? 1 : 0)) * a.tile_rows + row];
                const float m_new = max_or_nan(m, ml.x), m_use = m_new == -INFINITY ? 0.f : m_new;
                l = fmaf(l, ex2_f(m - m_use), ml.y * ex2_f(ml.x - m_use));
                m = m_new;
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) {
                const float m2 = __shfl_xor_sync(0xffffffffu, m, o), l2 = __shfl_xor_sync(0xffffffffu, l, o);
                const float m_new = max_or_nan(m, m2), m_use = m_new == -INFINITY ? 0.f : m_new;
                l = fmaf(l, ex2_f(m - m_use), l2 * ex2_f(m2 - m_use));
                m = m_new;
            }
            lse = l == 0.f ? -INFINITY : m + log2f(l);
        }
        if (lane == 0) lse_s[row] = lse;
    }
    __syncthreads();
    const int e = threadIdx.x % PAGE_TOKENS;
    for (int lp = chunk * SUM_PAGES + threadIdx.x / PAGE_TOKENS; lp < s.pages; lp += sc.sum_chunks * SUM_PAGES) {
        const int key = lp * PAGE_TOKENS + e, page = page_at(pt, s, lp), entry = s.list0 + lp - s.first;
        if (page < 0 || key >= s.kvl || entry >= sc.entries) continue;         // (the attention has reported a missing page)
        const float* z = sc.scores + ((size_t)entry * a.KV + g) * sc.score_rows * PAGE_TOKENS + e;
        float* m = sc.mass + ((size_t)page * a.KV + g) * PAGE_TOKENS + e;
        float sum = key < past ? *m : 0.f;
#pragma unroll 4
        for (int r = 0; r < rows; r++) sum += lse_s[r] == -INFINITY ? 0.f : ex2_f(z[r * PAGE_TOKENS] - lse_s[r]);
        *m = sum;
    }
}

// CTAs from `joining` on: sums of kept scores.
template <typename T, bool OWN, bool ALIGNED>
__global__ void __launch_bounds__(JOIN_WARPS * 32)
attn_rows_join_kernel(T* __restrict__ out, const int* __restrict__ cu_q, const int* __restrict__ kv_len, PageTable pt, RowsArgs a, RowsScratch sc,
                      int joining, int* __restrict__ status) {
    griddep_wait();
    SeqShape s;
    int g, tile, n;                                                // n: segments
    long long first, next, after;                                  // scratch rows of the tile's first row in its first, its second segment, and from one to the next
    if (OWN) {
        g = a.by_KV.mod(blockIdx.x);
        const int b = find_tile(cu_q, kv_len, pt, a, a.by_KV.div(blockIdx.x), tile, first, status);
        if (b < 0) return;
        s = seq_shape(cu_q, kv_len, pt, b, a, status);
        const OwnCut cut = own_cut(s, a);
        if (cut.n == 1) return;                                    // (it was whole)
        n = quotient((a.causal ? tile_pages<true>(s, tile, a) : s.pages) + cut.each - 1, cut.each);
        after = s.n_q * a.G;
        first += (long long)(g * cut.n) * after + tile * a.tile_rows;
        next = first + after;
        if (n == 1 || first + (n - 1) * after + min(a.tile_rows, s.n_q * a.G - tile * a.tile_rows) > a.cut_rows) return;
    } else {
        if ((int)blockIdx.x >= joining) {
            sum_scores(blockIdx.x - joining, cu_q, kv_len, pt, a, sc, status);
            return;
        }
        const int cta = a.by_group.div(blockIdx.x) + 1, sub = a.by_group.mod(blockIdx.x);   // (CTA 0 begins inside of nothing)
        const RowStart at = sc.starts[cta];
        if (at.b < 0 || at.from == 0 || at.from > at.each) return;
        s = seq_shape(cu_q, kv_len, pt, at.b, a, status);
        g = at.g;
        tile = at.item * a.group + sub;
        if (tile >= s.tiles) return;
        const int pages = a.causal ? tile_pages<true>(s, tile, a) : s.pages;
        if (pages <= at.from) return;                              // this tile ends before the cut: it was whole
        n = 2 + quotient(pages - at.from - 1, at.each);
        after = 2ll * a.group * a.tile_rows;
        next = 2ll * (cta * a.group + sub) * a.tile_rows;
        first = next - after + a.tile_rows;                        // (its CTA's second place)
    }
    const int lane = threadIdx.x & 31, rows = min(a.tile_rows, s.n_q * a.G - tile * a.tile_rows);
#pragma unroll 1
    for (int row = blockIdx.y * JOIN_WARPS + (threadIdx.x >> 5); row < rows; row += gridDim.y * JOIN_WARPS) {
        const int pr = tile * a.tile_rows + row, tok = a.by_G.div(pr), t = s.q_begin + tok, h = g * a.G + pr - tok * a.G;
        for (int col = lane * 4; col < a.HD; col += 128) {
            float m = -INFINITY, l = 0.f;
            float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
            for (int c0 = 0; c0 < n; c0 += JOIN_AHEAD) {
                float2 ml[JOIN_AHEAD];
                float4 y[JOIN_AHEAD];
#pragma unroll
                for (int c = 0; c < JOIN_AHEAD; c++) {
                    ml[c] = make_float2(-INFINITY, 0.f);           // (behind the last: no weight)
                    y[c] = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (c0 + c < n) {
                        const long long i = (c0 + c == 0 ? first : next + (c0 + c - 1) * after) + row;
                        ml[c] = sc.ml[i];
                        y[c] = *reinterpret_cast<const float4*>(sc.o + i * a.HD + col);
                    }
                }
#pragma unroll
                for (int c = 0; c < JOIN_AHEAD; c++) {
                    const float m_new = max_or_nan(m, ml[c].x), m_use = m_new == -INFINITY ? 0.f : m_new;
                    const float u = ex2_f(m - m_use), w = ex2_f(ml[c].x - m_use);
                    m = m_new;
                    l = fmaf(l, u, ml[c].y * w);
                    x.x = fmaf(x.x, u, y[c].x * w);
                    x.y = fmaf(x.y, u, y[c].y * w);
                    x.z = fmaf(x.z, u, y[c].z * w);
                    x.w = fmaf(x.w, u, y[c].w * w);
                }
            }
            const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);      // a NaN stays one
            T* o = out + (size_t)t * a.ldo + (size_t)h * a.HD + col;
            store4<ALIGNED>(o, x.x * inv, x.y * inv, x.z * inv, x.w * inv);
            if (col == 0 && sc.lse != nullptr) sc.lse[((size_t)g * a.T + s.q_begin) * a.G + pr] = l == 0.f ? -INFINITY : m + log2f(l);
        }
    }
    griddep_launch_late();
}

template <typename T, int TY, int TX, int NC, bool CAUSAL>
int go(const void* q, void* out, const RowsArgs& a, const void* k, const void* v, const int* cu_q, const int* kv_len, PageTable pt,
       const long long* masks, RowsScratch s, int* status, cudaStream_t stream) {
    constexpr int R = 4 * TY;
    const size_t smem = (size_t)R * (a.HD + 4) * 4 + (size_t)R * (KT + 4) * 4 + 4 * (size_t)KT * pitch_of<T>(a.HD) * sizeof(T);
    auto kern = attn_rows_kernel<T, TY, TX, NC, CAUSAL>;
    static std::atomic<unsigned long long> opted{0};
    const cudaError_t e = shared_memory_once(kern, MOST_SHARED, opted);
    if (e != cudaSuccess) return mynah_fail("attn_rows: %s", cudaGetErrorString(e));
    kern<<<a.ctas * a.group, TY * TX, smem, stream>>>((const T*)q, (T*)out, (const T*)k, (const T*)v, cu_q, kv_len, pt, masks, a, s, status);
    return mynah_check_launch("attn_rows");
}

template <typename T, bool CAUSAL>
int pick(const void* q, void* out, const RowsArgs& a, const void* k, const void* v, const int* cu_q, const int* kv_len, PageTable pt,
         const long long* masks, RowsScratch s, int* status, cudaStream_t stream) {
#define ROWS_GO(TY, TX, NC) return go<T, TY, TX, NC, CAUSAL>(q, out, a, k, v, cu_q, kv_len, pt, masks, s, status, stream)
    if (a.tile_rows == 16) {
        if (a.HD <= 128) ROWS_GO(4, 32, 1);
        ROWS_GO(4, 32, 2);
    }
    if (a.HD <= 64) ROWS_GO(16, 16, 1);
    if (a.HD <= 128) ROWS_GO(16, 16, 2);
    ROWS_GO(16, 16, 4);
#undef ROWS_GO
}

// Most tiles of a step: what its rows can make (they may lie in any number of its sequences).
long long most_tiles(const RowsArgs& a) { return (long long)a.T * a.G / a.tile_rows + a.B; }

}  // namespace

// Rows of scratch for cut items.
static long long scratch_rows(const RowsArgs& a) { return a.own ? a.cut_rows : a.whole_items ? 0 : 2ll * a.ctas * a.group * a.tile_rows; }

long long rows_scratch_floats(const RowsArgs& a) {
    return scratch_rows(a) * (a.HD + 2) + (a.own ? 0 : (long long)(sizeof(RowStart) / 4) * a.ctas);
}

RowsScratch rows_scratch(const RowsArgs& a, float* scratch, float* lse) {
    const long long rows = scratch_rows(a);
    RowsScratch s;
    s.o = scratch;                                                 // 16-byte rows first
    s.ml = reinterpret_cast<float2*>(scratch + rows * a.HD);
    s.starts = reinterpret_cast<RowStart*>(scratch + rows * (a.HD + 2));
    s.lse = lse;
    s.scores = s.mass = nullptr;
    s.score_rows = s.sum_chunks = 0;
    return s;
}

bool rows_plan(RowsArgs& a, int dtype, int max_q_len, int n_ids, bool aligned) {
    const bool tc = aligned && rows_tcgen05_takes(dtype, a.H, a.KV, a.HD);
    const long long longest = (long long)max_q_len * a.G;          // packed rows of the longest sequence
    // A page is little for the tensor cores and 20,000 clocks of FFMA for 64 rows: there every further CTA helps (3 trees of 19 in
    // fp32 behind 1,021 rows: 35 us with two pages a CTA at least, 25 with one; 8 trees of 24 on the tensor cores: the same).
    a.min_range = tc ? 2 : 1;
    a.q_aligned = aligned;
    a.group = 1;
    a.two = 0;
    a.whole_items = 0;
    a.ctas = 2 * mynah_sm_count();                                 // two CTAs an SM
    a.own = !tc;
    const long long rows = (long long)a.T * a.G;
    if (!tc) {
        a.tile_rows = longest <= 16 ? 16 : 64;                     // (both add a row's products, weights and outputs in the same order)
        a.most_rows = (int)(longest < 1 ? 1 : longest < a.tile_rows ? longest : a.tile_rows);      // (a step may be all padding)
        // Scratch of own_cut for all sequences together: each has up to OWN_PIECES * OWN_ROWS rows of cut items; its pieces of an item
        // are no more than OWN_PIECES / KV, and no more than its listed pages make.
        const long long most = OWN_PIECES / a.KV > 1 ? OWN_PIECES / a.KV : 1, seq_rows = (long long)(a.most_q < a.T ? a.most_q : a.T) * a.G;
        a.cut_rows = (long long)OWN_PIECES * OWN_ROWS * a.B;
        if (a.cut_rows > rows * a.KV * most) a.cut_rows = rows * a.KV * most;
        if (n_ids >= 0 && a.cut_rows > seq_rows * a.KV * (n_ids / a.min_range + a.B)) a.cut_rows = seq_rows * a.KV * (n_ids / a.min_range + a.B);
        a.finish();
        return false;
    }
    a.tile_rows = 128 / a.G * a.G;
    const long long each = (long long)a.B * a.tile_rows;
    if (a.causal && rows / a.tile_rows * a.KV >= mynah_sm_count()) {
        a.whole_items = 1;
        a.ctas = (int)(most_tiles(a) * a.KV);
    } else if (longest > a.tile_rows && 2 * rows >= 3 * each) {
        // From one and a half tiles a sequence on, on average, a CTA takes two; beyond that as many side by side as there are, up to
        // eight tiles (a sequence of fewer leaves CTAs idle).
        a.two = 1;
        a.tile_rows *= 2;
        a.ctas /= 2;
        const long long most = (longest + a.tile_rows - 1) / a.tile_rows, mean = (rows + each) / (2 * each);
        a.group = (int)(mean <= 1 ? 1 : mean > 4 ? 4 : mean);
        if (a.group > most) a.group = (int)most;
        a.ctas /= a.group;
    }
    a.most_rows = (int)(longest < 1 ? 1 : longest < a.tile_rows ? longest : a.tile_rows);      // (a step may be all padding)
    a.finish();
    return tc;
}

int launch_rows_generic(const void* q, void* out, int dtype, const RowsArgs& a, const void* k, const void* v, const int* cu_q,
                        const int* kv_len, PageTable pt, const long long* masks, RowsScratch s, int* status, cudaStream_t stream) {
    auto run = dtype == MYNAH_F32 ? (a.causal ? pick<float, true> : pick<float, false>) : (a.causal ? pick<bf16, true> : pick<bf16, false>);
    return run(q, out, a, k, v, cu_q, kv_len, pt, masks, s, status, stream);
}

template <typename T, bool OWN, bool ALIGNED>
static int join_go(void* out, const RowsArgs& a, const int* cu_q, const int* kv_len, PageTable pt, RowsScratch s, int joining, dim3 grid, int* status,
                   cudaStream_t stream) {
    const cudaError_t e = launch_behind(attn_rows_join_kernel<T, OWN, ALIGNED>, grid, dim3(JOIN_WARPS * 32), 0, stream, (T*)out, cu_q, kv_len, pt, a, s, joining, status);
    if (e != cudaSuccess) return mynah_fail("attn_rows_join: %s", cudaGetErrorString(e));
    return mynah_check_launch("attn_rows_join");
}

int launch_rows_join(void* out, int dtype, const RowsArgs& a, const int* cu_q, const int* kv_len, PageTable pt, RowsScratch s, int* status,
                     cudaStream_t stream) {
    const long long joining = a.own ? most_tiles(a) * a.KV : a.whole_items ? 0 : (a.ctas - 1) * a.group;       // (whole items: nothing is cut)
    long long ctas = joining;
    int helpers = min(ceil_div(a.most_rows, JOIN_WARPS), JOIN_HELPERS);
    if (a.own) {
        // (most tiles of many were not cut, and their CTAs only start to leave: no more than about four an SM beyond one a tile)
        const long long more = ceil_div_ll(4ll * mynah_sm_count(), joining);
        if (helpers > more) helpers = (int)more;
    }
    if (s.scores != nullptr) {
        // a run of at least four pages a CTA, about eight CTAs an SM: with few rows each waits for two reads more than it adds
        const long long bg = (long long)a.B * a.KV, pages = ceil_div_ll(s.entries, a.B), most = ceil_div_ll(8ll * mynah_sm_count(), bg);
        const long long chunks = ceil_div_ll(pages, SUM_PAGES) < most ? ceil_div_ll(pages, SUM_PAGES) : most;
        s.sum_chunks = (int)(chunks < 1 ? 1 : chunks);
        ctas += bg * s.sum_chunks;
    }
    MYNAH_REQUIRE(ctas < (1ll << 31), "attn_rows_join: launch too large");
    if (ctas == 0) return 0;
    const dim3 grid((unsigned)ctas, helpers);
    // (what is cut by the step is the tensor-core kernel's, which takes aligned rows of bfloat16)
    auto run = !a.own ? join_go<bf16, false, true>
             : dtype == MYNAH_F32 ? (a.q_aligned ? join_go<float, true, true> : join_go<float, true, false>)
                                  : (a.q_aligned ? join_go<bf16, true, true> : join_go<bf16, true, false>);
    return run(out, a, cu_q, kv_len, pt, s, (int)joining, grid, status, stream);
}

// Floats of scratch for the attention. n_ids: entries of the page lists, -1 for any number; aligned: whether q's and the output's rows
// are 16-byte aligned, -1 for either.
long long attn_rows_scratch_floats(int T, int B, int max_q_len, int H, int KV, int HD, int dtype, int causal, int n_ids, int aligned) {
    if (T <= 0 || B <= 0 || KV <= 0 || H % KV != 0 || H <= 0 || HD <= 0) return 0;
    long long need = 0;
    for (int al = 0; al < 2; al++) {
        if (aligned >= 0 && al != aligned) continue;
        RowsArgs a{};
        a.T = T, a.B = B, a.H = H, a.KV = KV, a.HD = HD, a.G = H / KV, a.causal = causal;
        a.most_q = causal ? max_q_len : INT_MAX;
        rows_plan(a, dtype, max_q_len, n_ids, al != 0);
        const long long n = rows_scratch_floats(a);
        if (n > need) need = n;
    }
    return (need + 3) & ~3ll;
}
MYNAH_API long long mynah_attn_tree_scratch_floats(int T, int B, int max_q_len, int H, int KV, int HD, int dtype, int n_ids, int aligned) {
    return attn_rows_scratch_floats(T, B, max_q_len, H, KV, HD, dtype, 0, n_ids, aligned);
}

// What mynah_attn_tree and mynah_attn_mass check and launch alike.
int attn_rows_run(const char* who, const void* q, void* out, int dtype, RowsArgs a, int max_q_len, const void* k_cache, const void* v_cache,
                  const int* cu_q, const int* kv_len, PageTable pt, const long long* masks, float* scratch, long long scratch_floats,
                  float* lse, float* scores, int score_rows, int n_ids, float* mass, int* status, cudaStream_t stream) {
    MYNAH_REQUIRE(dtype == MYNAH_F32 || dtype == MYNAH_BF16, "%s: dtype %d is neither float32 nor bfloat16", who, dtype);
    MYNAH_REQUIRE(a.KV > 0 && a.H > 0 && a.H % a.KV == 0 && a.KV <= 65535, "%s: %d heads over %d kv heads", who, a.H, a.KV);
    MYNAH_REQUIRE(a.HD > 0 && a.HD % 8 == 0 && a.HD <= MAX_HEAD, "%s: head_dim %d is no multiple of 8 up to %d", who, a.HD, MAX_HEAD);
    const int es = dtype == MYNAH_F32 ? 4 : 2;
    MYNAH_REQUIRE(a.ldq >= a.H * a.HD && a.ldo >= a.H * a.HD, "%s: rows of %d and %d values for %d heads of %d", who, a.ldq, a.ldo, a.H, a.HD);
    MYNAH_REQUIRE(((uintptr_t)k_cache & 15) == 0 && ((uintptr_t)v_cache & 15) == 0, "%s: the cache must be 16-byte aligned", who);
    MYNAH_REQUIRE((long long)a.T * a.G < (1ll << 30), "%s: %d rows of %d heads a kv head are too many", who, a.T, a.G);
    MYNAH_REQUIRE(status != nullptr && scratch != nullptr && ((uintptr_t)scratch & 15) == 0, "%s: a status word and 16-byte aligned scratch are required", who);
    const bool aligned = ((uintptr_t)q & 15) == 0 && ((uintptr_t)out & 15) == 0 && (long long)a.ldq * es % 16 == 0 && (long long)a.ldo * es % 16 == 0;
    const bool tc = rows_plan(a, dtype, max_q_len, n_ids, aligned);
    const long long need = rows_scratch_floats(a);
    MYNAH_REQUIRE(scratch_floats >= need, "%s: scratch holds %lld floats, %lld are needed", who, scratch_floats, need);
    RowsScratch s = rows_scratch(a, scratch, lse);
    s.scores = scores;
    s.score_rows = score_rows;
    s.entries = n_ids;
    s.mass = mass;
    const int rc = tc ? launch_rows_tcgen05(q, out, a, k_cache, v_cache, cu_q, kv_len, pt, masks, s, status, stream)
                      : launch_rows_generic(q, out, dtype, a, k_cache, v_cache, cu_q, kv_len, pt, masks, s, status, stream);
    if (rc != 0) return rc;
    return launch_rows_join(out, dtype, a, cu_q, kv_len, pt, s, status, stream);
}

// q [T, ldq] and out [T, ldo], head h in columns [h * HD, (h + 1) * HD); k_cache, v_cache [n_pages, KV, 64, HD], which hold the
// step's own rows already; cu_q [B + 1], kv_len [B]; masks [T, words]: bit j of a token's words says that it sees the step's row
// j of its sequence. scale 0: 1 / sqrt(HD). Rows of out behind the last sequence are left as they are.
// (The arguments come as one struct, which struct.pack fills: 26 ctypes conversions take 2.3 us more.)
struct AttnTreeCall {
    const void* q;
    void* out;
    int dtype, T, B, max_q_len, H, KV, HD, ldq, ldo;
    const void *k_cache, *v_cache;
    const int *cu_q, *kv_len, *page_indptr, *page_ids, *page_base;
    int n_pages, n_ids;
    const long long* masks;
    int words;
    float scale;
    float* scratch;
    long long scratch_floats;
    int* status;
    cudaStream_t stream;
};
static_assert(sizeof(AttnTreeCall) == 168, "as packed by the caller");
MYNAH_API int mynah_attn_tree(const AttnTreeCall* call) {
    const auto& [q, out, dtype, T, B, max_q_len, H, KV, HD, ldq, ldo, k_cache, v_cache, cu_q, kv_len, page_indptr, page_ids, page_base, n_pages, n_ids,
                 masks, words, scale, scratch, scratch_floats, status, stream] = *call;
    if (T <= 0 || B <= 0) return 0;
    MYNAH_REQUIRE(masks != nullptr && words > 0 && n_ids >= 0, "attn_tree: mask words and the number of page entries are required");
    MYNAH_REQUIRE(scale == 0.f || (scale >= 0x1p-120f && scale <= 0x1p120f), "attn_tree: the score scale %g is not between 2^-120 and 2^120, nor 0", scale);
    RowsArgs a{};
    a.T = T, a.B = B, a.H = H, a.KV = KV, a.HD = HD, a.G = KV > 0 ? H / KV : 0, a.ldq = ldq, a.ldo = ldo, a.words = words;
    a.most_q = INT_MAX;                                            // (max_q_len gives the tiles their size, and rows beyond it are more tiles)
    a.scale_log2 = (scale != 0.f ? scale : 1.0f / sqrtf((float)HD)) * 1.4426950408889634f;
    return attn_rows_run("attn_tree", q, out, dtype, a, max_q_len, k_cache, v_cache, cu_q, kv_len,
                         PageTable{page_indptr, page_ids, page_base, n_pages}, masks, scratch, scratch_floats, nullptr, nullptr, 0, n_ids, nullptr, status, stream);
}
