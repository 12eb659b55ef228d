// Attention of a few rows a sequence on the fifth-generation tensor cores (bfloat16, heads of 64 and 128): the formulas and the
// cut into units are those of attn_rows.cu and row_units.cuh. A unit is up to 128 packed rows (tokens times the query heads of a
// kv head: the lanes of tensor memory) against one chunk of the sequence's pages, 128 keys (two pages) a tile:
//
//   warp 0     one lane brings the rows' queries once (a box of 64 columns x the group's heads x the tile's tokens lands as the
//              packed rows) and then each tile's K and V pages with TMA (128-byte swizzle);
//   warp 1     one lane issues tcgen05.mma: S = Q.K^T into tensor memory, and O += P.V with P read from tensor memory and V as
//              an MN-major operand in shared memory;
//   warps 2-9  the softmax: two threads a row, one for each half of a tile's keys. Scores in registers, the row's maximum
//              exchanged through shared memory, O rescaled only when the reference maximum has to grow by more than 2^8,
//              weights written back over the scores as bfloat16 (they lose half a step, 2^-9 on average, as much as the output's
//              own rounding; their sum is of the unrounded ones in fp32). Warps whose rows do not exist only keep step.
//
// Bound by: bytes of K and V while a unit has few rows (a page of 32 KB against 64 keys x rows of softmax), by the softmax's
// instructions from about 128 rows on. A matrix instruction of 128 rows costs the same however many of them exist, which is a
// third of a page's share of the memory's time.
//
// A key that a row must not see gets the score -inf by a select, so its K cannot matter. Its V could: a weight of zero times a
// NaN is a NaN. So in tiles where some row does not see some key the values are looked through: rows that nobody sees are
// zeroed, and values that are not finite are zeroed and, behind the last tile, added to the rows that do see them.
//
// Every wait is bounded (2 s); one that runs out sets MYNAH_ST_TIMEOUT, and the CTA drains its copies, frees its tensor memory
// and returns.
#include "attn_rows.cuh"
#include "rows_tcgen05.cuh"

#include <math.h>

namespace {

using namespace tc5;

constexpr int BQ = 128;               // packed rows a tile at most (the lanes of tensor memory)
constexpr int BKV = 128;              // keys a tile
constexpr int THREADS = 320;
// Which of two packed bfloat16 are not finite, as a mask over their bits.
__device__ __forceinline__ uint32_t not_finite2(uint32_t w) {
    return ((w & 0x7f80u) == 0x7f80u ? 0xffffu : 0u) | ((w & 0x7f800000u) == 0x7f800000u ? 0xffff0000u : 0u);
}

template <int HD>
__global__ void __launch_bounds__(THREADS, 1)
attn_rows_tcgen05_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                         const __grid_constant__ CUtensorMap map_v, const bf16* __restrict__ v_cache, const int* __restrict__ cu_q,
                         const int* __restrict__ kv_len, PageTable pt, const long long* __restrict__ masks, RowsArgs a,
                         bf16* __restrict__ out, RowsScratch sc, int* __restrict__ status) {
    constexpr int HALVES = HD / 64;
    constexpr int TILE_BYTES = HALVES * HALF_BYTES;
    constexpr int NS = 2;                                      // stages of K, V and the scores
    constexpr int TMEM_COLS = 512, O_COL = NS * BKV;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    unsigned char* q_s = smem;
    unsigned char* k_s = q_s + TILE_BYTES;                     // NS stages
    unsigned char* v_s = k_s + NS * TILE_BYTES;                // NS stages
    uint64_t* bars = reinterpret_cast<uint64_t*>(v_s + NS * TILE_BYTES);
    const uint32_t q_full = smem_u32(bars), k_full = smem_u32(bars + 1), v_full = smem_u32(bars + 3);   // [2] each, 8 bytes apart
    const uint32_t s_full = smem_u32(bars + 5), v_free = smem_u32(bars + 7);
    const uint32_t p_full = smem_u32(bars + 9), o_done = smem_u32(bars + 11), x_full = smem_u32(bars + 12);
    const uint32_t o_last = smem_u32(bars + 14);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 15);
    int* flags = reinterpret_cast<int*>(bars + 16);            // [0] a page is missing, [1] a value that is not finite was zeroed
    float* xch = reinterpret_cast<float*>(bars + 18);          // [2 buffers][2 groups][128 rows]

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) flags[0] = flags[1] = 0;
    RowUnit u;
    if (!find_row_unit(cu_q, kv_len, a, blockIdx.x / a.KV, u, status)) return;     // the whole CTA: nothing is set up yet
    const int g = blockIdx.x % a.KV;
    const int n_rows = u.rows(a), past = u.past(), row0 = u.tile * a.tile_rows, kvl = u.s.kvl;
    const int pages = u.tile_pages(a), pg0 = u.chunk * u.cp, pg1 = min(pages, pg0 + u.cp);
    const int n_chunks = (pages + u.cp - 1) / u.cp;
    if (threadIdx.x == 0 && g == 0 && u.tile == u.s.tiles - 1 && u.chunk == 0) sc.info[u.b] = RowInfo{u.unit0, u.cp};
    if (u.chunk >= n_chunks) return;                           // a causal tile that ends before this chunk
    // every page of the chunk must be there: a chunk that lacks one counts as keys that nobody sees
    for (int p = pg0 + (int)threadIdx.x; p < pg1; p += THREADS)
        if (page_of(pt, u.b, p * PAGE_TOKENS) < 0) flags[0] = 1;
    const int active = (n_rows + 31) >> 5;                     // quadrants of the tile that have rows
    if (threadIdx.x == 0) {
        mbar_init(q_full, 1);
        for (int i = 0; i < 2; i++) {
            mbar_init(k_full + 8 * i, 1);
            mbar_init(v_full + 8 * i, 1);
            mbar_init(s_full + 8 * i, 1);
            mbar_init(v_free + 8 * i, 1);
            mbar_init(p_full + 8 * i, 8);                      // one arrival per softmax warp
            mbar_init(x_full + 8 * i, 2 * active);
        }
        mbar_init(o_done, 1);
        mbar_init(o_last, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        fence_async_smem();
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    const bool bad = flags[0] != 0;
    const int n_tiles = bad ? 0 : (pg1 - pg0 + 1) >> 1;
    const int key_begin = pg0 * PAGE_TOKENS, key_end = min(kvl, pg1 * PAGE_TOKENS);      // of this chunk
    const int first_tok = row0 / a.G;
    // Is there a key among [key0, key0 + n) that some row of the tile must not see?
    auto masked = [&](int key0, int n) { return key0 + n > key_end || (a.causal ? key0 + n - 1 > past + first_tok : key0 + n > past); };

    // Tile j uses stage j & 1 of K, V and the scores; its barriers are in their (j >> 1)-th use.
    if (warp == 0) {
        if (lane == 0) {                                       // ---- TMA producer
            if (bad) atomicOr(status, MYNAH_ST_PAGE_RANGE);
            bool q_asked = false;
            int k_issued = 0, v_issued = 0;
            for (int j = 0; j < n_tiles; j++) {
                const int st = j & 1;
                const uint32_t prev_use = ((j >> 1) & 1) ^ 1;  // parity of the stage's use before this one
                const int key0 = key_begin + j * BKV;
                const bool two = pg0 + 2 * j + 1 < pg1;
                const int p0 = page_of(pt, u.b, key0), p1 = two ? page_of(pt, u.b, key0 + PAGE_TOKENS) : 0;
                if (j >= NS && !mbar_wait(s_full + 8 * st, prev_use)) {     // the scores of tile j - 2 are done: its K is free
                    atomicOr(status, MYNAH_ST_TIMEOUT);
                    break;
                }
                unsigned char* kd = k_s + st * TILE_BYTES;
                const uint32_t bytes = (two ? 2 : 1) * HALVES * PAGE_BYTES;
                mbar_expect_tx(k_full + 8 * st, bytes);
#pragma unroll
                for (int hf = 0; hf < HALVES; hf++) {
                    tma_load_2d(smem_u32(kd + hf * HALF_BYTES), &map_k, hf * 64, (p0 * a.KV + g) * PAGE_TOKENS, k_full + 8 * st);
                    if (two) tma_load_2d(smem_u32(kd + hf * HALF_BYTES + PAGE_BYTES), &map_k, hf * 64, (p1 * a.KV + g) * PAGE_TOKENS, k_full + 8 * st);
                }
                k_issued = j + 1;
                if (!q_asked) {
                    mbar_expect_tx(q_full, HALVES * a.tile_rows * 128);
#pragma unroll
                    for (int hf = 0; hf < HALVES; hf++)
                        tma_load_3d(smem_u32(q_s + hf * HALF_BYTES), &map_q, hf * 64, g * a.G, u.s.q_begin + first_tok, q_full);
                    q_asked = true;
                }
                if (j >= NS && !mbar_wait(v_free + 8 * st, prev_use)) {     // the second product of tile j - 2 is done: its V is free
                    atomicOr(status, MYNAH_ST_TIMEOUT);
                    break;
                }
                unsigned char* vd = v_s + st * TILE_BYTES;
                mbar_expect_tx(v_full + 8 * st, bytes);
#pragma unroll
                for (int hf = 0; hf < HALVES; hf++) {
                    tma_load_2d(smem_u32(vd + hf * HALF_BYTES), &map_v, hf * 64, (p0 * a.KV + g) * PAGE_TOKENS, v_full + 8 * st);
                    if (two) tma_load_2d(smem_u32(vd + hf * HALF_BYTES + PAGE_BYTES), &map_v, hf * 64, (p1 * a.KV + g) * PAGE_TOKENS, v_full + 8 * st);
                }
                v_issued = j + 1;
            }
            // whatever was started still lands in this CTA's shared memory: wait for it before leaving (bounded)
            if (q_asked) mbar_wait(q_full, 0);
            for (int j = max(0, k_issued - NS); j < k_issued; j++) mbar_wait(k_full + 8 * (j & 1), (j >> 1) & 1);
            for (int j = max(0, v_issued - NS); j < v_issued; j++) mbar_wait(v_full + 8 * (j & 1), (j >> 1) & 1);
        }
    } else if (warp == 1) {
        if (lane == 0 && n_tiles > 0) {                        // ---- MMA issuer
            constexpr uint32_t idesc_s = idesc(BKV, false), idesc_o = idesc(HD, true);
            const uint32_t t_o = tmem_base + O_COL;
            const uint32_t q_addr = smem_u32(q_s), k_addr = smem_u32(k_s), v_addr = smem_u32(v_s);
            auto scores = [&](int j) {                         // S[stage of j] = Q . K_j^T
                const int st = j & 1;
#pragma unroll
                for (int k = 0; k < HD / 16; k++) {
                    const uint32_t off = (k / 4) * HALF_BYTES + (k % 4) * 32;
                    tc_mma(tmem_base + st * BKV, desc_k_major(q_addr + off), desc_k_major(k_addr + st * TILE_BYTES + off), idesc_s, k != 0);
                }
                tc_commit(s_full + 8 * st);
            };
            bool ok = mbar_wait(q_full, 0) && mbar_wait(k_full, 0);
            if (ok) {
                tc_fence_after();
                scores(0);
            }
            for (int j = 0; j < n_tiles && ok; j++) {
                const int st = j & 1;
                if (j + 1 < n_tiles) {                         // the next tile's scores, while the softmax works on this one.
                    // Their buffer held the weights of tile j - 1; the product that read them was issued before.
                    ok = mbar_wait(k_full + 8 * (st ^ 1), ((j + 1) >> 1) & 1);
                    if (!ok) break;
                    tc_fence_after();
                    scores(j + 1);
                }
                ok = mbar_wait(p_full + 8 * st, (j >> 1) & 1) && mbar_wait(v_full + 8 * st, (j >> 1) & 1);
                if (!ok) break;
                tc_fence_after();
#pragma unroll
                for (int k = 0; k < BKV / 16; k++)             // 16 keys a step: 8 columns of packed weights, 16 rows of V
                    tc_mma_ts(t_o, tmem_base + st * BKV + k * 8, desc_mn_major(v_addr + st * TILE_BYTES + k * 16 * 128, HALF_BYTES),
                              idesc_o, (j | k) != 0);
                tc_commit(v_free + 8 * st);
                // The last product has a barrier of its own: behind the last tile a warp may be two phases of o_done ahead of the
                // slowest, where a wait for a parity would be answered by the phase before.
                tc_commit(j + 1 < n_tiles ? o_done : o_last);
            }
            if (!ok) atomicOr(status, MYNAH_ST_TIMEOUT);
        }
    } else {
        // ---- softmax: warps 2..5 take the first 64 keys of a tile, warps 6..9 the other 64; a warp reads the lane quadrant
        // (warp % 4) of tensor memory, so two threads, one in each group, share a row.
        constexpr int HALF_KEYS = BKV / 2;
        const int grp = (warp - 2) >> 2, quad = warp & 3, row = quad * 32 + lane;
        const bool works = quad < active;
        const int tok = (row0 + row) / a.G;                    // of the sequence
        const long long* words = masks + (size_t)(u.s.q_begin + min(tok, u.s.n_q - 1)) * a.words;
        const uint32_t t_row = tmem_base + ((uint32_t)(quad * 32) << 16);
        const uint32_t t_o = t_row + O_COL + grp * (HD / 2);   // this thread's half of the row of O
        float m_ref = -INFINITY, l = 0.f;                      // the maximum that the sums are scaled by; the sum over this thread's keys
        bool ok = true;
        for (int j = 0; j < n_tiles; j++) {
            const int st = j & 1;
            const uint32_t use = (j >> 1) & 1;
            const int tile_key0 = key_begin + j * BKV, key0 = tile_key0 + grp * HALF_KEYS;     // this thread's first key
            const uint32_t t_s = t_row + st * BKV;
            if (!warp_wait(s_full + 8 * st, use)) { ok = false; break; }
            tc_fence_after();
            if (works) {
                float s[HALF_KEYS];
#pragma unroll
                for (int c = 0; c < 2; c++) tc_ld32_nowait(t_s + grp * HALF_KEYS + c * 32, reinterpret_cast<uint32_t(&)[32]>(s[c * 32]));
#pragma unroll
                for (int c = 0; c < 2; c++) tc_wait_ld(reinterpret_cast<uint32_t(&)[32]>(s[c * 32]));
                if (masked(key0, HALF_KEYS)) {
                    const unsigned long long vis = row < n_rows ? visible64(key0, key_end, past, tok, a.causal, words, a.words) : 0ull;
                    const uint32_t v0 = (uint32_t)vis, v1 = (uint32_t)(vis >> 32);
#pragma unroll
                    for (int e = 0; e < 32; e++) {
                        s[e] = (v0 >> e) & 1u ? s[e] : -INFINITY;
                        s[32 + e] = (v1 >> e) & 1u ? s[32 + e] : -INFINITY;
                    }
                }
                float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int e = 0; e < HALF_KEYS; e += 2) mx4[(e >> 1) & 3] = max3(mx4[(e >> 1) & 3], s[e], s[e + 1]);
                const float mx_own = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3]));
                // the row's maximum over both groups, through shared memory (two buffers: a value is read before the barrier of the
                // next tile, and overwritten only after it)
                xch[(st * 2 + grp) * BQ + row] = mx_own;
                __syncwarp();
                if (lane == 0) mbar_arrive(x_full + 8 * st);
                if (!warp_wait(x_full + 8 * st, use)) { ok = false; break; }
                const float m_new = fmaxf(mx_own, xch[(st * 2 + (grp ^ 1)) * BQ + row]) * a.scale_log2;
                // The reference follows the true maximum lazily: while that stays within 2^8 of it nothing is rescaled. Both
                // threads of a row take the same decision.
                float alpha = 1.0f;
                if (m_new > m_ref + 8.0f || (m_ref == -INFINITY && m_new != -INFINITY)) {
                    alpha = ex2_f(m_ref - m_new);              // 0 for the first seen key
                    m_ref = m_new;
                }
                const float m_use = m_ref == -INFINITY ? 0.f : m_ref;
                // O is touched only when some row of the warp has to be rescaled; then the product of the tile before must have
                // finished. (o_done can be at most one phase ahead of the tile whose weights have not been handed over yet.)
                if (j > 0 && __any_sync(0xffffffffu, alpha != 1.0f)) {
                    if (!warp_wait(o_done, (j - 1) & 1)) { ok = false; break; }
                    tc_fence_after();
#pragma unroll 1
                    for (int c = 0; c < HD / 64; c++) {
                        uint32_t r[32];
                        tc_ld32(t_o + c * 32, r);
#pragma unroll
                        for (int e = 0; e < 32; e++) r[e] = __float_as_uint(__uint_as_float(r[e]) * alpha);
                        tc_st32(t_o + c * 32, r);
                    }
                    tc_wait_st();
                }
                float sum4[4] = {0.f, 0.f, 0.f, 0.f};
                uint32_t pk[HALF_KEYS / 2];
#pragma unroll
                for (int e = 0; e < HALF_KEYS; e += 2) {
                    float x0, x1;
                    fma2(x0, x1, s[e], s[e + 1], a.scale_log2, -m_use);
                    const float p0 = ex2_f(x0), p1 = ex2_f(x1);                   // 2^-inf = 0
                    add2(sum4[e & 2], sum4[(e & 2) + 1], p0, p1);
                    pk[e >> 1] = pack2(p0, p1);
                }
                // over the scores: both groups have theirs in registers since the exchange above
                tc_st32(t_s + grp * (HALF_KEYS / 2), pk);
                tc_wait_st();
                l = l * alpha + ((sum4[0] + sum4[1]) + (sum4[2] + sum4[3]));
            }
            if (masked(tile_key0, BKV)) {                      // look through V: one thread a key's row and half of the columns
                if (!warp_wait(v_full + 8 * st, use)) { ok = false; break; }
                if (grp < HALVES) {
                    uint4* dst = reinterpret_cast<uint4*>(v_s + st * TILE_BYTES + grp * HALF_BYTES + row * 128);
                    if (tile_key0 + row >= key_end) {          // nobody's
#pragma unroll
                        for (int i = 0; i < 8; i++) dst[i] = make_uint4(0u, 0u, 0u, 0u);
                    } else {
#pragma unroll
                        for (int i = 0; i < 8; i++) {
                            uint4 x = dst[i];
                            const uint32_t n0 = not_finite2(x.x), n1 = not_finite2(x.y), n2 = not_finite2(x.z), n3 = not_finite2(x.w);
                            if (n0 | n1 | n2 | n3) {
                                x.x &= ~n0, x.y &= ~n1, x.z &= ~n2, x.w &= ~n3;
                                dst[i] = x;
                                flags[1] = 1;
                            }
                        }
                    }
                }
                fence_async_smem();
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(p_full + 8 * st);
        }
        asm volatile("bar.sync 1, 256;" ::: "memory");       // what any warp found in V is known to all
        if (ok && n_tiles > 0 && !warp_wait(o_last, 0)) ok = false;
        if (ok && works) {
            // the row sum over both groups, through the same exchange (its barriers are in use n_tiles by now)
            const int st = n_tiles & 1;
            xch[(st * 2 + grp) * BQ + row] = l;
            __syncwarp();
            if (lane == 0) mbar_arrive(x_full + 8 * st);
            if (!warp_wait(x_full + 8 * st, (n_tiles >> 1) & 1)) ok = false;
            else l += xch[(st * 2 + (grp ^ 1)) * BQ + row];
        }
        if (ok && works) {
            tc_fence_after();
            const bool poison = *(volatile int*)(flags + 1) != 0;
            const bool direct = n_chunks == 1;
            const float inv = direct ? (l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l)) : 1.f;      // a NaN stays one
            const int h = g * a.G + (row0 + row) % a.G;
            const size_t t = (size_t)u.s.q_begin + tok;
            const long long slot = (long long)blockIdx.x * a.tile_rows + row;     // [unit][kv head][row]
#pragma unroll 1
            for (int c = 0; c < HD / 64; c++) {
                const int col = grp * (HD / 2) + c * 32;
                uint32_t r[32];
                if (n_tiles > 0) tc_ld32(t_o + c * 32, r);
                else {
#pragma unroll
                    for (int e = 0; e < 32; e++) r[e] = 0u;
                }
                if (row < n_rows) {
                    if (poison) {                              // the values that were zeroed, to the rows that see them
                        for (int j = 0; j < n_tiles; j++) {
                            if (!masked(key_begin + j * BKV, BKV)) continue;
                            for (int k = 0; k < BKV; k++) {
                                const int key = key_begin + j * BKV + k;
                                if (key >= key_end) break;
                                if (!((visible64(key & ~63, key_end, past, tok, a.causal, words, a.words) >> (key & 63)) & 1ull)) continue;
                                const bf16* vr = v_cache + (((size_t)page_of(pt, u.b, key) * a.KV + g) * PAGE_TOKENS + key % PAGE_TOKENS) * HD + col;
                                // (r is indexed by constants alone, so that it stays in registers)
#pragma unroll
                                for (int e = 0; e < 32; e++) {
                                    const float x = __bfloat162float(vr[e]);
                                    if (!isfinite(x)) r[e] = __float_as_uint(__uint_as_float(r[e]) + x);
                                }
                            }
                        }
                    }
                    if (direct) {
                        bf16* o = out + t * a.ldo + (size_t)h * HD + col;
#pragma unroll
                        for (int i = 0; i < 4; i++)
                            reinterpret_cast<uint4*>(o)[i] =
                                make_uint4(pack2(__uint_as_float(r[8 * i]) * inv, __uint_as_float(r[8 * i + 1]) * inv),
                                           pack2(__uint_as_float(r[8 * i + 2]) * inv, __uint_as_float(r[8 * i + 3]) * inv),
                                           pack2(__uint_as_float(r[8 * i + 4]) * inv, __uint_as_float(r[8 * i + 5]) * inv),
                                           pack2(__uint_as_float(r[8 * i + 6]) * inv, __uint_as_float(r[8 * i + 7]) * inv));
                    } else {
                        uint4* o = reinterpret_cast<uint4*>(sc.o + slot * HD + col);
#pragma unroll
                        for (int i = 0; i < 8; i++) o[i] = make_uint4(r[4 * i], r[4 * i + 1], r[4 * i + 2], r[4 * i + 3]);
                    }
                }
            }
            if (row < n_rows && grp == 0) {
                if (!direct) sc.ml[slot] = make_float2(m_ref, l);
                else if (sc.lse != nullptr) sc.lse[((size_t)g * a.T + u.s.q_begin) * a.G + row0 + row] = l == 0.f ? -INFINITY : m_ref + log2f(l);
            }
        }
        if (!ok && lane == 0) atomicOr(status, MYNAH_ST_TIMEOUT);
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(TMEM_COLS) : "memory");
    }
}

template <int HD>
int go(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, const void* v, const int* cu_q, const int* kv_len, PageTable pt,
       const long long* masks, const RowsArgs& a, void* out, RowsScratch s, int* status, cudaStream_t stream) {
    constexpr size_t smem = 5 * (size_t)(HD / 64) * HALF_BYTES + 144 + 2 * 2 * BQ * sizeof(float) + 1024;
    auto kern = attn_rows_tcgen05_kernel<HD>;
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return mynah_fail("attn_rows: %s", cudaGetErrorString(e));
    kern<<<(unsigned)(row_units_max(a) * a.KV), THREADS, smem, stream>>>(mq, mk, mv, (const bf16*)v, cu_q, kv_len, pt, masks, a, (bf16*)out, s, status);
    return mynah_check_launch("attn_rows");
}

}  // namespace

bool rows_tcgen05_takes(int dtype, int H, int KV, int HD) {
    return dtype == MYNAH_BF16 && (HD == 64 || HD == 128) && KV > 0 && H % KV == 0 && H / KV <= BQ;
}

int launch_rows_tcgen05(const void* q, void* out, const RowsArgs& a, const void* k, const void* v, const int* cu_q,
                        const int* kv_len, PageTable pt, const long long* masks, RowsScratch s, int* status, cudaStream_t stream) {
    const long long rows = (long long)pt.n_pages * a.KV * PAGE_TOKENS;
    MYNAH_REQUIRE(rows < (1ll << 31) && row_units_max(a) * a.KV < (1ll << 31), "attn_rows: launch too large");
    if (pt.n_pages == 0) return mynah_fail("attn_rows: a cache without pages");
    CUtensorMap mq, mk, mv;
    if (make_map_rows(&mq, q, a.T, a.H, a.HD, a.G, a.ldq, a.tile_rows / a.G)) return -1;
    if (make_map(&mk, k, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, rows, a.HD, a.HD, PAGE_TOKENS, 64)) return -1;
    if (make_map(&mv, v, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, rows, a.HD, a.HD, PAGE_TOKENS, 64)) return -1;
    if (a.HD == 128) return go<128>(mq, mk, mv, v, cu_q, kv_len, pt, masks, a, out, s, status, stream);
    return go<64>(mq, mk, mv, v, cu_q, kv_len, pt, masks, a, out, s, status, stream);
}
