// Attention of a few rows a sequence on the fifth-generation tensor cores (bfloat16, heads of 64 and 128): the formulas are those
// of attn_rows.cu, the shares of the CTAs those of row_units.cuh. A tile is up to 128 packed rows (tokens times the query heads
// of a kv head: the lanes of tensor memory), the keys come a page of 64 at a time:
//
//   warp 0     one lane brings a tile's queries (a box of 64 columns x the group's heads x the tile's tokens lands as the packed
//              rows) and the pages' K and V with TMA (128-byte swizzle), in rings that run on from segment to segment;
//   warp 1     issues S = Q.K^T into tensor memory (two buffers),
//   warp 2     O += P.V, P read from tensor memory and V as an MN-major operand in shared memory: two warps, because an issuer
//              that waits for weights keeps the tensor cores from the next scores (one warp for both took 2,200 clocks a page of
//              two tiles, these 2,100). Both run whole, with one elected lane at the instructions: under `lane == 0` every
//              descriptor went through vector registers and a product took 85 clocks to issue, under elect.sync 55;
//   warps 3-6  the softmax, a thread a row: 64 scores in registers, O rescaled only when the reference maximum has to grow by
//              more than 2^8, weights written back over the scores as bfloat16 (half a step is lost, as much as the output's own
//              rounding loses; their sum is of the unrounded ones in fp32). Warps whose rows do not exist only keep step.
//
// NT = 1: one tile, two CTAs an SM (107 KB and 256 columns of tensor memory each): one's softmax runs under the other's products
// and its start and end under the other's pages. NT = 2: two tiles of 128 rows on the same pages, with warps 7-10 for the second,
// one CTA an SM: a page is brought into shared memory once for 256 rows. Bound by the bytes of K and V while there are few rows;
// a page takes the tensor cores about 640 clocks a tile whatever its rows (Q.K^T of 64 columns waits for shared memory), the
// exponentials of 128 rows 512, its share of the memory's time is 1,400.
//
// A key that a row must not see gets the score -inf by a select, so its K cannot matter. Its V could: a weight of zero times a
// NaN is a NaN. So in pages where some row does not see some key the values are looked through: rows that nobody sees are
// zeroed, and values that are not finite are zeroed and, behind the segment's last page, added to the rows that do see them.
//
// Every wait is bounded (2 s); one that runs out sets MYNAH_ST_TIMEOUT, and the CTA drains its copies, frees its tensor memory
// and returns.
#include "attn_rows.cuh"
#include "rows_tcgen05.cuh"

#include <math.h>

namespace {

using namespace tc5;

constexpr int BQ = 128;               // packed rows a tile at most (the lanes of tensor memory)
constexpr int KEYS = PAGE_TOKENS;     // keys a step
constexpr int STAGE_PITCH = 20;       // floats: rows of 80 bytes, whose 16-byte pieces meet no bank twice in eight lanes
template <int HD, int NT> constexpr int STAGES = HD == 128 ? 2 * NT : 4 * NT;       // of K and of V

// Which of two packed bfloat16 are not finite, as a mask over their bits.
__device__ __forceinline__ uint32_t not_finite2(uint32_t w) {
    return ((w & 0x7f80u) == 0x7f80u ? 0xffffu : 0u) | ((w & 0x7f800000u) == 0x7f800000u ? 0xffff0000u : 0u);
}

template <int HD, int NT, bool CAUSAL>
__global__ void __launch_bounds__(96 + 128 * NT, 3 - NT)
attn_rows_tcgen05_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                         const __grid_constant__ CUtensorMap map_v, const bf16* __restrict__ v_cache, const int* __restrict__ cu_q,
                         const int* __restrict__ kv_len, PageTable pt, const long long* __restrict__ masks, RowsArgs a,
                         bf16* __restrict__ out, RowsScratch sc, int* __restrict__ status) {
    constexpr int HALVES = HD / 64, NS = STAGES<HD, NT>;
    constexpr int PAGE_TILE = HALVES * PAGE_BYTES;             // one page of K or of V
    constexpr int TMEM_COLS = 256 * NT, O_COL = 2 * KEYS * NT; // two score buffers a tile, the outputs behind them
    constexpr int Q_TILE = HALVES * HALF_BYTES;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    unsigned char* q_s = smem;
    unsigned char* k_s = q_s + NT * Q_TILE;                    // NS stages
    unsigned char* v_s = k_s + NS * PAGE_TILE;                 // NS stages
    float* stage_s = reinterpret_cast<float*>(v_s + NS * PAGE_TILE);       // [softmax warps][32 rows][16 columns]
    uint64_t* bars = reinterpret_cast<uint64_t*>(stage_s + NT * 4 * 32 * STAGE_PITCH);
    const uint32_t k_full = smem_u32(bars), v_full = smem_u32(bars + 8), k_free = smem_u32(bars + 16), v_free = smem_u32(bars + 24);   // [NS]
    const uint32_t s_full = smem_u32(bars + 32), p_full = smem_u32(bars + 36);       // [NT][2]: scores ready, weights ready
    const uint32_t q_full = smem_u32(bars + 40), q_free = smem_u32(bars + 41);       // once a segment
    const uint32_t p_free = smem_u32(bars + 42);               // [NT][2]: the output has the page, its buffer is free
    const uint32_t o_free = smem_u32(bars + 46);               // once a segment: the outputs have been read
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 47);
    int* flags = reinterpret_cast<int*>(bars + 48);            // [0], [1]: 1 + the last segment (even, odd) in which a value that is
                                                               // not finite was zeroed; [2 .. 9]: the same for missing pages, by
                                                               // segment % 8 (the producer is up to three segments ahead)
    __shared__ RowWalk<CAUSAL, false> walk_s;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (warp == 0) {
        find_start(cu_q, kv_len, pt, a, &walk_s, sc.starts, status);
    } else if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    } else if (threadIdx.x == 96) {
        for (int i = 0; i < NS; i++) {
            mbar_init(k_full + 8 * i, 1);
            mbar_init(v_full + 8 * i, 1);
            mbar_init(k_free + 8 * i, 1);
            mbar_init(v_free + 8 * i, 1);
        }
        for (int i = 0; i < 2 * NT; i++) {
            mbar_init(s_full + 8 * i, 1);
            mbar_init(p_full + 8 * i, 4);                      // one arrival per softmax warp of the tile
            mbar_init(p_free + 8 * i, 1);
        }
        mbar_init(q_full, 1);
        mbar_init(q_free, 1);
        mbar_init(o_free, 4 * NT);
        for (int i = 0; i < 10; i++) flags[i] = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        fence_async_smem();
    } else if (threadIdx.x == 64) {
        for (const CUtensorMap* m : {&map_q, &map_k, &map_v}) asm volatile("prefetch.tensormap [%0];" ::"l"(m) : "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    RowWalk<CAUSAL, false> u = walk_s;
    const bool any = u.b >= 0;
    const int tile_rows = NT == 2 ? a.tile_rows >> 1 : a.tile_rows;                    // of one tile; a tile exists if the CTA's rows reach it

    // Page number i of the CTA (over all segments) uses stage i % NS of K and V, in that stage's use i / NS; the pages of a tile number
    // c use its score buffer c & 1.
    if (warp == 0) {
        if (lane == 0 && any) {                                // ---- TMA producer
            int i = 0, seg = 0, k_issued = 0, v_issued = 0, q_issued = 0;
            bool ok = true;
            do {
                for (int p = u.pg0; p < u.pg1; p++, i++) {
                    const int st = i % NS;
                    const uint32_t prev = ((i / NS) & 1) ^ 1;  // parity of the stage's use before this one
                    int page = page_at(pt, u.s, p);
                    if (page < 0) {                            // the segment will count as keys that nobody sees
                        atomicOr(status, MYNAH_ST_PAGE_RANGE);
                        *(volatile int*)(flags + 2 + (seg & 7)) = seg + 1;
                        page = 0;
                    }
                    if (i >= NS && !mbar_wait(k_free + 8 * st, prev)) { ok = false; break; }
                    mbar_expect_tx(k_full + 8 * st, PAGE_TILE);
#pragma unroll
                    for (int hf = 0; hf < HALVES; hf++)
                        tma_load_2d(smem_u32(k_s + st * PAGE_TILE + hf * PAGE_BYTES), &map_k, hf * 64, (page * a.KV + u.g) * PAGE_TOKENS, k_full + 8 * st);
                    k_issued = i + 1;
                    if (p == u.pg0) {
                        if (seg > 0 && !mbar_wait(q_free, (seg - 1) & 1)) { ok = false; break; }
                        const int nt = NT == 1 || u.rows(a) <= tile_rows ? 1 : NT;
                        mbar_expect_tx(q_full, nt * HALVES * tile_rows * 128);
                        for (int x = 0; x < nt; x++)
#pragma unroll
                            for (int hf = 0; hf < HALVES; hf++)
                                tma_load_3d(smem_u32(q_s + x * Q_TILE + hf * HALF_BYTES), &map_q, hf * 64, u.g * a.G,
                                            u.s.q_begin + a.by_G.div(u.tile * a.tile_rows + x * tile_rows), q_full);
                        q_issued = seg + 1;
                    }
                    if (i >= NS && !mbar_wait(v_free + 8 * st, prev)) { ok = false; break; }
                    mbar_expect_tx(v_full + 8 * st, PAGE_TILE);
#pragma unroll
                    for (int hf = 0; hf < HALVES; hf++)
                        tma_load_2d(smem_u32(v_s + st * PAGE_TILE + hf * PAGE_BYTES), &map_v, hf * 64, (page * a.KV + u.g) * PAGE_TOKENS, v_full + 8 * st);
                    v_issued = i + 1;
                }
                seg++;
            } while (ok && u.next(cu_q, kv_len, pt, a, status));
            if (!ok) atomicOr(status, MYNAH_ST_TIMEOUT);
            // whatever was started still lands in this CTA's shared memory: wait for it before leaving (bounded)
            if (q_issued > 0) mbar_wait(q_full, (q_issued - 1) & 1);
            for (int j = max(0, k_issued - NS); j < k_issued; j++) mbar_wait(k_full + 8 * (j % NS), (j / NS) & 1);
            for (int j = max(0, v_issued - NS); j < v_issued; j++) mbar_wait(v_full + 8 * (j % NS), (j / NS) & 1);
        }
    } else if (warp == 1) {
        if (any) {                                             // ---- scores: S = Q . K^T
            constexpr uint32_t idesc_s = idesc(KEYS, false);
            const bool leader = elect_one();
            const uint32_t q_addr = smem_u32(q_s), k_addr = smem_u32(k_s);
            int c[NT] = {};                                    // pages of each tile so far
            int i = 0, seg = 0;
            bool ok = true;
            do {
                const int n = u.pg1 - u.pg0, nt = NT == 1 || u.rows(a) <= tile_rows ? 1 : NT;
                ok = warp_wait(q_full, seg & 1);
                for (int j = 0; j < n && ok; j++, i++) {
                    const int st = i % NS;
                    ok = warp_wait(k_full + 8 * st, (i / NS) & 1);
#pragma unroll
                    for (int x = 0; x < NT; x++) {
                        if (x >= nt || !ok) break;
                        const int buf = c[x] & 1;
                        // the buffer held the weights of the page before the last
                        ok = c[x] < 2 || warp_wait(p_free + 8 * (2 * x + buf), ((c[x] >> 1) & 1) ^ 1);
                        if (!ok) break;
                        tc_fence_after();
                        if (leader) {
#pragma unroll
                            for (int k = 0; k < HD / 16; k++)
                                tc_mma(tmem_base + (2 * x + buf) * KEYS, desc_k_major(q_addr + x * Q_TILE + (k / 4) * HALF_BYTES + (k % 4) * 32),
                                       desc_k_major(k_addr + st * PAGE_TILE + (k / 4) * PAGE_BYTES + (k % 4) * 32), idesc_s, k != 0);
                            tc_commit(s_full + 8 * (2 * x + buf));
                        }
                        __syncwarp();
                        c[x]++;
                    }
                    if (!ok) break;
                    if (leader) {
                        tc_commit(k_free + 8 * st);
                        if (j + 1 == n) tc_commit(q_free);
                    }
                    __syncwarp();
                }
                seg++;
            } while (ok && u.next(cu_q, kv_len, pt, a, status));
            if (!ok && lane == 0) atomicOr(status, MYNAH_ST_TIMEOUT);
        }
    } else if (warp == 2) {
        if (any) {                                             // ---- outputs: O += P . V
            constexpr uint32_t idesc_o = idesc(HD, true);
            const bool leader = elect_one();
            const uint32_t v_addr = smem_u32(v_s);
            int c[NT] = {};
            int i = 0, seg = 0;
            bool ok = true;
            do {
                const int n = u.pg1 - u.pg0, nt = NT == 1 || u.rows(a) <= tile_rows ? 1 : NT;
                if (seg > 0) ok = warp_wait(o_free, (seg - 1) & 1);            // the segment before has been read out
                for (int j = 0; j < n && ok; j++, i++) {
                    const int st = i % NS;
                    ok = warp_wait(v_full + 8 * st, (i / NS) & 1);
#pragma unroll
                    for (int x = 0; x < NT; x++) {             // (the first tile's warps have looked through V before they hand over)
                        if (x >= nt || !ok) break;
                        const int buf = c[x] & 1;
                        ok = warp_wait(p_full + 8 * (2 * x + buf), (c[x] >> 1) & 1);
                        if (!ok) break;
                        tc_fence_after();
                        if (leader) {
#pragma unroll
                            for (int k = 0; k < KEYS / 16; k++)        // 16 keys a step: 8 columns of packed weights, 16 rows of V
                                tc_mma_ts(tmem_base + O_COL + x * HD, tmem_base + (2 * x + buf) * KEYS + k * 8,
                                          desc_mn_major(v_addr + st * PAGE_TILE + k * 16 * 128, PAGE_BYTES), idesc_o, (j | k) != 0);
                            tc_commit(p_free + 8 * (2 * x + buf));
                        }
                        __syncwarp();
                        c[x]++;
                    }
                    if (!ok) break;
                    if (leader) tc_commit(v_free + 8 * st);
                    __syncwarp();
                }
                seg++;
            } while (ok && u.next(cu_q, kv_len, pt, a, status));
            if (!ok && lane == 0) atomicOr(status, MYNAH_ST_TIMEOUT);
        }
    } else if (any) {
        // ---- softmax: a warp reads the lane quadrant (warp % 4) of tensor memory, a thread a row
        const int mine = (warp - 3) >> 2, quad = warp & 3, row = quad * 32 + lane;       // (of its own tile)
        const uint32_t t_row = tmem_base + ((uint32_t)(quad * 32) << 16) + mine * 2 * KEYS;
        const uint32_t t_o = tmem_base + ((uint32_t)(quad * 32) << 16) + O_COL + mine * HD;
        const uint32_t s_mine = s_full + 16 * mine, p_mine = p_full + 16 * mine, f_mine = p_free + 16 * mine;
        int i = 0, c_own = 0, seg = 0;
        bool ok = true;
        do {
            const int n = u.pg1 - u.pg0, past = u.past(), kvl = u.s.kvl;
            const int row0 = u.tile * a.tile_rows + mine * tile_rows, n_rows = max(0, min(tile_rows, u.rows(a) - mine * tile_rows));
            const bool there = NT == 1 || n_rows > 0, works = quad * 32 < n_rows;
            const int first_tok = a.by_G.div(u.tile * a.tile_rows), tok = a.by_G.div(row0 + row);            // of the sequence
            const long long* words = masks + (size_t)(u.s.q_begin + min(tok, u.s.n_q - 1)) * a.words;
            // Is there a key in the page that some row of the CTA must not see?
            auto masked = [&](int key0) { return key0 + KEYS > kvl || (CAUSAL ? key0 + KEYS - 1 > past + first_tok : key0 + KEYS > past); };
            float m_ref = -INFINITY, l = 0.f;                  // the maximum that the sums are scaled by; the sum
            for (int j = 0; j < n && ok && there; j++, i++, c_own++) {
                const int st = i % NS, key0 = (u.pg0 + j) * KEYS, buf = c_own & 1;
                const uint32_t t_s = t_row + buf * KEYS;
                const bool mask = masked(key0);
                if (!warp_wait(s_mine + 8 * buf, (c_own >> 1) & 1)) { ok = false; break; }
                tc_fence_after();
                if (works) {
                    float s[KEYS];
#pragma unroll
                    for (int c = 0; c < 2; c++) tc_ld32_nowait(t_s + c * 32, reinterpret_cast<uint32_t(&)[32]>(s[c * 32]));
#pragma unroll
                    for (int c = 0; c < 2; c++) tc_wait_ld(reinterpret_cast<uint32_t(&)[32]>(s[c * 32]));
                    if (mask) {
                        const unsigned long long vis = row < n_rows ? visible64<CAUSAL>(key0, kvl, past, tok, words, a.words) : 0ull;
                        const uint32_t v0 = (uint32_t)vis, v1 = (uint32_t)(vis >> 32);
#pragma unroll
                        for (int e = 0; e < 32; e++) {
                            s[e] = (v0 >> e) & 1u ? s[e] : -INFINITY;
                            s[32 + e] = (v1 >> e) & 1u ? s[32 + e] : -INFINITY;
                        }
                    }
                    const int entry = u.s.list0 + u.pg0 + j - u.s.first;       // of the page lists
                    if (CAUSAL && sc.scores != nullptr && row0 + row < sc.score_rows && row < n_rows && entry >= u.s.list0 && entry < min(u.s.list1, sc.entries)) {
                        // for the sums of the weights (one tile, of few rows)
                        float4* to = reinterpret_cast<float4*>(sc.scores + (((size_t)entry * a.KV + u.g) * sc.score_rows + row0 + row) * KEYS);
#pragma unroll
                        for (int e = 0; e < KEYS; e += 4)
                            to[e >> 2] = make_float4(s[e] * a.scale_log2, s[e + 1] * a.scale_log2, s[e + 2] * a.scale_log2, s[e + 3] * a.scale_log2);
                    }
                    float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                    for (int e = 0; e < KEYS; e += 2) mx4[(e >> 1) & 3] = max3(mx4[(e >> 1) & 3], s[e], s[e + 1]);
                    const float m_new = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])) * a.scale_log2;
                    // The reference follows the true maximum lazily: while that stays within 2^8 of it nothing is rescaled.
                    float alpha = 1.0f;
                    if (m_new > m_ref + 8.0f || (m_ref == -INFINITY && m_new != -INFINITY)) {
                        alpha = ex2_f(m_ref - m_new);          // 0 for the first seen key
                        m_ref = m_new;
                    }
                    const float m_use = m_ref == -INFINITY ? 0.f : m_ref;
                    // O is touched only when some row of the warp has to be rescaled; then the product of the page before must have
                    // finished. (That page's scores were issued behind the product of the page two before it, in the same buffer:
                    // the wait below cannot be answered by an older phase.)
                    if (j > 0 && __any_sync(0xffffffffu, alpha != 1.0f)) {
                        if (!warp_wait(f_mine + 8 * (buf ^ 1), ((c_own - 1) >> 1) & 1)) { ok = false; break; }
                        tc_fence_after();
#pragma unroll 1
                        for (int c = 0; c < HD / 32; c++) {
                            uint32_t r[32];
                            tc_ld32(t_o + c * 32, r);
#pragma unroll
                            for (int e = 0; e < 32; e++) r[e] = __float_as_uint(__uint_as_float(r[e]) * alpha);
                            tc_st32(t_o + c * 32, r);
                        }
                        tc_wait_st();
                    }
                    float sum4[4] = {0.f, 0.f, 0.f, 0.f};
                    uint32_t pk[KEYS / 2];
#pragma unroll
                    for (int e = 0; e < KEYS; e += 2) {
                        float x0, x1;
                        fma2(x0, x1, s[e], s[e + 1], a.scale_log2, -m_use);
                        const float p0 = ex2_f(x0), p1 = ex2_f(x1);               // 2^-inf = 0
                        add2(sum4[e & 2], sum4[(e & 2) + 1], p0, p1);
                        pk[e >> 1] = pack2(p0, p1);
                    }
                    tc_st32(t_s, pk);                          // over the scores, which are in registers
                    tc_wait_st();
                    l = l * alpha + ((sum4[0] + sum4[1]) + (sum4[2] + sum4[3]));
                }
                if (mask && mine == 0) {                       // look through V: a thread a key's row of 64 columns
                    if (!warp_wait(v_full + 8 * st, (i / NS) & 1)) { ok = false; break; }
                    const int key = row & 63, hf = row >> 6;
                    if (hf < HALVES) {
                        uint4* dst = reinterpret_cast<uint4*>(v_s + st * PAGE_TILE + hf * PAGE_BYTES + key * 128);
                        if (key0 + key >= kvl) {               // nobody's
#pragma unroll
                            for (int e = 0; e < 8; e++) dst[e] = make_uint4(0u, 0u, 0u, 0u);
                        } else {
#pragma unroll
                            for (int e = 0; e < 8; e++) {
                                uint4 x = dst[e];
                                const uint32_t n0 = not_finite2(x.x), n1 = not_finite2(x.y), n2 = not_finite2(x.z), n3 = not_finite2(x.w);
                                if (n0 | n1 | n2 | n3) {
                                    x.x &= ~n0, x.y &= ~n1, x.z &= ~n2, x.w &= ~n3;
                                    dst[e] = x;
                                    *(volatile int*)(flags + (seg & 1)) = seg + 1;
                                }
                            }
                        }
                    }
                    fence_async_smem();
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(p_mine + 8 * buf);
            }
            if (!there) i += n;
            asm volatile("bar.sync 1, %0;" ::"n"(128 * NT) : "memory");       // what any warp found in V is known to all
            if (ok && there && !warp_wait(f_mine + 8 * ((c_own - 1) & 1), ((c_own - 1) >> 1) & 1)) ok = false;      // the last page is in
            if (ok) {
                tc_fence_after();
                const bool poison = *(volatile int*)(flags + (seg & 1)) == seg + 1, lost = *(volatile int*)(flags + 2 + (seg & 7)) == seg + 1;
                const bool whole = u.whole();
                if (lost) m_ref = -INFINITY, l = 0.f;          // a page was missing: nothing counts
                const float inv = whole ? (l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l)) : 1.f;      // a NaN stays one
                const long long slot0 = whole ? 0 : u.scratch_row(a) + mine * tile_rows;         // of the tile
                if (works) {
                    const uint32_t mine_s = smem_u32(stage_s) + (warp - 3) * 32 * STAGE_PITCH * 4;     // this warp's rows, 16 columns at a time
                    const int rows_here = min(32, n_rows - quad * 32);
                    // where the four rows that this lane writes a part of begin (four lanes a row, 4 of 16 columns each)
                    size_t to[4];
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const int pr = row0 + quad * 32 + e * 8 + (lane >> 2), tk = a.by_G.div(pr);
                        to[e] = (whole ? (size_t)(u.s.q_begin + tk) * a.ldo + (size_t)(u.g * a.G + pr - tk * a.G) * HD
                                       : (size_t)(slot0 + quad * 32 + e * 8 + (lane >> 2)) * HD) + (lane & 3) * 4;
                    }
                    // 64 columns at a time out of tensor memory (one wait for all), 16 at a time through shared memory
#pragma unroll 1
                    for (int c = 0; c < HD / 64; c++) {
                        uint32_t r[64];
                        tc_ld32_nowait(t_o + c * 64, reinterpret_cast<uint32_t(&)[32]>(r[0]));
                        tc_ld32_nowait(t_o + c * 64 + 32, reinterpret_cast<uint32_t(&)[32]>(r[32]));
                        tc_wait_ld(reinterpret_cast<uint32_t(&)[32]>(r[0]));
                        tc_wait_ld(reinterpret_cast<uint32_t(&)[32]>(r[32]));
                        if (poison && !lost && row < n_rows) { // the values that were zeroed, to the rows that see them
#pragma unroll 1
                            for (int key = u.pg0 * KEYS; key < min(u.pg1 * KEYS, kvl); key++) {
                                if (!masked(key & ~63) || !((visible64<CAUSAL>(key & ~63, kvl, past, tok, words, a.words) >> (key & 63)) & 1ull)) continue;
                                const bf16* vr = v_cache + (((size_t)page_at(pt, u.s, key / PAGE_TOKENS) * a.KV + u.g) * PAGE_TOKENS + key % PAGE_TOKENS) * HD + c * 64;
#pragma unroll
                                for (int e = 0; e < 64; e++) {
                                    const float x = __bfloat162float(vr[e]);
                                    if (!isfinite(x)) r[e] = __float_as_uint(__uint_as_float(r[e]) + x);
                                }
                            }
                        }
                        __syncwarp();
#pragma unroll
                        for (int f = 0; f < 4; f++) {
#pragma unroll
                            for (int e = 0; e < 4; e++) {
                                float v[4];
#pragma unroll
                                for (int d = 0; d < 4; d++) v[d] = lost ? 0.f : __uint_as_float(r[16 * f + 4 * e + d]) * inv;
                                st_shared(mine_s + (lane * STAGE_PITCH + 4 * e) * 4, make_float4(v[0], v[1], v[2], v[3]));
                            }
                            __syncwarp();
#pragma unroll
                            for (int e = 0; e < 4; e++) {
                                const int rr = e * 8 + (lane >> 2);
                                const float4 x = ld_shared(mine_s + (rr * STAGE_PITCH + (lane & 3) * 4) * 4);
                                if (rr < rows_here) {
                                    if (whole) *reinterpret_cast<uint2*>(out + to[e] + c * 64 + f * 16) = make_uint2(pack2(x.x, x.y), pack2(x.z, x.w));
                                    else *reinterpret_cast<float4*>(sc.o + to[e] + c * 64 + f * 16) = x;
                                }
                            }
                            __syncwarp();                      // (before the next columns go over these)
                        }
                    }
                    if (row < n_rows) {
                        if (!whole) sc.ml[slot0 + row] = make_float2(m_ref, l);
                        else if (CAUSAL) sc.lse[((size_t)u.g * a.T + u.s.q_begin) * a.G + row0 + row] = l == 0.f ? -INFINITY : m_ref + log2f(l);
                    }
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(o_free);
            }
            seg++;
        } while (u.next(cu_q, kv_len, pt, a, status));             // (a warp that has given up goes on to keep the others' barriers)
        if (!ok && lane == 0) atomicOr(status, MYNAH_ST_TIMEOUT);
    }
    griddep_launch_late();
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(TMEM_COLS) : "memory");
    }
}

template <int HD, int NT, bool CAUSAL>
int go(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, const void* v, const int* cu_q, const int* kv_len, PageTable pt,
       const long long* masks, const RowsArgs& a, void* out, RowsScratch s, int* status, cudaStream_t stream) {
    constexpr size_t smem = (size_t)(HD / 64) * (NT * HALF_BYTES + 2 * STAGES<HD, NT> * PAGE_BYTES) + NT * 4 * 32 * STAGE_PITCH * 4 + 448 + 1024;
    auto kern = attn_rows_tcgen05_kernel<HD, NT, CAUSAL>;
    static std::atomic<unsigned long long> opted{0};
    const cudaError_t e = shared_memory_once(kern, smem, opted);
    if (e != cudaSuccess) return mynah_fail("attn_rows: %s", cudaGetErrorString(e));
    kern<<<a.ctas * a.group, 96 + 128 * NT, smem, stream>>>(mq, mk, mv, (const bf16*)v, cu_q, kv_len, pt, masks, a, (bf16*)out, s, status);
    return mynah_check_launch("attn_rows");
}

}  // namespace

bool rows_tcgen05_takes(int dtype, int H, int KV, int HD) {
    return dtype == MYNAH_BF16 && (HD == 64 || HD == 128) && KV > 0 && H % KV == 0 && H / KV <= BQ;
}

int launch_rows_tcgen05(const void* q, void* out, const RowsArgs& a, const void* k, const void* v, const int* cu_q,
                        const int* kv_len, PageTable pt, const long long* masks, RowsScratch s, int* status, cudaStream_t stream) {
    const long long rows = (long long)pt.n_pages * a.KV * PAGE_TOKENS;
    MYNAH_REQUIRE(rows < (1ll << 31), "attn_rows: launch too large");
    if (pt.n_pages == 0) return mynah_fail("attn_rows: a cache without pages");
    CUtensorMap mq, mk, mv;
    if (make_map_rows(&mq, q, a.T, a.H, a.HD, a.G, a.ldq, a.tile_rows / (a.two ? 2 : 1) / a.G)) return -1;
    if (make_map(&mk, k, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, rows, a.HD, a.HD, PAGE_TOKENS, 64)) return -1;
    if (make_map(&mv, v, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, rows, a.HD, a.HD, PAGE_TOKENS, 64)) return -1;
#define ROWS_GO(HD, NT) return (a.causal ? go<HD, NT, true> : go<HD, NT, false>)(mq, mk, mv, v, cu_q, kv_len, pt, masks, a, out, s, status, stream)
    if (a.two) {
        if (a.HD == 128) ROWS_GO(128, 2);
        ROWS_GO(64, 2);
    }
    if (a.HD == 128) ROWS_GO(128, 1);
    ROWS_GO(64, 1);
#undef ROWS_GO
}
