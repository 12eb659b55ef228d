// The sums of attention weights (attn_mass.cu) on the fifth-generation tensor cores, for bfloat16 heads of 64 and 128.
//
// The products are taken transposed, S^T = K.Q^T with 128 keys as the rows of the accumulator and up to 128 packed rows as its
// columns: a key is then a lane of tensor memory, and its sum stays in one thread's register (two threads a key, one for each
// half of the columns) without any exchange between lanes. w = 2^(s scale log2(e) - lse) needs one multiply-add, one
// exponential and one addition an element; the exponentials (16 a clock and SM) bound it: a product of 128 x 128 scores takes an
// SM 1,024 clocks of them, measured 1,600 in long prompts (8,000 tokens of 32 heads, 370 us; with the selects of masked tiles in
// every tile 424; a quarter of the exponentials as polynomials 342, not kept for their range and size). 2,048 tokens of 16 heads
// are 34 million scores, 7.5 us, and take 30: units of unequal length, and 4 us until a CTA's first product.
//
//   warp 0      one lane loads by TMA: one operand stays (a key tile against many row tiles, or a sequence's only row tile
//               against several key tiles), the other streams through two stages;
//   warp 1      one lane issues the products into two accumulators;
//   warps 2-9   the sums;
//   warp 10     brings the row tile's lse values into shared memory.
//
// Two CTAs an SM (96 KB of tiles, 256 columns of tensor memory each), so that one's start and end run under the other's work.
// Every wait is bounded; one that runs out sets MYNAH_ST_TIMEOUT.
#include "attn_mass.cuh"
#include "rows_tcgen05.cuh"

namespace {

using namespace tc5;

constexpr int THREADS = 352;
constexpr int KEYS = 128, ROWS = 128;

template <int HD>
__global__ void __launch_bounds__(THREADS, 2)
attn_mass_tcgen05_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, const float* __restrict__ lse,
                         float* __restrict__ mass, float* __restrict__ part, const int* __restrict__ cu_q, const int* __restrict__ kv_len,
                         PageTable pt, MassArgs a, int* __restrict__ status) {
    constexpr int HALVES = HD / 64;
    constexpr int TILE_BYTES = HALVES * HALF_BYTES;
    constexpr int TMEM_COLS = 256;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    unsigned char* fix_s = smem;                               // the operand that stays
    unsigned char* str_s = smem + TILE_BYTES;                  // [2] the one that streams
    float* lse_s = reinterpret_cast<float*>(str_s + 2 * TILE_BYTES);       // [2][ROWS] minus the rows' lse
    float* xch = lse_s + 2 * ROWS;                             // [2][KEYS] the second group's sums
    uint64_t* bars = reinterpret_cast<uint64_t*>(xch + 2 * KEYS);
    const uint32_t f_full = smem_u32(bars), s_full = smem_u32(bars + 1), d_full = smem_u32(bars + 3), d_free = smem_u32(bars + 5);
    const uint32_t l_full = smem_u32(bars + 7);                // [2] each but the first
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 9);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    MassUnit u;
    const bool any = find_mass_unit(cu_q, kv_len, pt, a, blockIdx.x / a.r.KV, u, status);
    griddep_wait();
    if (!any) return;
    const int g = blockIdx.x % a.r.KV, G = a.r.G, past = u.s.kvl - u.s.n_q, n_rows = u.s.n_q * G;
    const int r0 = max(u.piece * u.rt, a.by_keys ? 0 : mass_first_tile(u, a));
    const int r1 = (int)min((long long)mass_rtiles(u.s, a), (long long)(u.piece + 1) * u.rt);
    if (r0 >= r1) return;                                      // no token of this piece sees the keys
    const int n = a.by_keys ? u.kt1 - u.kt0 : r1 - r0;         // products of this unit
    auto ktile = [&](int i) { return a.by_keys ? u.kt0 + i : u.kt0; };
    auto rtile = [&](int i) { return a.by_keys ? 0 : r0 + i; };

    if (threadIdx.x == 0) {
        mbar_init(f_full, 1);
        for (int i = 0; i < 2; i++) {
            mbar_init(s_full + 8 * i, 1);
            mbar_init(d_full + 8 * i, 1);
            mbar_init(d_free + 8 * i, 8);
            mbar_init(l_full + 8 * i, 1);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    // Rows of a query tile that no box fills (128 is no multiple of G) are zero: their scores are finite, their lse is infinite.
    if (a.rows < ROWS) {
        const int tail = (ROWS - a.rows) * 8;                  // 16-byte pieces a half
        for (int i = threadIdx.x; i < 3 * HALVES * tail; i += THREADS)
            reinterpret_cast<uint4*>(smem + (i / tail) * HALF_BYTES + a.rows * 128)[i % tail] = make_uint4(0u, 0u, 0u, 0u);
    }
    fence_async_smem();
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;

    if (warp == 0) {
        if (lane == 0) {                                       // ---- TMA producer
            auto bring_k = [&](unsigned char* dst, int kt, uint32_t bar) {
                const int key0 = kt * KEYS;
                const bool two = key0 + PAGE_TOKENS < u.s.kvl;
                int p0 = page_of(pt, u.b, key0), p1 = two ? page_of(pt, u.b, key0 + PAGE_TOKENS) : 0;
                if (p0 < 0 || p1 < 0) {                        // (such keys have no place to put their sums either)
                    atomicOr(status, MYNAH_ST_PAGE_RANGE);
                    p0 = max(p0, 0), p1 = max(p1, 0);
                }
                mbar_expect_tx(bar, (two ? 2 : 1) * HALVES * PAGE_BYTES);
#pragma unroll
                for (int hf = 0; hf < HALVES; hf++) {
                    tma_load_2d(smem_u32(dst + hf * HALF_BYTES), &map_k, hf * 64, (p0 * a.r.KV + g) * PAGE_TOKENS, bar);
                    if (two) tma_load_2d(smem_u32(dst + hf * HALF_BYTES + PAGE_BYTES), &map_k, hf * 64, (p1 * a.r.KV + g) * PAGE_TOKENS, bar);
                }
            };
            auto bring_q = [&](unsigned char* dst, int rt, uint32_t bar) {
                mbar_expect_tx(bar, HALVES * a.rows * 128);
#pragma unroll
                for (int hf = 0; hf < HALVES; hf++)
                    tma_load_3d(smem_u32(dst + hf * HALF_BYTES), &map_q, hf * 64, g * G, u.s.q_begin + rt * (a.rows / G), bar);
            };
            if (a.by_keys) bring_q(fix_s, 0, f_full);
            else bring_k(fix_s, u.kt0, f_full);
            int issued = 0;
            for (int i = 0; i < n; i++) {
                const int st = i & 1;
                if (i >= 2 && !mbar_wait(d_full + 8 * st, ((i >> 1) & 1) ^ 1)) {     // product i - 2 is done: its stage is free
                    atomicOr(status, MYNAH_ST_TIMEOUT);
                    break;
                }
                if (a.by_keys) bring_k(str_s + st * TILE_BYTES, ktile(i), s_full + 8 * st);
                else bring_q(str_s + st * TILE_BYTES, rtile(i), s_full + 8 * st);
                issued = i + 1;
            }
            mbar_wait(f_full, 0);                              // nothing may land after this CTA has left
            for (int i = max(0, issued - 2); i < issued; i++) mbar_wait(s_full + 8 * (i & 1), (i >> 1) & 1);
        }
    } else if (warp == 1) {
        // ---- MMA issuer (the whole warp runs, one elected lane issues: see attn_rows_tcgen05.cu)
        constexpr uint32_t idesc_s = idesc(ROWS, false);
        const bool leader = elect_one();
        const uint32_t fix = smem_u32(fix_s), str = smem_u32(str_s);
        bool ok = warp_wait(f_full, 0);
        for (int i = 0; i < n && ok; i++) {
            const int st = i & 1;
            ok = warp_wait(s_full + 8 * st, (i >> 1) & 1) && (i < 2 || warp_wait(d_free + 8 * st, ((i >> 1) & 1) ^ 1));
            if (!ok) break;
            tc_fence_after();
            const uint32_t k_addr = a.by_keys ? str + st * TILE_BYTES : fix, q_addr = a.by_keys ? fix : str + st * TILE_BYTES;
            if (leader) {
#pragma unroll
                for (int k = 0; k < HD / 16; k++) {
                    const uint32_t off = (k / 4) * HALF_BYTES + (k % 4) * 32;
                    tc_mma(tmem_base + st * ROWS, desc_k_major(k_addr + off), desc_k_major(q_addr + off), idesc_s, k != 0);
                }
                tc_commit(d_full + 8 * st);
            }
            __syncwarp();
        }
        if (!ok && lane == 0) atomicOr(status, MYNAH_ST_TIMEOUT);
    } else if (warp == 10) {                                   // ---- lse
        bool ok = true;
        for (int i = 0; i < n && ok; i++) {
            const int st = i & 1;
            if (i >= 2) ok = warp_wait(d_free + 8 * st, ((i >> 1) & 1) ^ 1);
            if (!ok) break;
            const int row0 = rtile(i) * a.rows;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int r = e * 32 + lane;
                float x = INFINITY;
                if (r < a.rows && row0 + r < n_rows) x = lse[((size_t)g * a.r.T + u.s.q_begin) * G + row0 + r];
                lse_s[st * ROWS + r] = x == -INFINITY ? -INFINITY : -x;
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(l_full + 8 * st);
        }
        if (!ok && lane == 0) atomicOr(status, MYNAH_ST_TIMEOUT);
    } else {
        // ---- sums: a thread a key and half of the columns
        const int grp = (warp - 2) >> 2, quad = warp & 3, key = quad * 32 + lane;
        const uint32_t t_row = tmem_base + ((uint32_t)(quad * 32) << 16) + grp * 64;
        float sum4[4] = {0.f, 0.f, 0.f, 0.f};
        bool ok = true;
        int flushes = 0;
        for (int i = 0; i < n; i++) {
            const int st = i & 1;
            const uint32_t use = (i >> 1) & 1;
            if (ok && !(warp_wait(l_full + 8 * st, use) && warp_wait(d_full + 8 * st, use))) ok = false;
            const int pos = ktile(i) * KEYS + key;             // the key's row in the sequence
            if (ok) {
                tc_fence_after();
                const int row0 = rtile(i) * a.rows;
                // the columns that see this key: from its own token's first on, up to the sequence's last row
                const int lo = max(0, pos - past) * G - row0 - grp * 64, hi = min(n_rows - row0, a.rows) - grp * 64;
                const bool mask = max(0, ktile(i) * KEYS + KEYS - 1 - past) * G > row0 || n_rows - row0 < a.rows;
#pragma unroll
                for (int c = 0; c < 2; c++) {
                    float w[32];
                    tc_ld32(t_row + st * ROWS + c * 32, reinterpret_cast<uint32_t(&)[32]>(w));
                    const float4* z4 = reinterpret_cast<const float4*>(lse_s + st * ROWS + grp * 64 + c * 32);
                    if (!mask) {
#pragma unroll
                        for (int e = 0; e < 32; e += 4) {
                            const float4 z = z4[e >> 2];
                            float x[4];
                            fma2v(x[0], x[1], w[e], w[e + 1], a.r.scale_log2, z.x, z.y);
                            fma2v(x[2], x[3], w[e + 2], w[e + 3], a.r.scale_log2, z.z, z.w);
                            add2(sum4[0], sum4[1], ex2_f(x[0]), ex2_f(x[1]));
                            add2(sum4[2], sum4[3], ex2_f(x[2]), ex2_f(x[3]));
                        }
                    } else {
#pragma unroll
                        for (int e = 0; e < 32; e += 4) {
                            const float4 z = z4[e >> 2];
                            float x[4];
                            fma2v(x[0], x[1], w[e], w[e + 1], a.r.scale_log2, z.x, z.y);
                            fma2v(x[2], x[3], w[e + 2], w[e + 3], a.r.scale_log2, z.z, z.w);
#pragma unroll
                            for (int f = 0; f < 4; f++) x[f] = (c * 32 + e + f >= lo && c * 32 + e + f < hi) ? ex2_f(x[f]) : 0.f;
                            add2(sum4[0], sum4[1], x[0], x[1]);
                            add2(sum4[2], sum4[3], x[2], x[3]);
                        }
                    }
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(d_free + 8 * st);
            }
            if (a.by_keys || i + 1 == n) {                     // the key's sum is whole: both groups' halves together
                const float sum = (sum4[0] + sum4[1]) + (sum4[2] + sum4[3]);
                float* x = xch + (flushes & 1) * KEYS;         // (two buffers: read before the next barrier, written behind it)
                flushes++;
                if (grp == 1) x[key] = sum;
                asm volatile("bar.sync 1, 256;" ::: "memory");
                if (grp == 0 && ok && pos < u.s.kvl) {
                    if (u.pieces > 1) {
                        part[(long long)blockIdx.x * KEYS + key] = sum + x[key];
                    } else {
                        const long long at = mass_at(pt, u.b, pos, a.r.KV, g);
                        if (at >= 0) mass[at] = (pos < past ? mass[at] : 0.f) + (sum + x[key]);
                    }
                }
#pragma unroll
                for (int e = 0; e < 4; e++) sum4[e] = 0.f;
            }
        }
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

template <int HD>
int go(const CUtensorMap& mq, const CUtensorMap& mk, const float* lse, float* mass, float* part, const int* cu_q, const int* kv_len,
       PageTable pt, const MassArgs& a, int n_ids, int* status, cudaStream_t stream) {
    constexpr size_t smem = 3 * (size_t)(HD / 64) * HALF_BYTES + 4 * 128 * sizeof(float) + 80 + 1024;
    auto kern = attn_mass_tcgen05_kernel<HD>;
    static std::atomic<unsigned long long> opted{0};
    const cudaError_t e = shared_memory_once(kern, smem, opted);
    if (e != cudaSuccess) return mynah_fail("attn_mass: %s", cudaGetErrorString(e));
    const dim3 grid((unsigned)(mass_units_max(a, n_ids) * a.r.KV));
    const cudaError_t err = launch_behind(kern, grid, dim3(THREADS), smem, stream, mq, mk, lse, mass, part, cu_q, kv_len, pt, a, status);
    if (err != cudaSuccess) return mynah_fail("attn_mass: %s", cudaGetErrorString(err));
    return mynah_check_launch("attn_mass");
}

}  // namespace

bool mass_tcgen05_takes(int dtype, int H, int KV, int HD) { return rows_tcgen05_takes(dtype, H, KV, HD); }

int launch_mass_tcgen05(const void* q, const void* k, const float* lse, float* mass, float* part, const int* cu_q, const int* kv_len,
                        PageTable pt, const MassArgs& a, int n_ids, int* status, cudaStream_t stream) {
    const long long rows = (long long)pt.n_pages * a.r.KV * PAGE_TOKENS;
    MYNAH_REQUIRE(rows < (1ll << 31) && pt.n_pages > 0, "attn_mass: launch too large");
    CUtensorMap mq, mk;
    if (make_map_rows(&mq, q, a.r.T, a.r.H, a.r.HD, a.r.G, a.r.ldq, a.rows / a.r.G)) return -1;
    if (make_map(&mk, k, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, rows, a.r.HD, a.r.HD, PAGE_TOKENS, 64)) return -1;
    if (a.r.HD == 128) return go<128>(mq, mk, lse, mass, part, cu_q, kv_len, pt, a, n_ids, status, stream);
    return go<64>(mq, mk, lse, mass, part, cu_q, kv_len, pt, a, n_ids, status, stream);
}
