// Causal attention that also adds up, for every cached row and kv head, the softmax weight that the step's tokens give it: what
// an eviction by accumulated attention weight goes by.
//
//   mass[r, g] = (r < past ? mass[r, g] : 0) + sum_i sum_{h of g} w_ihr        (w as in attn_rows.cu, r <= past + i)
//
// The attention itself is that of attn_rows.cu and leaves log2 of every row's sum, lse_ih. With it a weight needs no second
// softmax: w_ihr = 2^(scale log2(e) q_ih . k_gr - lse_ih), so the sums take one more look at the keys alone, with the keys as
// the resident operand and the step's packed rows going by: a key's sum stays with its thread, no two CTAs add to the same
// word, and the order of the sum does not depend on timing. Sums are fp32.
//
// Long sequences are cut over their rows too (attn_mass.cuh): the cut pieces' sums are left in scratch and added in order by a
// second launch. Steps of few rows on the tensor cores do not look at the keys again: the attention keeps its scores, and the
// launch that joins its segments adds them up (sum_scores in attn_rows.cu). This file holds the general kernel (fp32, and bfloat16
// heads that the tensor-core kernel does not take: 2 pieces of 150 tokens behind 333 rows, 6 heads of 48 on 3, 10 us of 37, bound
// by its launches and its FFMA fed from shared memory), the addition of pieces and the entry points.
#include "attn_mass.cuh"

#include <math.h>

int attn_rows_run(const char* who, const void* q, void* out, int dtype, RowsArgs a, int max_q_len, const void* k_cache, const void* v_cache,
                  const int* cu_q, const int* kv_len, PageTable pt, const long long* masks, float* scratch, long long scratch_floats,
                  float* lse, float* scores, int score_rows, int n_ids, float* mass, int* status, cudaStream_t stream);

namespace {

constexpr int GK = 64, GR = 32;      // keys (a page) and packed rows a tile of the general kernel

// 16 x 16 threads; thread (ty, tx) has the keys ty + 16 i (i < 4) of the page and the rows tx + 16 j of a tile.
template <typename T>
__global__ void __launch_bounds__(256)
attn_mass_kernel(const T* __restrict__ q, const T* __restrict__ k_cache, const float* __restrict__ lse, float* __restrict__ mass,
                 float* __restrict__ part, const int* __restrict__ cu_q, const int* __restrict__ kv_len, PageTable pt, MassArgs a,
                 int* __restrict__ status) {
    extern __shared__ __align__(16) unsigned char smem_mass[];
    const int HD = a.r.HD, p = HD + 4;
    float* k_s = reinterpret_cast<float*>(smem_mass);              // [GK][p]
    float* q_s = k_s + GK * p;                                     // [GR][p]
    __shared__ float lse_s[GR];
    MassUnit u;
    const bool any = find_mass_unit(cu_q, kv_len, pt, a, blockIdx.x, u, status);
    griddep_wait();
    if (!any) return;
    const int g = blockIdx.y, G = a.r.G, past = u.s.kvl - u.s.n_q, key0 = u.kt0 * GK, n_rows = u.s.n_q * G;
    const int tiles = mass_rtiles(u.s, a);
    const int r0 = max(u.piece * u.rt, mass_first_tile(u, a)), r1 = (int)min((long long)tiles, (long long)(u.piece + 1) * u.rt);
    if (r0 >= r1) return;                                          // no token of this piece sees the page
    const int page = page_of(pt, u.b, key0);
    if (page < 0) {
        if (threadIdx.x == 0) atomicOr(status, MYNAH_ST_PAGE_RANGE);
        return;
    }
    const T* k = k_cache + ((size_t)page * a.r.KV + g) * PAGE_TOKENS * HD;
    const int quads = HD >> 2;
    for (int i = threadIdx.x; i < GK * quads; i += 256) {
        const int r = a.r.by_quads.div(i);
        *reinterpret_cast<float4*>(k_s + r * p + (i - r * quads) * 4) = four_of(k + i * 4);
    }
    const int ty = threadIdx.x >> 4, tx = threadIdx.x & 15;
    float sum[4] = {0.f, 0.f, 0.f, 0.f};
    for (int rt = r0; rt < r1; rt++) {
        __syncthreads();
#pragma unroll 2
        for (int i = threadIdx.x; i < GR * quads; i += 256) {
            const int r = a.r.by_quads.div(i), d = (i - r * quads) * 4, pr = rt * GR + r, tok = a.r.by_G.div(pr);
            float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
            if (pr < n_rows) {
                const T* at = q + (size_t)(u.s.q_begin + tok) * a.r.ldq + (size_t)(g * G + pr - tok * G) * HD + d;
                x = a.r.q_aligned ? four_of(at) : four_apart(at);
            }
            *reinterpret_cast<float4*>(q_s + r * p + d) = x;
        }
        if (threadIdx.x < GR) {
            const int pr = rt * GR + threadIdx.x;
            const float z = pr < n_rows ? lse[((size_t)g * a.r.T + u.s.q_begin) * G + pr] : 0.f;
            lse_s[threadIdx.x] = z == -INFINITY ? INFINITY : z;    // a row that saw nothing gives no weight
        }
        __syncthreads();
        float s[4][2];
#pragma unroll
        for (int i = 0; i < 4; i++) s[i][0] = s[i][1] = 0.f;
#pragma unroll 4
        for (int d = 0; d < HD; d += 4) {
            const float4 q0 = four_of(q_s + tx * p + d), q1 = four_of(q_s + (tx + 16) * p + d);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float4 kv = four_of(k_s + (ty + 16 * i) * p + d);
                s[i][0] = fmaf(q0.x, kv.x, s[i][0]);
                s[i][0] = fmaf(q0.y, kv.y, s[i][0]);
                s[i][0] = fmaf(q0.z, kv.z, s[i][0]);
                s[i][0] = fmaf(q0.w, kv.w, s[i][0]);
                s[i][1] = fmaf(q1.x, kv.x, s[i][1]);
                s[i][1] = fmaf(q1.y, kv.y, s[i][1]);
                s[i][1] = fmaf(q1.z, kv.z, s[i][1]);
                s[i][1] = fmaf(q1.w, kv.w, s[i][1]);
            }
        }
#pragma unroll
        for (int j = 0; j < 2; j++) {
            const int r = tx + 16 * j, pr = rt * GR + r;
            if (pr >= n_rows) continue;
            const int last = past + a.r.by_G.div(pr);                        // the last key that the row sees
            const float z = lse_s[r];
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (key0 + ty + 16 * i <= last) sum[i] += exp2f(fmaf(s[i][j], a.r.scale_log2, -z));
        }
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], o);
        const int key = key0 + ty + 16 * i;
        if (tx != 0 || key >= u.s.kvl) continue;
        if (u.pieces > 1) {
            part[((long long)blockIdx.x * a.r.KV + g) * GK + ty + 16 * i] = sum[i];
        } else {
            float* m = mass + ((size_t)page * a.r.KV + g) * PAGE_TOKENS + ty + 16 * i;
            *m = key < past ? *m + sum[i] : sum[i];
        }
    }
    griddep_launch_late();
}

// Adds the pieces of every key's sum in order. A thread a key of a key tile; key tiles are numbered sequence by sequence.
__global__ void attn_mass_add_kernel(float* __restrict__ mass, const float* __restrict__ part, const int* __restrict__ cu_q,
                                     const int* __restrict__ kv_len, PageTable pt, MassArgs a, int* __restrict__ status) {
    MassUnit u;
    // the units of key tile n of the step: unit numbers are found as the first launch's were, from the tile's first piece on
    const bool any = find_mass_unit(cu_q, kv_len, pt, a, blockIdx.x, u, status);
    griddep_wait();
    if (!any) return;
    if (u.piece != 0 || u.pieces <= 1) return;                     // one CTA a key tile; uncut tiles are done
    const int g = blockIdx.y, past = u.s.kvl - u.s.n_q, key = u.kt0 * a.keys + threadIdx.x;
    if (threadIdx.x >= a.keys || key >= u.s.kvl) return;
    const long long at = mass_at(pt, u.b, key, a.r.KV, g);
    if (at < 0) return;                                            // reported by the first launch
    float sum = key < past ? mass[at] : 0.f;
    const int first = mass_first_tile(u, a);
    for (int c = first / u.rt; c < u.pieces; c++) sum += part[((long long)(blockIdx.x + c) * a.r.KV + g) * a.keys + threadIdx.x];
    mass[at] = sum;
}

int launch_mass_generic(const void* q, const void* k, const float* lse, float* mass, float* part, int dtype, const int* cu_q,
                        const int* kv_len, PageTable pt, const MassArgs& a, dim3 grid, int* status, cudaStream_t stream) {
    const size_t smem = (size_t)(GK + GR) * (a.r.HD + 4) * sizeof(float);
    auto kf = attn_mass_kernel<float>;
    auto kb = attn_mass_kernel<bf16>;
    static std::atomic<unsigned long long> opted_f{0}, opted_b{0};
    constexpr size_t most = (size_t)(GK + GR) * (256 + 4) * sizeof(float);
    cudaError_t e = dtype == MYNAH_F32 ? shared_memory_once(kf, most, opted_f) : shared_memory_once(kb, most, opted_b);
    if (e == cudaSuccess)
        e = dtype == MYNAH_F32 ? launch_behind(kf, grid, dim3(256), smem, stream, (const float*)q, (const float*)k, lse, mass, part, cu_q, kv_len, pt, a, status)
                               : launch_behind(kb, grid, dim3(256), smem, stream, (const bf16*)q, (const bf16*)k, lse, mass, part, cu_q, kv_len, pt, a, status);
    if (e != cudaSuccess) return mynah_fail("attn_mass: %s", cudaGetErrorString(e));
    return mynah_check_launch("attn_mass");
}

// Rows of a kv head up to which the attention keeps its scores for the sums rather than having the keys looked at again: they are
// 256 bytes a row and page written and read, the keys of 128 columns 16 KB.
constexpr int SCORE_ROWS = 8;

// Which kernel takes the sums, and its tiles.
bool mass_plan(MassArgs& a, int dtype, bool aligned, int max_q_len) {
    const bool tc = aligned && mass_tcgen05_takes(dtype, a.r.H, a.r.KV, a.r.HD);
    a.keys = tc ? 128 : GK;
    a.rows = tc ? 128 / a.r.G * a.r.G : GR;
    a.by_keys = (long long)max_q_len * a.r.G <= a.rows;
    a.own_pieces = tc ? 0 : 16;                                    // (2 pieces of 150, 10 row tiles each: 35.4 us with 16, 38.2 with 8, 39.0 with 4)
    a.r.most_q = max_q_len;
    a.r.tile_rows = a.rows;
    a.r.group = a.r.ctas = 1;
    a.r.q_aligned = aligned;
    a.r.finish();
    a.target = tc ? 4 * mynah_sm_count() : 0;
    a.score_rows = tc && (long long)max_q_len * a.r.G <= SCORE_ROWS ? max_q_len * a.r.G : 0;
    return tc;
}

long long mass_scratch(const MassArgs& a, int n_ids) {
    const long long lse = ((long long)a.r.T * a.r.H + 3) & ~3ll;
    if (a.score_rows > 0) return lse + (long long)n_ids * a.r.KV * a.score_rows * PAGE_TOKENS;
    return lse + (a.by_keys ? 0 : mass_units_max(a, n_ids) * a.r.KV * a.keys);
}

}  // namespace

long long attn_rows_scratch_floats(int T, int B, int max_q_len, int H, int KV, int HD, int dtype, int causal, int n_ids, int aligned);

// Floats of scratch for mynah_attn_mass. aligned: q's and the output's rows are 16-byte aligned (1) or not (0), which decides what
// takes the call; -1: enough for either.
MYNAH_API long long mynah_attn_mass_scratch_floats(int T, int B, int max_q_len, int H, int KV, int HD, int dtype, int n_ids, int aligned) {
    if (T <= 0 || B <= 0 || KV <= 0 || H % KV != 0 || H <= 0 || HD <= 0) return 0;
    long long need = 0;
    for (int al = 0; al < 2; al++) {
        if (aligned >= 0 && al != aligned) continue;
        MassArgs a{};
        a.r.T = T, a.r.B = B, a.r.H = H, a.r.KV = KV, a.r.HD = HD, a.r.G = H / KV;
        mass_plan(a, dtype, al != 0, max_q_len);
        const long long n = mass_scratch(a, n_ids);
        if (n > need) need = n;
    }
    return attn_rows_scratch_floats(T, B, max_q_len, H, KV, HD, dtype, 1, n_ids, aligned) + need;
}

// As mynah_attn_tree with causal rows, and mass [n_pages, KV, 64] fp32. n_ids: entries of page_ids (no fewer than the
// sequences' pages together). A sequence of more than max_q_len rows is refused through the status word.
struct AttnMassCall {
    const void* q;
    void* out;
    float* mass;
    int dtype, T, B, max_q_len, H, KV, HD, ldq, ldo;
    const void *k_cache, *v_cache;
    const int *cu_q, *kv_len, *page_indptr, *page_ids, *page_base;
    int n_pages, n_ids;
    float scale;
    float* scratch;
    long long scratch_floats;
    int* status;
    cudaStream_t stream;
};
static_assert(sizeof(AttnMassCall) == 168, "as packed by the caller");
MYNAH_API int mynah_attn_mass(const AttnMassCall* call) {
    const auto& [q, out, mass, dtype, T, B, max_q_len, H, KV, HD, ldq, ldo, k_cache, v_cache, cu_q, kv_len, page_indptr, page_ids, page_base,
                 n_pages, n_ids, scale, scratch, scratch_floats, status, stream] = *call;
    if (T <= 0 || B <= 0) return 0;
    MYNAH_REQUIRE(mass != nullptr && n_ids >= 0, "attn_mass: sums and the number of page entries are required");
    MYNAH_REQUIRE(scale == 0.f || (scale >= 0x1p-120f && scale <= 0x1p120f), "attn_mass: the score scale %g is not between 2^-120 and 2^120, nor 0", scale);
    MYNAH_REQUIRE(KV > 0 && H > 0 && H % KV == 0, "attn_mass: %d heads over %d kv heads", H, KV);
    MYNAH_REQUIRE(scratch != nullptr && ((uintptr_t)scratch & 15) == 0, "attn_mass: 16-byte aligned scratch is required");
    RowsArgs r{};
    r.T = T, r.B = B, r.H = H, r.KV = KV, r.HD = HD, r.G = H / KV, r.ldq = ldq, r.ldo = ldo, r.causal = 1;
    r.most_q = max_q_len;                                          // (how the sums are cut, and the scores that are kept, go by it)
    r.scale_log2 = (scale != 0.f ? scale : 1.0f / sqrtf((float)HD)) * 1.4426950408889634f;
    const int es = dtype == MYNAH_F32 ? 4 : 2;
    // (as the attention has it: which kernel takes that decides whether there are scores to keep)
    const bool aligned = ((uintptr_t)q & 15) == 0 && ((uintptr_t)out & 15) == 0 && (long long)ldq * es % 16 == 0 && (long long)ldo * es % 16 == 0;
    MassArgs a{};
    a.r = r;
    const bool tc = mass_plan(a, dtype, aligned, max_q_len);
    const long long need = mynah_attn_mass_scratch_floats(T, B, max_q_len, H, KV, HD, dtype, n_ids, aligned);
    MYNAH_REQUIRE(scratch_floats >= need, "attn_mass: scratch holds %lld floats, %lld are needed", scratch_floats, need);
    const long long attn = attn_rows_scratch_floats(T, B, max_q_len, H, KV, HD, dtype, 1, n_ids, aligned);
    float* lse = scratch + attn;
    float* part = lse + (((long long)T * H + 3) & ~3ll);
    const PageTable pt{page_indptr, page_ids, page_base, n_pages};
    const int rc = attn_rows_run("attn_mass", q, out, dtype, r, max_q_len, k_cache, v_cache, cu_q, kv_len, pt, nullptr, scratch, attn, lse,
                                 a.score_rows > 0 ? part : nullptr, a.score_rows, n_ids, mass, status, stream);
    if (rc != 0) return rc;
    if (a.score_rows > 0) return 0;                                // the joining launch has added them up
    const long long units = mass_units_max(a, n_ids);
    MYNAH_REQUIRE(units * KV < (1ll << 31) && KV <= 65535, "attn_mass: launch too large");
    const dim3 grid((unsigned)units, KV);
    if (tc) {
        if (launch_mass_tcgen05(q, k_cache, lse, mass, part, cu_q, kv_len, pt, a, n_ids, status, stream)) return -1;
    } else if (launch_mass_generic(q, k_cache, lse, mass, part, dtype, cu_q, kv_len, pt, a, grid, status, stream)) {
        return -1;
    }
    if (a.by_keys) return 0;                                       // nothing was cut over its rows
    const cudaError_t e = launch_behind(attn_mass_add_kernel, grid, dim3(a.keys), 0, stream, mass, (const float*)part, cu_q, kv_len, pt, a, status);
    if (e != cudaSuccess) return mynah_fail("attn_mass: %s", cudaGetErrorString(e));
    return mynah_check_launch("attn_mass_add");
}
