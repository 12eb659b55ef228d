// What the attention of a few rows a sequence (attn_rows.cu, attn_rows_tcgen05.cu) and the sums of its weights (attn_mass.cu)
// hand to one another.
#pragma once
#include "row_units.cuh"

#include <atomic>

// Partial results of cut items, and what every launch of one call reads.
struct RowsScratch {
    RowStart* starts;                 // [ctas]: where every CTA begins (not OWN)
    float2* ml;                       // [rows]: reference maximum (base 2, scaled) and sum (RowWalk::scratch_row says whose)
    float* o;                         // [rows][HD], not normalised
    float* scores;                    // [entries of the page lists][KV][score_rows][64]: scores * scale_log2, -inf for unseen keys; null: not wanted
    int score_rows, entries;          // (entries: of the page lists)
    float* mass;                      // [n_pages][KV][64]: the sums that the kept scores are added to
    int sum_chunks;                   // CTAs that add for one sequence and kv head
    float* lse;                       // [KV][T][G]: log2 of the sum of 2^score, -inf for a row that sees nothing; null: not wanted
};

// fp32 words of scratch that attention of this shape needs (without lse), and how it is laid out.
long long rows_scratch_floats(const RowsArgs& a);
RowsScratch rows_scratch(const RowsArgs& a, float* scratch, float* lse);

// Fills tile_rows, min_range, ctas and so on; true where the tcgen05 kernel takes the call. n_ids: entries of the page
// lists (-1: any number).
bool rows_plan(RowsArgs& a, int dtype, int max_q_len, int n_ids, bool aligned);

int launch_rows_generic(const void* q, void* out, int dtype, const RowsArgs& a, const void* k, const void* v, const int* cu_q,
                        const int* kv_len, PageTable pt, const long long* masks, RowsScratch s, int* status, cudaStream_t stream);
int launch_rows_tcgen05(const void* q, void* out, const RowsArgs& a, const void* k, const void* v, const int* cu_q,
                        const int* kv_len, PageTable pt, const long long* masks, RowsScratch s, int* status, cudaStream_t stream);
int launch_rows_join(void* out, int dtype, const RowsArgs& a, const int* cu_q, const int* kv_len, PageTable pt, RowsScratch s, int* status,
                     cudaStream_t stream);
bool rows_tcgen05_takes(int dtype, int H, int KV, int HD);

// Four values of a row whose pieces of four are aligned.
__device__ __forceinline__ float4 four_of(const float* p) { return *reinterpret_cast<const float4*>(p); }
__device__ __forceinline__ float4 four_of(const bf16* p) {
    const uint2 w = *reinterpret_cast<const uint2*>(p);
    return make_float4(__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xffff0000u), __uint_as_float(w.y << 16), __uint_as_float(w.y & 0xffff0000u));
}
// The same where rows are not aligned (volatile: read one by one, whatever is made of the other branch).
__device__ __forceinline__ float4 four_apart(const float* p) {
    const volatile float* w = p;
    return make_float4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ float4 four_apart(const bf16* p) { return make_float4(to_f32(p[0]), to_f32(p[1]), to_f32(p[2]), to_f32(p[3])); }

__device__ __forceinline__ float ex2_f(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Lets a kernel use so much shared memory, once a device (`done` has a bit for each).
template <typename K> static inline cudaError_t shared_memory_once(K kernel, size_t bytes, std::atomic<unsigned long long>& done) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess || (dev < 64 && (done.load(std::memory_order_relaxed) >> dev & 1ull))) return e;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    if (e == cudaSuccess && dev < 64) done.fetch_or(1ull << dev, std::memory_order_relaxed);
    return e;
}

// A launch that may begin while the kernel before it on the stream finishes. (Always, whatever mynah_pdl_enabled() says: that is about
// launches of one operator behind another's, which cost a decode step more than they gave; this is an operator's own second or
// third launch, and 2,048 tokens with sums took 75 us instead of 80.) Every CTA of it waits for that one (griddep_wait), so
// that it cannot end first, and before the wait it reads only what was there before both (the step's description, the page lists).
template <typename... KArgs, typename... Args>
static inline cudaError_t launch_behind(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream, Args&&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...);
}
