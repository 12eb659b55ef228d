// What the attention of a few rows a sequence (attn_rows.cu, attn_rows_tcgen05.cu) and the sums of its weights (attn_mass.cu)
// hand to one another.
#pragma once
#include "row_units.cuh"

// Partial results of a cut tile, and what every launch of one call reads.
struct RowsScratch {
    RowInfo* info;                    // [B]
    float2* ml;                       // [units][KV][tile_rows]: reference maximum (base 2, scaled) and sum
    float* o;                         // [units][KV][tile_rows][HD], not normalised
    float* lse;                       // [KV][T][G]: log2 of the sum of 2^score, -inf for a row that sees nothing; null: not wanted
};

// fp32 words of scratch that attention of this shape needs (without lse), and how it is laid out.
long long rows_scratch_floats(const RowsArgs& a);
RowsScratch rows_scratch(const RowsArgs& a, float* scratch, float* lse);

// Fills tile_rows, min_pages and target for the kernel that takes these sizes; `tc` says which.
bool rows_plan(RowsArgs& a, int dtype, int max_q_len, bool aligned);

int launch_rows_generic(const void* q, void* out, int dtype, const RowsArgs& a, const void* k, const void* v, const int* cu_q,
                        const int* kv_len, PageTable pt, const long long* masks, RowsScratch s, int* status, cudaStream_t stream);
int launch_rows_tcgen05(const void* q, void* out, const RowsArgs& a, const void* k, const void* v, const int* cu_q,
                        const int* kv_len, PageTable pt, const long long* masks, RowsScratch s, int* status, cudaStream_t stream);
int launch_rows_merge(void* out, int dtype, const RowsArgs& a, const int* cu_q, const int* kv_len, RowsScratch s, int* status,
                      cudaStream_t stream);
bool rows_tcgen05_takes(int dtype, int H, int KV, int HD);

__device__ __forceinline__ float ex2_f(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
