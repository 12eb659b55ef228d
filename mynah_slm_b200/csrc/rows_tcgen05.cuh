// What the tcgen05 kernels on packed rows share beyond tcgen05.cuh: staged rows, the queries' tensor map.
#pragma once
#include "tcgen05.cuh"

namespace tc5 {

constexpr int HALF_BYTES = 128 * 128; // 128 rows of 128 bytes: one 64-column half of a tile
constexpr int PAGE_BYTES = PAGE_TOKENS * 128;

// One lane of a converged warp, the same every time.
static __device__ __forceinline__ bool elect_one() {
    uint32_t on;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(on));
    return on != 0;
}
static __device__ __forceinline__ void st_shared(uint32_t addr, float4 x) {
    asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "f"(x.x), "f"(x.y), "f"(x.z), "f"(x.w) : "memory");
}
static __device__ __forceinline__ float4 ld_shared(uint32_t addr) {
    float4 x;
    asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(x.x), "=f"(x.y), "=f"(x.z), "=f"(x.w) : "r"(addr) : "memory");
    return x;
}
static __device__ __forceinline__ void fma2v(float& x0, float& x1, float a0, float a1, float b, float c0, float c1) {
    asm("{ .reg .b64 ra, rb, rc, rd;\n\t mov.b64 ra, {%2, %3};\n\t mov.b64 rb, {%4, %4};\n\t mov.b64 rc, {%5, %6};\n\t"
        " fma.rn.f32x2 rd, ra, rb, rc;\n\t mov.b64 {%0, %1}, rd; }"
        : "=f"(x0), "=f"(x1) : "f"(a0), "f"(a1), "f"(b), "f"(c0), "f"(c1));
}
static __device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
                 ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z) : "memory");
}
// q as [T][H][HD] with a row pitch of ld elements; boxes of 64 columns x G heads x `tokens` tokens, 128-byte swizzle.
static inline int make_map_rows(CUtensorMap* map, const void* q, long long T, int H, int HD, int G, int ld, int tokens) {
    EncodeTiledFn fn = encode_fn();
    if (fn == nullptr) return mynah_fail("tensor map: the driver does not provide cuTensorMapEncodeTiled");
    const cuuint64_t dims[3] = {(cuuint64_t)HD, (cuuint64_t)H, (cuuint64_t)T};
    const cuuint64_t strides[2] = {(cuuint64_t)HD * 2, (cuuint64_t)ld * 2};
    const cuuint32_t box[3] = {64, (cuuint32_t)G, (cuuint32_t)tokens};
    const cuuint32_t estr[3] = {1, 1, 1};
    const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(q), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return mynah_fail("tensor map: cuTensorMapEncodeTiled failed with code %d", (int)r);
    return 0;
}

}  // namespace tc5
