// Cache row order and warp-level matrix helpers shared by the attention kernels.
#pragma once
#include "common.cuh"

namespace icua {

// KV rows are stored with their sixteen 16-byte chunks permuted by the row's position:
// element d of position p lives at chunk (d / 8) ^ (p & 7).  Eight consecutive rows then cover
// eight different bank groups, so ldmatrix reads from bulk-copied rows are conflict-free.
__host__ __device__ __forceinline__ int kv_swz(int d, int pos) { return (((d >> 3) ^ (pos & 7)) << 3) | (d & 7); }

__device__ __forceinline__ void ldsm_x4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr));
}

__device__ __forceinline__ void ldsm_x4_trans(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr));
}

template <typename KVT>
__device__ __forceinline__ void mma_kv(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma_kv<__half>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    mma_16816(d, a, b0, b1);
}
template <>
__device__ __forceinline__ void mma_kv<__nv_bfloat16>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <typename KVT>
__device__ __forceinline__ uint32_t pack2(KVT lo, KVT hi);
template <>
__device__ __forceinline__ uint32_t pack2<__half>(__half lo, __half hi) {
    return (uint32_t)__half_as_ushort(lo) | ((uint32_t)__half_as_ushort(hi) << 16);
}
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(__nv_bfloat16 lo, __nv_bfloat16 hi) {
    return (uint32_t)__bfloat16_as_ushort(lo) | ((uint32_t)__bfloat16_as_ushort(hi) << 16);
}

}  // namespace icua
