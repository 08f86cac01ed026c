// lp_mx_mma.cuh - the block-scaled tensor core instruction on e2m1 weights and e4m3 activations, its scales, the weights' tensor map.
#pragma once

#include "lp_mx.cuh"
#include "lp_tc.cuh"

namespace lp {
namespace mx {

#ifdef __CUDACC__

// CG: CTAs that work on one product, 1 or 2 (a pair of SMs: 128 rows of A and half of B's in the shared memory of each).
// kind::mxf8f6f4: D fp32, A e2m1, B e4m3, both K-major, scales ue8m0; 128 CG rows of A, n of B; the byte of the scale words that this step takes
template <int CG>
__device__ __forceinline__ uint32_t idesc_mx(int n, int byte) {
    return (static_cast<uint32_t>(byte) << 4) | (5u << 7) | (static_cast<uint32_t>(n >> 3) << 17) | (1u << 23) | (8u * CG << 24) | (static_cast<uint32_t>(byte) << 29);
}
template <int CG>
__device__ __forceinline__ void mma_mx(uint32_t d, uint64_t ad, uint64_t bd, uint32_t idesc, uint32_t sfa, uint32_t sfb, uint32_t acc) {
    if constexpr (CG == 1)
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
            :: "r"(d), "l"(ad), "l"(bd), "r"(idesc), "r"(sfa), "r"(sfb), "r"(acc) : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
            :: "r"(d), "l"(ad), "l"(bd), "r"(idesc), "r"(sfa), "r"(sfb), "r"(acc) : "memory");
}
// 32 rows of 16 bytes -> 4 TMEM columns of every quadrant (of both CTAs, each from its own shared memory); the first column a multiple of four
template <int CG>
__device__ __forceinline__ void copy_scales(uint32_t taddr, uint32_t smem) {
    const uint64_t d = static_cast<uint64_t>((smem >> 4) & 0x3fffu) | (static_cast<uint64_t>(128 >> 4) << 16) | (static_cast<uint64_t>(128 >> 4) << 32) | (static_cast<uint64_t>(1) << 46);
    if constexpr (CG == 1) asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" :: "r"(taddr), "l"(d) : "memory");
    else asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" :: "r"(taddr), "l"(d) : "memory");
}
// ---- clusters whose CTAs send results into one another's shared memory ----
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }
__device__ __forceinline__ void arrive_release(uint32_t remote_bar) { asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" :: "r"(remote_bar) : "memory"); }
__device__ __forceinline__ void st_cluster(uint32_t addr, float v) { asm volatile("st.shared::cluster.f32 [%0], %1;" :: "r"(addr), "f"(v) : "memory"); }
__device__ __forceinline__ void st_cluster4(uint32_t addr, float a, float b, float c, float d) {
    asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" :: "r"(addr), "f"(a), "f"(b), "f"(c), "f"(d) : "memory");
}
// *p = v where `on`, without a branch (with one the 32 stores of a column block no longer overlap: experts' products 36 -> 61 us)
__device__ __forceinline__ void store_if(bool on, float* p, float v) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %2, 0;\n\t@p st.global.f32 [%0], %1;\n\t}" :: "l"(p), "f"(v), "r"(static_cast<uint32_t>(on)) : "memory");
}
// 32 lanes x 8 columns
__device__ __forceinline__ void ld8(uint32_t taddr, float (&v)[8]) {
    uint32_t r[8];
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]) : "r"(taddr));
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(r[i]);
}

#endif

// The tiles' rows one after the other, 128 values in 64 bytes each; a copy spreads the 8 bytes of 16 values over 16 of shared memory and
// counts 64 bytes a row at the barrier.
inline bool mx_weights_map(CUtensorMap* m, const uint8_t* q, size_t tiles) {
    return tc::make_map_2d(m, CU_TENSOR_MAP_DATA_TYPE_16U4_ALIGN16B, q, 128, static_cast<uint64_t>(tiles) * 128, 64, 128, 128, CU_TENSOR_MAP_SWIZZLE_128B, "MXFP4 weights");
}

}  // namespace mx
}  // namespace lp
