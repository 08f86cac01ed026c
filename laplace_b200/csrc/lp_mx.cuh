// lp_mx.cuh - what the MXFP4 kernels share: sizes of the packed layout (lp_mx.cu), conversions, arguments of a product.
#pragma once

#include "lp_common.cuh"

namespace lp {
namespace mx {

constexpr int Q_TILE = 128 * 64;      // bytes of 128 rows x 128 e2m1 values
constexpr int SF_TILE = 512;          // bytes of their scales: 128 rows x 4

// Where quantized activations go: the image and its scales, rows in the image, 128-row groups of scales. A token tile's scales
// begin with a group of their own (the tensor core takes them from TMEM columns whose number is a multiple of four).
struct ActDst { uint8_t* img; uint8_t* sf; int rows, groups, tile_w, tile_groups; };

struct MxArgs {
    const uint8_t* q;            // packed weights
    const uint8_t* sfa;          // their scales
    const uint8_t* img;          // quantized activations
    const uint8_t* sfb;
    float*         y;
    int            M, N, kts, rts, img_rows, groups, tile_w;
    int            tile_groups;  // 128-row groups of scales of a token tile
    // experts: {expert, first row in the image, rows, first group} of every token tile, their number, and the pair of every image row
    const int4*    tab;
    const int*     n_tiles;
    const int*     out_row;
    int            tiles_m;      // token tiles of one matrix
    float*         part;         // sums of cut tiles, and how many of a tile's parts there are so far
    unsigned*      counters;
    int*           err;
};
#ifdef __CUDACC__

// two values as e2m1, the first in the low four bits: to nearest, ties to even, magnitudes over 6 become 6
__device__ __forceinline__ uint32_t e2m1x2(float a, float b) {
    uint32_t r;
    asm("{\n\t.reg .b8 t;\n\tcvt.rn.satfinite.e2m1x2.f32 t, %2, %1;\n\tcvt.u32.u8 %0, t;\n\t}" : "=r"(r) : "f"(a), "f"(b));
    return r;
}
// four values as e4m3, the first in the lowest byte
__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
    uint16_t lo, hi;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %2, %1;" : "=h"(lo) : "f"(a), "f"(b));
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %2, %1;" : "=h"(hi) : "f"(c), "f"(d));
    return static_cast<uint32_t>(lo) | (static_cast<uint32_t>(hi) << 16);
}

#endif

constexpr int MIN_STEPS = 2;          // least k steps of 128 that a CTA takes of cut tiles

}  // namespace mx

size_t mx_gemm_part_bytes(int nt, int cut_tiles);
int    launch_mx_gemm(const mx::MxArgs& a, int nt, long long tiles, bool grouped, cudaStream_t st);

}  // namespace lp
