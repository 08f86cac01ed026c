// lp_mx.cuh - what the MXFP4 kernels share: sizes of the packed layout (lp_mx.cu), conversions, arguments of a product.
#pragma once

#include "lp_common.cuh"

namespace lp {
namespace mx {

constexpr int Q_TILE = 128 * 64;      // bytes of 128 rows x 128 e2m1 values
constexpr int SF_TILE = 512;          // bytes of their scales: 128 rows x 4

// Where quantized activations go: the image and its scales, rows in the image, 128-row groups of scales.
struct ActDst { uint8_t* img; uint8_t* sf; int rows, groups; };

struct MxArgs {
    const uint8_t* q;            // packed weights
    const uint8_t* sfa;          // their scales
    const uint8_t* img;          // quantized activations
    const uint8_t* sfb;
    float*         y;
    int            M, N, kts, rts, img_rows, groups, tile_w;
    // experts: {expert, first row in the image, rows, -} of every token tile, their number, and the pair of every image row
    const int4*    tab;
    const int*     n_tiles;
    const int*     out_row;
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
__device__ __forceinline__ float e4m3_value(uint32_t b) {
    const uint32_t e = (b >> 3) & 15, m = b & 7;
    float f = e ? __uint_as_float(((e + 120) << 23) | (m << 20)) : static_cast<float>(m) * 0.001953125f;
    if ((b & 0x7f) == 0x7f) f = __uint_as_float(0x7fc00000u);
    return b & 0x80 ? -f : f;
}

#endif

}  // namespace mx
}  // namespace lp
