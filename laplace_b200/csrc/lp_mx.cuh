// lp_mx.cuh - what the MXFP4 kernels share: sizes of the packed layout (lp_mx.cu), conversions, arguments of a product.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>

#include "lp_common.cuh"

namespace lp {
namespace mx {

constexpr int Q_TILE = 128 * 64;      // bytes of 128 rows x 128 e2m1 values
constexpr int SF_TILE = 512;          // bytes of their scales: 128 rows x 4

// laplace_cuda_mxfp4_last_kernel: one of these, and 16 times the CTAs that share out k
enum : int { KERNEL_SMALL = 1, KERNEL_SINGLE = 2, KERNEL_PAIR = 3 };

// Where quantized activations go: the image and its scales, rows in the image, 128-row groups of scales. A token tile's scales
// begin with a group of their own (the tensor core takes them from TMEM columns whose number is a multiple of four).
struct ActDst { uint8_t* img; uint8_t* sf; int rows, groups, tile_w, tile_groups; };

// Tiles of 256 weight rows x 256 tokens over n pairs of SMs: `cut` of `tiles` are cut, over `ctas` pairs.
struct Cut { int tiles, cut, ctas; };
// What a cut costs where nothing comes after it, in k steps of a whole tile (512 cycles): once, and for every part of a tile that is read back.
constexpr int CUT_COST = 14, PIECE_COST = 6;
__host__ __device__ inline int cut_cost(int kts, int parts) { return parts == 1 ? kts : (kts + parts - 1) / parts + CUT_COST + (parts - 1) * PIECE_COST; }
constexpr int MAX_PARTS = 32;
// Tiles that do not make a round of n. Without a whole round each is cut in `parts` parts, the number that costs least. Where whole rounds follow, the
// tiles before them may be cut over all pairs, into parts of eight steps at least; their sums are joined during the whole tiles, but the way to
// memory and back costs all the same (512 x 4096 x 14336, 38 tiles of 32 steps over, 74 pairs: 33.8 us cut, 31.8 whole; 2048 x 14336 x 4096,
// 54 of 112 steps: 108 either way).
__host__ __device__ inline int over_cost(int left, int kts, int ctas) { return static_cast<int>((static_cast<long long>(left) * kts + ctas - 1) / ctas) + CUT_COST + 3 * ctas / left; }
__host__ __device__ inline Cut cut_of(int tiles, int kts, int n, int parts) {
    Cut c{tiles, 0, 0};
    const int left = tiles % n;
    if (!left) return c;
    if (tiles > n) parts = 1 + kts / 8;
    const long long most = static_cast<long long>(left) * parts;
    const int ctas = most < n ? static_cast<int>(most) : n;
    if (ctas > left && (tiles < n || over_cost(left, kts, ctas) < kts)) { c.cut = left; c.ctas = ctas; }
    return c;
}
__host__ __device__ inline int most_parts(int tiles, int kts, int n) {
    const int left = tiles % n, m = left ? n / left : 1;
    return m < kts ? (m < MAX_PARTS ? m : MAX_PARTS) : (kts < MAX_PARTS ? kts : MAX_PARTS);
}

struct MxArgs {
    const uint8_t* q;            // packed weights
    const uint8_t* sfa;          // their scales
    const uint8_t* img;          // quantized activations
    const uint8_t* sfb;
    float*         y;
    int            M, N, kts, rts, img_rows, groups, tile_w;
    int            tile_groups;  // 128-row groups of scales of a token tile
    // experts: {expert, first row in the image, rows, first group} of every token tile, their number, and the pair of every image row (-1: a bad one)
    const int4*    tab;
    const int4*    work;         // {row tiles of all token tiles, how many of them are cut, over how many units, -}
    const int*     out_row;
    int            tiles_m;      // token tiles of one matrix
    int            row_tiles;    // row tiles of a matrix: rts, or those of 256 rows
    float*         part;         // parts of cut tiles, and their counters
    unsigned*      counters;
    int*           err;
    Cut            dense;        // the same of one matrix
};
#ifdef __CUDACC__

// eight values as e2m1, the first in the lowest four bits: to nearest, ties to even, magnitudes over 6 become 6
__device__ __forceinline__ uint32_t e2m1x8(const float (&v)[8]) {
    uint32_t r;
    asm("{\n\t.reg .b8 a, b, c, d;\n\tcvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\tcvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\tcvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\tmov.b32 %0, {a, b, c, d};\n\t}"
        : "=r"(r) : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
    return r;
}
// the values of two e2m1 codes
__device__ __forceinline__ float2 e2m1x2_value(uint32_t c) {
    uint32_t h;
    asm("{\n\t.reg .b8 t;\n\tcvt.u8.u32 t, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, t;\n\t}" : "=r"(h) : "r"(c));
    return __half22float2(*reinterpret_cast<const __half2*>(&h));
}
// four values as e4m3, the first in the lowest byte
__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
    uint16_t lo, hi;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %2, %1;" : "=h"(lo) : "f"(a), "f"(b));
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %2, %1;" : "=h"(hi) : "f"(c), "f"(d));
    return static_cast<uint32_t>(lo) | (static_cast<uint32_t>(hi) << 16);
}
// Eight values as they lie in memory; their fp32 values; the bits, as fp32, of their largest magnitude (infinity and NaN at or above 0x7f800000).
template <class T> struct Eight;
template <> struct Eight<float> {
    float4 a, b;
    __device__ __forceinline__ void load(const float* p) { a = __ldg(reinterpret_cast<const float4*>(p)); b = __ldg(reinterpret_cast<const float4*>(p) + 1); }
    __device__ __forceinline__ void zero() { a = b = make_float4(0.f, 0.f, 0.f, 0.f); }
    __device__ __forceinline__ void values(float (&v)[8]) const { v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w; }
    __device__ __forceinline__ uint32_t amax() const {
        float v[8];
        values(v);
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
        return m;
    }
};
// two 16-bit values a word: magnitudes compare as unsigned halves
__device__ __forceinline__ uint32_t amax16(const uint4& w) {
    const uint32_t m = __vmaxu2(__vmaxu2(w.x & 0x7fff7fffu, w.y & 0x7fff7fffu), __vmaxu2(w.z & 0x7fff7fffu, w.w & 0x7fff7fffu));
    return max(m & 0xffffu, m >> 16);
}
template <> struct Eight<__half> {
    uint4 w;
    __device__ __forceinline__ void load(const __half* p) { w = __ldg(reinterpret_cast<const uint4*>(p)); }
    __device__ __forceinline__ void zero() { w = make_uint4(0, 0, 0, 0); }
    __device__ __forceinline__ void values(float (&v)[8]) const {
        const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&x[i]));
            v[2 * i] = f.x; v[2 * i + 1] = f.y;
        }
    }
    __device__ __forceinline__ uint32_t amax() const { return __float_as_uint(__half2float(__ushort_as_half(static_cast<unsigned short>(amax16(w))))) & 0x7fffffffu; }
};
template <> struct Eight<__nv_bfloat16> {
    uint4 w;
    __device__ __forceinline__ void load(const __nv_bfloat16* p) { w = __ldg(reinterpret_cast<const uint4*>(p)); }
    __device__ __forceinline__ void zero() { w = make_uint4(0, 0, 0, 0); }
    __device__ __forceinline__ void values(float (&v)[8]) const {
        const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) { v[2 * i] = __uint_as_float(x[i] << 16); v[2 * i + 1] = __uint_as_float(x[i] & 0xffff0000u); }
    }
    __device__ __forceinline__ uint32_t amax() const { return amax16(w) << 16; }
};
__device__ __forceinline__ void load8(const float* p, float (&v)[8]) {
    Eight<float> e;
    e.load(p);
    e.values(v);
}
__device__ __forceinline__ float amax8(const float (&v)[8]) {
    float a = fabsf(v[0]);
#pragma unroll
    for (int i = 1; i < 8; ++i) a = max_nan(a, fabsf(v[i]));
    return a;
}
// 2^e for e in [-127, 127]
__device__ __forceinline__ float pow2(int e) { return e == -127 ? __uint_as_float(0x00400000u) : __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }

// Eight values of a 32-value block that four neighbouring lanes hold -> their e4m3 bytes; sc: the scale bytes of the lane's 16-lane half
// (128 values), lowest block first. A block with an infinity or a NaN is NaN, scale and values.
__device__ __forceinline__ uint2 mxfp8_block8(const float (&v)[8], int lane, uint32_t& sc) {
    float a = amax8(v);
    a = max_nan(a, __shfl_xor_sync(0xffffffffu, a, 1));
    a = max_nan(a, __shfl_xor_sync(0xffffffffu, a, 2));
    const bool bad = !(a < __uint_as_float(0x7f800000u));
    const uint32_t bits = __float_as_uint(a);
    int s = static_cast<int>(bits >> 23) - 135 + ((bits & 0x7fffffu) > 0x600000u);      // a = m 2^e, 1 <= m < 2: e - 8 up to m = 1.75, else e - 7
    if (s < -127) s = -127;
    const float inv = pow2(-s);
    uint2 q;
    q.x = bad ? 0x7f7f7f7fu : e4m3x4(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv);
    q.y = bad ? 0x7f7f7f7fu : e4m3x4(v[4] * inv, v[5] * inv, v[6] * inv, v[7] * inv);
    sc = (bad ? 255u : static_cast<uint32_t>(s + 127)) << (8 * ((lane >> 2) & 3));
    sc |= __shfl_xor_sync(0xffffffffu, sc, 4);
    sc |= __shfl_xor_sync(0xffffffffu, sc, 8);
    return q;
}

#endif

}  // namespace mx

size_t mx_pair_part_bytes();
int    mx_pair_counters();
int    launch_mx_pair(const CUtensorMap& map, const mx::MxArgs& a, bool grouped, cudaStream_t st);
long long mx_mid_ns(long long tiles, int kts, int tokens);
int    launch_mx_mid(const CUtensorMap& map, const mx::MxArgs& a, int nt, long long tiles, bool grouped, cudaStream_t st);
bool   mx_small_takes(int rows, bool grouped);
int    launch_mx_small(const float* x, int x_rows, const uint8_t* packed, const int* pair_expert, const int* pair_row, int rows, int experts, float* y, int K, int N, cudaStream_t st);

}  // namespace lp
