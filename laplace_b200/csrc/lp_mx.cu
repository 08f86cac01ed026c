// lp_mx.cu - MXFP4 weights (GGUF type 39): quantizer, the layout in HBM that the products read, and the products with
// MXFP8 activations - one matrix, or experts with ragged numbers of rows. No reference counterpart (Laplace has no such type).
//
// Formats. Blocks of 32 values of a row share a power of two 2^s, held as s + 127 in one byte (255: the block is NaN).
//   MXFP4  e2m1 values 0, .5, 1, 1.5, 2, 3, 4, 6 and their negatives. GGUF block, 17 bytes: s + 127, then 16 bytes, value l in the low,
//          value l + 16 in the high half of byte l. Quantizer: s = floor(log2(amax)) - 2, nearest, ties to even, magnitudes over 6 held as 6.
//   MXFP8  e4m3 values up to 448, for activations: the smallest s with amax <= 448 * 2^s, so that no value is cut off (with
//          floor(log2(amax)) - 8 a fifth of the blocks would lose up to an eighth of their largest value).
// Scaling by a power of two is exact and the roundings are the hardware's, so the quantized values are the definition's to the bit.
//
// Packed weights. A matrix of N rows of K values is cut into tiles of 128 rows x 128 values; rows and values behind the end are 0.
//   q   [matrix][row tile][k tile][128 rows][64 bytes]    value 2 i in the low, 2 i + 1 in the high half of byte i
//   sf  [matrix][row tile][k tile][512 bytes]             behind all q: the scale byte of (row r, 32-value block b of the four) at
//                                                         (r % 32) * 16 + (r / 32) * 4 + b, the order in which the tensor core takes them
// A tile is 8 KB in one piece (rows apart would be read 64 bytes at a time), 0.53 bytes per value as in the file.
// Quantized activations (workspace): image [k tile][row][128 bytes], 16-byte pieces of a row swizzled by row % 8 as the tensor core
// reads them, and the scales [k tile][128-row group][512 bytes] in the order above, the rows of a token tile in groups of their own.
#include <cuda_bf16.h>

#include "lp_mx.cuh"
#include "lp_mx_mma.cuh"

namespace lp {
namespace {

using namespace mx;

// ---- values -> GGUF blocks ---------------------------------------------------------------------------------------
// A block per 4 lanes, 8 values each; 64 blocks a round, whose loads all go first, gathered in shared memory (a block is 17 bytes) and written in order.
// us with 2 / 4 / 8 rounds a CTA: 14336 x 4096 bf16 34.7 / 28.9 / 26.5 (5.6 TB/s; instructions are some 60 % of what the SMs can issue), fp32 41.9 / 39.9 / 40.6
// (6.7 TB/s, what a copy reaches), 1001 x 2848 fp16 2.85 / 3.05 / 3.4, 1 x 4096 1.7 / 1.85 / 2.35. One round and 16-byte stores by half as many lanes: bf16 50, fp32 55.
constexpr int QB = 64;
template <class T> int quantize_rounds(long long blocks) {
    const long long round = static_cast<long long>(QB) * ctx().sm_count;       // an SM's CTAs have a round each
    return blocks < 16 * round ? 2 : sizeof(T) == 2 && blocks > 64 * round ? 8 : 4;
}
template <class T, int ROUNDS>
__global__ void __launch_bounds__(256) mxfp4_quantize_kernel(const T* __restrict__ x, uint8_t* __restrict__ w, long long n_blocks) {
    __shared__ __align__(16) uint8_t out[QB * ROUNDS * 17];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int part = threadIdx.x & 3;
    const long long b0 = static_cast<long long>(blockIdx.x) * (QB * ROUNDS);
    const int here = n_blocks - b0 < QB * ROUNDS ? static_cast<int>(n_blocks - b0) : QB * ROUNDS;
    Eight<T> in[ROUNDS];
#pragma unroll
    for (int i = 0; i < ROUNDS; ++i) {
        const int blk = (threadIdx.x >> 2) + QB * i;
        if (blk < here) in[i].load(x + (b0 + blk) * 32 + part * 8);
        else in[i].zero();
    }
#pragma unroll
    for (int i = 0; i < ROUNDS; ++i) {
        const int blk = (threadIdx.x >> 2) + QB * i;
        uint32_t a = in[i].amax();
        a = max(a, __shfl_xor_sync(0xffffffffu, a, 1));
        a = max(a, __shfl_xor_sync(0xffffffffu, a, 2));
        const bool bad = a >= 0x7f800000u;                                // infinity or NaN: the block stands for NaN
        const int s = max(static_cast<int>(a >> 23) - 129, -127);         // floor(log2(a)) - 2; 0 and numbers below the normal ones: the lowest
        const float inv = pow2(-s);
        float v[8];
        in[i].values(v);
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] *= inv;
        const uint32_t c = bad ? 0 : e2m1x8(v);                           // eight codes, value i in bits 4 i
        const uint32_t o = __shfl_xor_sync(0xffffffffu, c, 2);            // lanes 0 and 1 hold values 0..15, lanes 2 and 3 16..31
        // bytes 8 (part & 1) + 4 (part >> 1) .. + 3 of the sixteen: four codes of c and o each, spread over bytes
        const int h = part >> 1;
        uint32_t lo = __byte_perm(c, o, h ? 0x4476 : 0x4410), hi = __byte_perm(c, o, h ? 0x4432 : 0x4454);
        lo = (lo & 0xffu) | ((lo & 0xff00u) << 8);
        hi = (hi & 0xffu) | ((hi & 0xff00u) << 8);
        lo = (lo | (lo << 4)) & 0x0f0f0f0fu;
        hi = (hi | (hi << 4)) & 0x0f0f0f0fu;
        const uint32_t bytes = lo | (hi << 4);
        uint8_t* d = out + blk * 17 + 1 + (part & 1) * 8 + h * 4;
#pragma unroll
        for (int k = 0; k < 4; ++k) d[k] = static_cast<uint8_t>(bytes >> (8 * k));
        if (part == 0) out[blk * 17] = static_cast<uint8_t>(bad ? 255 : s + 127);
    }
    __syncthreads();
    uint8_t* dst = w + b0 * 17;
    const int bytes = here * 17;
    if ((reinterpret_cast<uintptr_t>(dst) & 15) == 0) {
        for (int i = threadIdx.x; i < bytes / 16; i += 256) reinterpret_cast<uint4*>(dst)[i] = reinterpret_cast<const uint4*>(out)[i];
        for (int i = (bytes & ~15) + threadIdx.x; i < bytes; i += 256) dst[i] = out[i];
    } else {
        for (int i = threadIdx.x; i < bytes; i += 256) dst[i] = out[i];
    }
}

template <class T>
int launch_quantize(const void* x, uint8_t* w, long long blocks, cudaStream_t st) {
    const int r = quantize_rounds<T>(blocks);
    const long long grid = (blocks + QB * r - 1) / (QB * r);
    if (grid > 0x7fffffffll) return fail(LAPLACE_ERR_LIMIT, "mxfp4_quantize: n=%lld", blocks * 32);
    const dim3 g(static_cast<unsigned>(grid));
    const T* p = static_cast<const T*>(x);
    ctx().launches++;
    if (r == 2) return launch_early(mxfp4_quantize_kernel<T, 2>, g, 256, 0, st, p, w, blocks);
    if constexpr (sizeof(T) == 2)
        if (r == 8) return launch_early(mxfp4_quantize_kernel<T, 8>, g, 256, 0, st, p, w, blocks);
    return launch_early(mxfp4_quantize_kernel<T, 4>, g, 256, 0, st, p, w, blocks);
}

// ---- GGUF blocks -> values (dequantize) ----------------------------------------------------------------------------
// 256 blocks a CTA through shared memory, from the 16-byte boundary below their first byte; then four values a thread and store, in order.
// Bound by the stores (4 bytes a value): 14336 x 4096 42 us, 6.4 TB/s; 71 with a thread per 16 values that reads its block by the byte.
constexpr int DB = 256;
__global__ void __launch_bounds__(256) mxfp4_dequantize_kernel(const uint8_t* __restrict__ w, float* __restrict__ dst, long long n_blocks) {
    __shared__ __align__(16) uint8_t in[DB * 17 + 32];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const long long b0 = static_cast<long long>(blockIdx.x) * DB;
    const int here = n_blocks - b0 < DB ? static_cast<int>(n_blocks - b0) : DB;
    const uint8_t* src = w + b0 * 17;
    const int off = static_cast<int>(reinterpret_cast<uintptr_t>(src) & 15), bytes = here * 17;
    // whole 16-byte pieces inside the blocks, and what lies before and behind them by the byte
    const int first = off ? 16 - off : 0, pieces = bytes > first ? (bytes - first) / 16 : 0, tail = first + pieces * 16;
    for (int i = threadIdx.x; i < pieces; i += 256) *reinterpret_cast<uint4*>(in + off + first + 16 * i) = __ldg(reinterpret_cast<const uint4*>(src + first) + i);
    for (int i = threadIdx.x; i < first && i < bytes; i += 256) in[off + i] = src[i];
    for (int i = tail + threadIdx.x; i < bytes; i += 256) in[off + i] = src[i];
    __syncthreads();
    float4* o = reinterpret_cast<float4*>(dst + b0 * 32);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int at = i * 256 + threadIdx.x, blk = at >> 3, part = at & 7;
        if (blk >= here) break;
        const uint8_t* b = in + off + blk * 17;
        const uint32_t e = b[0], h = (part >> 2) * 4;
        const float d = __uint_as_float(e == 255 ? 0x7fc00000u : e ? e << 23 : 0x00400000u);
        const uint8_t* q = b + 1 + (part & 3) * 4;
        const uint32_t c0 = ((q[0] >> h) & 15u) | (((q[1] >> h) & 15u) << 4), c1 = ((q[2] >> h) & 15u) | (((q[3] >> h) & 15u) << 4);
        const float2 lo = e2m1x2_value(c0), hi = e2m1x2_value(c1);
        __stcs(o + at, make_float4(__fmul_rn(d, lo.x), __fmul_rn(d, lo.y), __fmul_rn(d, hi.x), __fmul_rn(d, hi.y)));
    }
}

// ---- GGUF blocks -> packed tiles -----------------------------------------------------------------------------------
// A thread per block: rows of a tile x its four blocks. Blocks start at any byte: 17 bytes lie in five aligned words, whose bytes
// outside the block share a word with it.
__global__ void __launch_bounds__(512) mxfp4_pack_kernel(const uint8_t* __restrict__ w, uint8_t* __restrict__ q, uint8_t* __restrict__ sf, int N, int K, int rts, int kts) {
    const int kt = blockIdx.x, rt = blockIdx.y % rts, e = blockIdx.y / rts;
    const int r = threadIdx.x >> 2, b = threadIdx.x & 3;
    const int row = rt * 128 + r, k32 = kt * 4 + b, bpr = K / 32;
    uint4 o = make_uint4(0, 0, 0, 0);
    uint8_t scale = 127;
    if (row < N && k32 < bpr) {
        const uint8_t* p = w + ((static_cast<size_t>(e) * N + row) * bpr + k32) * 17;
        const uint32_t* a = reinterpret_cast<const uint32_t*>(reinterpret_cast<uintptr_t>(p) & ~static_cast<uintptr_t>(3));
        const uint32_t sh = (reinterpret_cast<uintptr_t>(p) & 3) * 8;
        const uint32_t x0 = __ldg(a), x1 = __ldg(a + 1), x2 = __ldg(a + 2), x3 = __ldg(a + 3), x4 = __ldg(a + 4);
        const uint32_t y0 = __funnelshift_r(x0, x1, sh), y1 = __funnelshift_r(x1, x2, sh), y2 = __funnelshift_r(x2, x3, sh), y3 = __funnelshift_r(x3, x4, sh),
                       y4 = x4 >> sh;
        scale = static_cast<uint8_t>(y0);
        const uint32_t in[4] = {__funnelshift_r(y0, y1, 8), __funnelshift_r(y1, y2, 8), __funnelshift_r(y2, y3, 8), __funnelshift_r(y3, y4, 8)};
        uint32_t lo[4], hi[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t l = in[i] & 0x0f0f0f0fu, h = (in[i] >> 4) & 0x0f0f0f0fu;
            lo[i] = l | (l >> 4);                 // bytes 0 and 2: two neighbours each
            hi[i] = h | (h >> 4);
        }
        o = make_uint4(__byte_perm(lo[0], lo[1], 0x6420), __byte_perm(lo[2], lo[3], 0x6420), __byte_perm(hi[0], hi[1], 0x6420), __byte_perm(hi[2], hi[3], 0x6420));
    }
    const size_t tile = (static_cast<size_t>(e) * rts + rt) * kts + kt;
    *reinterpret_cast<uint4*>(q + tile * Q_TILE + r * 64 + b * 16) = o;
    sf[tile * SF_TILE + (r & 31) * 16 + (r >> 5) * 4 + b] = scale;
}

// What follows in the stream may read the tiles before it has waited for the kernel before it: that is this one, which begins when the tiles are written.
__global__ void mxfp4_packed_kernel() {}

// ---- fp32 rows -> MXFP8 image -------------------------------------------------------------------------------------
// A warp takes SEGS pieces of 256 values of a row: a 32-value block per 4 lanes, all loads first. 2048 x 14336 (147 MB in and out) 22 us, 28 with one piece a
// warp. GROUPED: the row of x and the place in the image by
// pair; a pair whose row is none of x's is taken out of the list of results and reported.
template <bool GROUPED, int SEGS>
__global__ void __launch_bounds__(256) mx_act_kernel(const float* __restrict__ x, int x_rows, int K, int kts, int rows, ActDst d, const int* __restrict__ pair_row,
                                                     const int2* __restrict__ place, int* __restrict__ out_row, unsigned* __restrict__ counters, int n_counters, int* err) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int lane = threadIdx.x & 31, per_row = (kts + 2 * SEGS - 1) / (2 * SEGS);
    const long long id = static_cast<long long>(blockIdx.x) * 8 + (threadIdx.x >> 5);
    if (blockIdx.x == 0)
        for (int i = threadIdx.x; i < n_counters; i += 256) counters[i] = 0;
    const int row = static_cast<int>(id / per_row), seg = static_cast<int>(id % per_row) * SEGS;
    if (row >= rows) return;
    int src = row, dst = row, at;                  // at: row in the groups of scales
    if (GROUPED) {
        const int2 p = place[row];
        if (pair_row) src = pair_row[row];
        dst = p.x; at = p.y;
        if (dst < 0) return;
        if (static_cast<unsigned>(src) >= static_cast<unsigned>(x_rows)) {
            if (lane == 0 && seg == 0) { out_row[dst] = -1; atomicCAS(err, DEV_OK, DEV_BAD_INDEX); }
            return;
        }
    } else {
        at = row / d.tile_w * (d.tile_groups * 128) + row % d.tile_w;
    }
    const float* xr = x + static_cast<size_t>(src) * K + lane * 8;
    float v[SEGS][8] = {};
#pragma unroll
    for (int i = 0; i < SEGS; ++i)
        if ((seg + i) * 256 + lane * 8 < K) load8(xr + (seg + i) * 256, v[i]);         // K is a multiple of 32: all eight or none
#pragma unroll
    for (int i = 0; i < SEGS; ++i) {
        if ((seg + i) * 2 >= kts) break;
        uint32_t sc;
        const uint2 q = mxfp8_block8(v[i], lane, sc);
        const int kt = (seg + i) * 2 + (lane >> 4), piece = (lane & 15) >> 1;
        if (kt < kts) {
            *reinterpret_cast<uint2*>(d.img + (static_cast<size_t>(kt) * d.rows + dst) * 128 + ((piece ^ (dst & 7)) << 4) + (lane & 1) * 8) = q;
            if ((lane & 15) == 0)
                *reinterpret_cast<uint32_t*>(d.sf + (static_cast<size_t>(kt) * d.groups + (at >> 7)) * SF_TILE + (at & 31) * 16 + ((at >> 5) & 3) * 4) = sc;
        }
    }
}
// pieces a warp takes: four where there are enough rows to keep the SMs busy all the same (64 warps each)
template <bool GROUPED, class... A>
int launch_act(long long rows, int kts, cudaStream_t st, A... args) {
    const long long segs = rows * ((kts + 1) / 2);
    if (segs > 64ll * ctx().sm_count) return launch_early(mx_act_kernel<GROUPED, 4>, dim3(static_cast<unsigned>((rows * ((kts + 7) / 8) + 7) / 8)), 256, 0, st, args...);
    return launch_early(mx_act_kernel<GROUPED, 1>, dim3(static_cast<unsigned>((segs + 7) / 8)), 256, 0, st, args...);
}

// ---- pairs -> places in the image and a table of token tiles --------------------------------------------------------
// A block per expert (or a few). With all experts' counts it knows where its own begins: each gets whole groups of 8 rows of the image and token tiles
// of its own. Its warps have a run of the pairs each, and with the counts of the warps before them they give every pair its place - by
// its number, not by timing. The counts are made by every block for itself (shared-memory atomics) or, from COUNT_FROM pairs on, by a launch
// of their own. 2,048 / 16,384 pairs, 128 experts, us under ncu: a warp per expert, 32 of them to a block 24 / 158, one block with match
// instructions 12 / 27, counts by every block of 1024 threads 7.4 / 19, by a launch 14 / 19; now 5.6 / 5.5 + 8.4.
constexpr int GROUP_THREADS = 1024;
constexpr int NO_EXPERT = -1, BAD_EXPERT = -2;
__device__ __forceinline__ int expert_of(const int* __restrict__ pair_expert, int p, int P, int E) {
    int e = NO_EXPERT;
    if (p < P) e = __ldg(pair_expert + p);
    return e < 0 ? NO_EXPERT : e >= E ? BAD_EXPERT : e;
}
__global__ void __launch_bounds__(GROUP_THREADS) mx_count_kernel(const int* __restrict__ pair_expert, int P, int E, int2* __restrict__ place,
                                                                 int* __restrict__ counts, int* err) {
    __shared__ int part[GROUP_THREADS / 32];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int mine = blockIdx.x; mine < E; mine += gridDim.x) {
        int k = 0;
        constexpr int U = 8;
        for (int q = threadIdx.x; q < P; q += U * GROUP_THREADS) {
            int e[U];
#pragma unroll
            for (int i = 0; i < U; ++i) e[i] = expert_of(pair_expert, q + i * GROUP_THREADS, P, E);
#pragma unroll
            for (int i = 0; i < U; ++i) {
                k += e[i] == mine;
                if (mine == 0 && e[i] < 0 && q + i * GROUP_THREADS < P) {
                    place[q + i * GROUP_THREADS] = make_int2(-1, -1);
                    if (e[i] == BAD_EXPERT) atomicCAS(err, DEV_OK, DEV_BAD_INDEX);
                }
            }
        }
        k = __reduce_add_sync(0xffffffffu, k);
        __syncthreads();
        if (lane == 0) part[warp] = k;
        __syncthreads();
        if (warp == 0) {
            k = __reduce_add_sync(0xffffffffu, part[lane]);
            if (lane == 0) counts[mine] = k;
        }
    }
}
constexpr int COUNT_FROM = 4097;
__global__ void __launch_bounds__(GROUP_THREADS) mx_group_kernel(const int* __restrict__ pair_expert, int P, int E, int tile_log2, int tile_groups,
                                                                 const int* __restrict__ counts, int2* __restrict__ place, int* __restrict__ out_row, int4* __restrict__ tab,
                                                                 int4* __restrict__ work, int row_tiles, int kts, int n, int* err) {
    constexpr int U = 16;
    const int threads = blockDim.x, W = threads >> 5;
    __shared__ int before[GROUP_THREADS / 32], sum_rows[GROUP_THREADS / 32], sum_tiles[GROUP_THREADS / 32];
    extern __shared__ int sm[];
    int* count = sm;
    int* start = sm + E;                   // first row of an expert in the image
    int* tile0 = sm + 2 * E;               // its first token tile
    if (!counts)
        for (int i = threadIdx.x; i < E; i += threads) count[i] = 0;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int run = ((P + W - 1) / W + 31) & ~31, p0 = warp * run, p1 = min(p0 + run, P);
    int x[U];                              // experts of the run's pairs; kept over everything below where they are no more than that
    auto load = [&](int q) {
#pragma unroll
        for (int i = 0; i < U; ++i) x[i] = expert_of(pair_expert, q + 32 * i + lane, p1, E);
    };
    const bool once = run <= 32 * U;
    if (once) load(p0);
    if (counts) {
        for (int i = threadIdx.x; i < E; i += threads) count[i] = __ldg(counts + i);
    } else {                               // (COUNT_FROM is such that the run is loaded)
        __syncthreads();
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const int p = p0 + 32 * i + lane;
            if (x[i] >= 0) atomicAdd(count + x[i], 1);
            else if (blockIdx.x == 0 && p < p1) {
                place[p] = make_int2(-1, -1);
                if (x[i] == BAD_EXPERT) atomicCAS(err, DEV_OK, DEV_BAD_INDEX);
            }
        }
    }
    __syncthreads();
    int rows = 0, tiles = 0;               // of the experts before
    for (int e0 = 0; e0 < E; e0 += threads) {
        const int e = e0 + threadIdx.x, c = e < E ? count[e] : 0;
        const int r = (c + 7) & ~7, t = (c + (1 << tile_log2) - 1) >> tile_log2;
        int ri = r, ti = t;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int a = __shfl_up_sync(0xffffffffu, ri, o), b = __shfl_up_sync(0xffffffffu, ti, o);
            if (lane >= o) { ri += a; ti += b; }
        }
        if (lane == 31) { sum_rows[warp] = ri; sum_tiles[warp] = ti; }
        __syncthreads();
        const int wr = lane < W ? sum_rows[lane] : 0, wt = lane < W ? sum_tiles[lane] : 0;
        if (e < E) {
            start[e] = rows + ri - r;
            tile0[e] = tiles + ti - t;
        }
        const int br = __reduce_add_sync(0xffffffffu, lane < warp ? wr : 0), bt = __reduce_add_sync(0xffffffffu, lane < warp ? wt : 0);
        if (e < E) { start[e] += br; tile0[e] += bt; }
        rows += __reduce_add_sync(0xffffffffu, wr);
        tiles += __reduce_add_sync(0xffffffffu, wt);
        __syncthreads();
    }
    if (blockIdx.x == 0 && warp == 0) {
        // how the tiles are shared out (cut_of): a number of parts per lane
        const int all = tiles * row_tiles, most = most_parts(all, kts, n);
        const int best = __reduce_min_sync(0xffffffffu, lane < most ? cut_cost(kts, lane + 1) * MAX_PARTS + lane : 0x7fffffff);
        const Cut c = cut_of(all, kts, n, best % MAX_PARTS + 1);
        if (lane == 0) *work = make_int4(c.tiles, c.cut, c.ctas, 0);
    }
    for (int e = blockIdx.x; e < E; e += gridDim.x) {
        const int c = count[e];
        if (!c) continue;
        int k = 0;
        for (int q = p0; q < p1; q += 32 * U) {
            if (!once) load(q);
#pragma unroll
            for (int i = 0; i < U; ++i) k += x[i] == e;
        }
        k = __reduce_add_sync(0xffffffffu, k);
        __syncthreads();                   // (what the expert before left there is read)
        if (lane == 0) before[warp] = k;
        __syncthreads();
        int at = __reduce_add_sync(0xffffffffu, lane < warp ? before[lane] : 0);
        const int s = start[e], t0 = tile0[e];
        for (int q = p0; q < p1; q += 32 * U) {
            if (!once) load(q);
#pragma unroll
            for (int i = 0; i < U; ++i) {
                if (q + 32 * i >= p1) break;
                const unsigned all = __ballot_sync(0xffffffffu, x[i] == e);
                if (x[i] == e) {
                    const int r = at + __popc(all & ((1u << lane) - 1)), p = q + 32 * i + lane;
                    place[p] = make_int2(s + r, (t0 + (r >> tile_log2)) * tile_groups * 128 + (r & ((1 << tile_log2) - 1)));
                    out_row[s + r] = p;
                }
                at += __popc(all);
            }
        }
        for (int i = threadIdx.x; i << tile_log2 < c; i += threads)
            tab[t0 + i] = make_int4(e, s + (i << tile_log2), min(1 << tile_log2, c - (i << tile_log2)), (t0 + i) * tile_groups);
    }
}
// threads of the grouping block: the instructions of all its warps are what the launch waits for (2,048 pairs: 1024 threads 8.7 us, 256 5.6)
int group_threads(int pairs) { return pairs < COUNT_FROM ? 256 : GROUP_THREADS; }
static_assert(COUNT_FROM - 1 <= 256 * 16, "a warp's run of pairs is counted from registers");
constexpr int MAX_EXPERTS = 4000;          // three words each in the 48 KB of shared memory that a launch may have without asking

// How the tiles of one matrix on pairs of SMs are shared out, and what that takes by the model below: cycles.
struct Shared { Cut cut; long long cycles; };
Shared share_out(int tiles, int width, int kts, int n) {
    const int most = most_parts(tiles, kts, n);
    int parts = 1;
    for (int q = 2; q <= most; ++q)
        if (cut_cost(kts, q) < cut_cost(kts, parts)) parts = q;
    const Cut c = cut_of(tiles, kts, n, parts);
    long long steps = static_cast<long long>(tiles / n) * kts;
    if (c.cut && tiles < n) steps = cut_cost(kts, parts);
    else if (c.cut) steps += over_cost(c.cut, kts, c.ctas);
    else if (tiles % n) steps += kts;
    // A step brings 16 KB of weights and 64 bytes a token into a CTA's shared memory and out again, 128 bytes a cycle; results leave at 18 cycles a
    // token. (512 x 4096 x 4096: tiles of 256 tokens 19.4 us, of 192 17.9, of 128 16.9.)
    return {c, steps * (256 + width) + 18ll * width};
}
int round32(int n) { return (n + 31) & ~31; }

size_t align256(size_t n) { return (n + 255) & ~static_cast<size_t>(255); }

// What a call keeps in its workspace, and where.
struct Plan {
    int    kts, rts, row_tiles, img_rows, groups, nt, tile_w, tile_groups, tiles_m, max_tiles, n_counters;
    Cut    share;                  // tiles of one matrix
    size_t img, sf, counters, part, place, out_row, tab, work, counts, bytes;
};
Plan plan_of(int rows, int experts, int K, int N) {
    Plan p{};
    p.kts = (K + 127) / 128;
    p.rts = (N + 127) / 128;
    const long long most = experts ? rows + 7ll * (experts < rows ? experts : rows) : rows;
    p.img_rows = static_cast<int>((most + 7) & ~7ll);
    const int per = experts ? (rows + experts - 1) / experts : rows;
    p.nt = per <= 32 ? 32 : per <= 64 ? 64 : per <= 128 ? 128 : 256;
    bool pairs = p.nt == 256;
    p.row_tiles = pairs ? (p.rts + 1) / 2 : p.rts;
    p.tiles_m = (rows + p.nt - 1) / p.nt;
    p.tile_w = p.nt;
    p.share = Cut{p.tiles_m * p.row_tiles, 0, 0};
    if (pairs && !experts) {
        long long least = 1ll << 62;
        const int first = p.tiles_m;
        for (int m = first; m <= 4 * first && m <= first + 8; ++m) {
            const int w = round32((rows + m - 1) / m), tiles_m = (rows + w - 1) / w;
            const Shared s = share_out(tiles_m * p.row_tiles, w, p.kts, ctx().sm_count / 2);
            if (s.cycles < least) { least = s.cycles; p.tiles_m = tiles_m; p.tile_w = w; p.share = s.cut; }
        }
        // Or tiles of 128 rows x 128 tokens at the most on single SMs, whose launch and first copies take 4 us less (us, pairs / single SMs: 256 x 4096 x 4096
        // 15.3 / 13.2, 512 x 4096 x 4096 17.4 / 14.9, 300 x 2816 x 1408 15.0 / 9.7; two rounds of tiles: 600 x 4096 x 4096 18.3 on pairs)
        const int m = (rows + 127) / 128, w = ((rows + m - 1) / m + 7) & ~7, tiles_m = (rows + w - 1) / w;
        if (mx_mid_ns(static_cast<long long>(tiles_m) * p.rts, p.kts, w) < least * 100 / 185 + 4000) {
            pairs = false;
            p.nt = 128; p.tile_w = w; p.tiles_m = tiles_m; p.row_tiles = p.rts;
            p.share = Cut{tiles_m * p.rts, 0, 0};
        }
    }
    p.n_counters = pairs ? mx_pair_counters() : 0;
    p.tile_groups = (p.tile_w + 127) / 128;
    p.max_tiles = experts ? rows / p.tile_w + (experts < rows ? experts : rows) : p.tiles_m;
    p.groups = p.max_tiles * p.tile_groups;
    size_t at = 0;
    auto take = [&](size_t n) { const size_t here = at; at += align256(n); return here; };
    p.img = take(static_cast<size_t>(p.kts) * p.img_rows * 128);
    p.sf = take(static_cast<size_t>(p.kts) * p.groups * SF_TILE);
    p.counters = take(p.n_counters * sizeof(unsigned));
    p.part = take(pairs ? mx_pair_part_bytes() : 0);
    if (experts) {
        p.place = take(static_cast<size_t>(rows) * sizeof(int2));
        p.out_row = take(static_cast<size_t>(p.img_rows) * 4);
        p.tab = take(static_cast<size_t>(p.max_tiles) * sizeof(int4));
        p.work = take(sizeof(int4));
        p.counts = take(static_cast<size_t>(experts) * 4);
    }
    p.bytes = at;
    return p;
}

template <bool GROUPED>
int launch_product(const float* x, int x_rows, const uint8_t* packed, const int* pair_expert, const int* pair_row, int rows, int experts, float* y, int K, int N,
                   uint8_t* ws, cudaStream_t st) {
    if (mx_small_takes(rows, GROUPED)) return launch_mx_small(x, x_rows, packed, pair_expert, pair_row, rows, experts, y, K, N, st);
    const Plan p = plan_of(rows, GROUPED ? experts : 0, K, N);
    Context& c = ctx();
    MxArgs a{};
    a.q = packed;
    a.sfa = packed + static_cast<size_t>(GROUPED ? experts : 1) * p.rts * p.kts * Q_TILE;
    a.img = ws + p.img; a.sfb = ws + p.sf; a.y = y;
    a.M = rows; a.N = N; a.kts = p.kts; a.rts = p.rts; a.img_rows = p.img_rows; a.groups = p.groups; a.tile_w = p.tile_w; a.tiles_m = p.tiles_m; a.tile_groups = p.tile_groups; a.row_tiles = p.row_tiles;
    a.part = reinterpret_cast<float*>(ws + p.part); a.counters = reinterpret_cast<unsigned*>(ws + p.counters); a.err = c.d_err;
    int2* place = nullptr;
    const int units = c.sm_count / 2;
    int rc;
    if (GROUPED) {
        place = reinterpret_cast<int2*>(ws + p.place);
        a.out_row = reinterpret_cast<int*>(ws + p.out_row);
        a.tab = reinterpret_cast<int4*>(ws + p.tab);
        a.work = reinterpret_cast<int4*>(ws + p.work);
        const dim3 grid(experts < c.sm_count ? experts : c.sm_count);
        int* counts = reinterpret_cast<int*>(ws + p.counts);
        if (rows >= COUNT_FROM) {
            rc = launch_early(mx_count_kernel, grid, GROUP_THREADS, 0, st, pair_expert, rows, experts, place, counts, c.d_err);
            c.launches++;
            if (rc) return rc;
        }
        rc = launch_early(mx_group_kernel, grid, group_threads(rows), 3 * static_cast<size_t>(experts) * sizeof(int), st, pair_expert, rows, experts, __builtin_ctz(p.tile_w), p.tile_groups,
                          static_cast<const int*>(rows >= COUNT_FROM ? counts : nullptr), place, reinterpret_cast<int*>(ws + p.out_row), reinterpret_cast<int4*>(ws + p.tab),
                          reinterpret_cast<int4*>(ws + p.work), p.row_tiles, p.kts, units, c.d_err);
        c.launches++;
        if (rc) return rc;
    }
    a.dense = p.share;
    rc = launch_act<GROUPED>(rows, p.kts, st, x, x_rows, K, p.kts, rows, ActDst{ws + p.img, ws + p.sf, p.img_rows, p.groups, p.tile_w, p.tile_groups}, pair_row, static_cast<const int2*>(place),
                             GROUPED ? reinterpret_cast<int*>(ws + p.out_row) : nullptr, reinterpret_cast<unsigned*>(ws + p.counters), p.n_counters, c.d_err);
    c.launches++;
    if (rc) return rc;
    CUtensorMap map;
    if (!mx_weights_map(&map, a.q, static_cast<size_t>(GROUPED ? experts : 1) * p.rts * p.kts)) return LAPLACE_ERR_CUDA;
    if (p.nt == 256) return launch_mx_pair(map, a, GROUPED, st);
    return launch_mx_mid(map, a, p.nt, GROUPED ? static_cast<long long>(experts < rows ? experts : rows) * p.rts : p.share.tiles, GROUPED, st);
}

// Limits of a call. Tiles of weights: the tensor map counts their rows of 64 bytes in 31 bits. Rows: token tiles times row tiles are counted in 32 bits.
long long tiles_of(int n) { return (n + 127ll) / 128; }
bool too_large(long long experts, int N, int K) { return experts > 0xffffff || experts * tiles_of(N) > 0xffffff || experts * tiles_of(N) * tiles_of(K) > 0xffffff; }
bool too_many(long long rows, long long experts, int N) { return rows > 1 << 24 || (rows / 32 + experts + 1) * tiles_of(N) > 0x3fffffffll; }
int bad_shape(const char* what, int K, int N, long long experts) {
    if (K <= 0 || N <= 0 || experts <= 0 || K % 32) return fail(LAPLACE_ERR_ARG, "%s: K=%d (a positive multiple of 32) N=%d experts=%lld", what, K, N, experts);
    if (too_large(experts, N, K)) return fail(LAPLACE_ERR_LIMIT, "%s: %lld x %d x %d values are more than one call takes", what, experts, N, K);
    return LAPLACE_OK;
}
bool misaligned(const void* p, unsigned n) { return reinterpret_cast<uintptr_t>(p) % n != 0; }

}  // namespace

int launch_mxfp4_dequantize(const uint8_t* w, float* dst, long long n, cudaStream_t st) {
    const long long blocks = n / 32, grid = (blocks + DB - 1) / DB;
    if (grid > 0x7fffffffll) return fail(LAPLACE_ERR_LIMIT, "dequantize: n=%lld", n);
    ctx().launches++;
    return launch_early(mxfp4_dequantize_kernel, dim3(static_cast<unsigned>(grid)), 256, 0, st, w, dst, blocks);
}

}  // namespace lp

using namespace lp;

extern "C" {

#define MX_READY() if (!ctx().ready) return fail(LAPLACE_ERR_STATE, "laplace_cuda_init has not been called (or found no GPU)")
#define MX_STREAM(s) ((s) ? static_cast<cudaStream_t>(s) : ctx().stream)

int laplace_cuda_mxfp4_quantize_dev(const void* x, uint32_t x_type, uint8_t* w, long long n, void* stream) {
    MX_READY();
    if (x_type != 0 && x_type != 1 && x_type != 30) return LAPLACE_UNSUPPORTED;
    if (n == 0) return LAPLACE_OK;
    if (!x || !w || n < 0 || n % 32) return fail(LAPLACE_ERR_ARG, "mxfp4_quantize: n=%lld is not a multiple of 32, or a null pointer", n);
    if (misaligned(x, 16)) return fail(LAPLACE_ERR_ARG, "mxfp4_quantize: x must be 16-byte aligned");
    cudaStream_t st = MX_STREAM(stream);
    return x_type == 0 ? launch_quantize<float>(x, w, n / 32, st) : x_type == 1 ? launch_quantize<__half>(x, w, n / 32, st) : launch_quantize<__nv_bfloat16>(x, w, n / 32, st);
}

size_t laplace_cuda_mxfp4_packed_size(int n_experts, int N, int K) {
    if (n_experts <= 0 || N <= 0 || K <= 0 || K % 32 || too_large(n_experts, N, K)) return 0;
    return static_cast<size_t>(n_experts * tiles_of(N) * tiles_of(K)) * (Q_TILE + SF_TILE);
}

int laplace_cuda_mxfp4_pack_dev(const uint8_t* w, uint8_t* packed, int n_experts, int N, int K, void* stream) {
    MX_READY();
    if (const int rc = bad_shape("mxfp4_pack", K, N, n_experts)) return rc;
    if (!w || !packed || misaligned(packed, 128)) return fail(LAPLACE_ERR_ARG, "mxfp4_pack: null pointer, or packed is not 128-byte aligned");
    const int rts = (N + 127) / 128, kts = (K + 127) / 128;
    // row tiles on the grid's second axis, 65535 a launch: whole experts at a time, or (one expert with more tiles) refused
    if (rts > 65535) return fail(LAPLACE_ERR_LIMIT, "mxfp4_pack: N=%d", N);
    const int step = 65535 / rts;
    const size_t n_tiles = static_cast<size_t>(n_experts) * rts * kts;
    for (int e = 0; e < n_experts; e += step) {
        const int here = n_experts - e < step ? n_experts - e : step;
        const size_t t0 = static_cast<size_t>(e) * rts * kts;
        mxfp4_pack_kernel<<<dim3(kts, rts * here), 512, 0, MX_STREAM(stream)>>>(w + static_cast<size_t>(e) * N * (K / 32) * 17, packed + t0 * Q_TILE,
                                                                                packed + n_tiles * Q_TILE + t0 * SF_TILE, N, K, rts, kts);
        ctx().launches++;
    }
    mxfp4_packed_kernel<<<1, 32, 0, MX_STREAM(stream)>>>();
    ctx().launches++;
    return cuda_check(cudaGetLastError(), "mxfp4_pack launch");
}

size_t laplace_cuda_mxfp4_workspace_size(int rows, int n_experts, int K, int N) {
    if (!ctx().ready || rows <= 0 || n_experts < 0 || K <= 0 || N <= 0 || K % 32 || mx_small_takes(rows, n_experts > 0)) return 0;
    if (n_experts > MAX_EXPERTS || too_large(n_experts ? n_experts : 1, N, K) || too_many(rows, n_experts ? n_experts : 1, N)) return 0;
    return plan_of(rows, n_experts, K, N).bytes;
}

int laplace_cuda_mxfp4_last_kernel(void) { return ctx().last_mx; }

int laplace_cuda_mxfp4_gemm_dev(const float* x, const uint8_t* packed, float* y, int M, int K, int N, void* workspace, size_t workspace_bytes, void* stream) {
    MX_READY();
    if (const int rc = bad_shape("mxfp4_gemm", K, N, 1)) return rc;
    if (M < 0) return fail(LAPLACE_ERR_ARG, "mxfp4_gemm: M=%d", M);
    if (M == 0) return LAPLACE_OK;
    if (too_many(M, 1, N)) return fail(LAPLACE_ERR_LIMIT, "mxfp4_gemm: M=%d", M);
    const size_t need = laplace_cuda_mxfp4_workspace_size(M, 0, K, N);
    if (!x || !packed || !y || (need && !workspace)) return fail(LAPLACE_ERR_ARG, "mxfp4_gemm: null pointer");
    if (misaligned(x, 16) || misaligned(packed, 128) || misaligned(workspace, 256) || misaligned(y, 4))
        return fail(LAPLACE_ERR_ARG, "mxfp4_gemm: x must be 16-byte, packed 128-byte, workspace 256-byte aligned");
    if (workspace_bytes < need) return fail(LAPLACE_ERR_ARG, "mxfp4_gemm: workspace of %zu bytes, %zu needed", workspace_bytes, need);
    return launch_product<false>(x, M, packed, nullptr, nullptr, M, 1, y, K, N, static_cast<uint8_t*>(workspace), MX_STREAM(stream));
}

int laplace_cuda_mxfp4_moe_grouped_dev(const float* x, int x_rows, const uint8_t* packed, const int* pair_expert, const int* pair_row, int n_pairs, int n_experts_total, float* y,
                                       int K, int N, void* workspace, size_t workspace_bytes, void* stream) {
    MX_READY();
    if (const int rc = bad_shape("mxfp4_moe_grouped", K, N, n_experts_total)) return rc;
    if (n_pairs < 0 || x_rows < 0) return fail(LAPLACE_ERR_ARG, "mxfp4_moe_grouped: n_pairs=%d x_rows=%d", n_pairs, x_rows);
    if (n_pairs == 0) return LAPLACE_OK;
    if (too_many(n_pairs, n_experts_total, N)) return fail(LAPLACE_ERR_LIMIT, "mxfp4_moe_grouped: n_pairs=%d", n_pairs);
    if (n_experts_total > MAX_EXPERTS) return fail(LAPLACE_ERR_LIMIT, "mxfp4_moe_grouped: %d experts, %d at most", n_experts_total, MAX_EXPERTS);
    const size_t need = laplace_cuda_mxfp4_workspace_size(n_pairs, n_experts_total, K, N);
    if (!x || !packed || !pair_expert || !y || (need && !workspace)) return fail(LAPLACE_ERR_ARG, "mxfp4_moe_grouped: null pointer");
    if (!pair_row && x_rows < n_pairs) return fail(LAPLACE_ERR_ARG, "mxfp4_moe_grouped: %d rows of x for %d pairs", x_rows, n_pairs);
    if (misaligned(x, 16) || misaligned(packed, 128) || misaligned(workspace, 256) || misaligned(y, 4) || misaligned(pair_expert, 4) || misaligned(pair_row, 4))
        return fail(LAPLACE_ERR_ARG, "mxfp4_moe_grouped: x must be 16-byte, packed 128-byte, workspace 256-byte aligned");
    if (workspace_bytes < need) return fail(LAPLACE_ERR_ARG, "mxfp4_moe_grouped: workspace of %zu bytes, %zu needed", workspace_bytes, need);
    return launch_product<true>(x, x_rows, packed, pair_expert, pair_row, n_pairs, n_experts_total, y, K, N, static_cast<uint8_t*>(workspace), MX_STREAM(stream));
}

}  // extern "C"
