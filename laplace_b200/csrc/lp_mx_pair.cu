// lp_mx_pair.cu - products of packed MXFP4 weights and quantized rows on pairs of SMs (cta_group::2), tiles of 256 weight rows x up to 256 tokens: more
// than 128 rows of one matrix where the model of its time is below that of single SMs (plan_of in lp_mx.cu), or experts with more than 128 pairs on average. Formats and layouts: lp_mx.cu, the instruction: lp_mx_mma.cuh.
//
// Either CTA of a pair has its 128 weight rows and half of the tokens in shared memory. What bounds one CTA with 128 x 256 is the way from L2, 41 KB a
// k step of 128 that takes the tensor core 512 cycles; a pair's CTAs take 25 KB each.
//
// Work. Tiles over G pairs, whole ones one after the other; the last ones, where they do not come out even, may be cut: their k steps, in tile
// order, go in equal runs to the pairs (cut_of in lp_mx.cuh says when that pays). Of a
// cut tile's pairs the last one to arrive (a counter) keeps its sums in registers; the others leave theirs in the workspace, on which
// it waits - they are running, so it does not wait long - and it adds all up in the order of k: the result does not depend on who was last.
//
// Roles by warp: 0 copies, 1 MMA issue in the even CTA (owns the TMEM), word of the filled stages in the odd one, 4-11 drain (lane =
// weight row). All waits are bounded; a wait that gives up raises the status word and the roles leave their loops.
//
// 2048 x 14336 x 4096: 540 cycles a step (512 are the tensor core's), 240 Gop in 84 us in the first milliseconds, 102 once the card's power limit holds the clock at 1.46 GHz; with
// the quantizer 107 and 127. One CTA with 128 x 256 took 610 cycles a step. 512 x 4096 x 14336, in a graph, quantizer and all, 32 us and (1.73 GHz) 36, 1000 x 4096 x 14336 55 at first.
#include "lp_mx.cuh"
#include "lp_mx_mma.cuh"
#include "lp_tc.cuh"

namespace lp {
namespace {

using namespace mx;
using namespace tc;

constexpr int THREADS = 384;
constexpr int DRAIN = 256;                     // threads of the drain: two warps per quadrant of TMEM lanes
constexpr int A_STAGE = 128 * 128;             // 128 rows x 128 values, a byte each after the copy
constexpr uint32_t SF_COL = 480;               // TMEM columns of the scales: two sets of 16 (4 of the weights, up to 8 of the activations)

constexpr int NT = 256;                        // tokens of a tile
struct Lay {
    static constexpr int B_STAGE = NT / 2 * 128;
    static constexpr int GROUPS = (NT + 127) / 128;       // 128-row groups of scales
    static constexpr int STAGE = A_STAGE + B_STAGE + SF_TILE + GROUPS * SF_TILE;
    static constexpr int STAGES = (226 * 1024 - 1024) / STAGE;
    static constexpr uint32_t A = 0, B = A + STAGES * A_STAGE, SFA = B + STAGES * B_STAGE, SFB = SFA + STAGES * SF_TILE, BAR = SFB + STAGES * GROUPS * SF_TILE;
    static constexpr uint32_t FULL = BAR, EMPTY = FULL + 8 * STAGES, TFULL = EMPTY + 8 * STAGES, TEMPTY = TFULL + 16, PTR = TEMPTY + 16, ABORT = PTR + 4, SAY = ABORT + 4,
                              BYTES = SAY + 8 + 1024;
    static_assert(BYTES <= 227 * 1024, "shared memory");
};

// rt: row tile, of 256 rows
struct Seg { int expert, rt, row0, n, group, k0, k1, cut; };      // group: first 128-row group of its scales; cut: number of the cut tile, -1 for a whole one
struct Work { int tiles, cut, ctas; long long units; };

__device__ __forceinline__ long long cut_start(const Work& w, int c) { return w.units * c / w.ctas; }
// the unit whose run holds step u
__device__ __forceinline__ int cut_owner(const Work& w, long long u) {
    int c = static_cast<int>(u * w.ctas / w.units);
    while (c + 1 < w.ctas && cut_start(w, c + 1) <= u) ++c;
    while (c > 0 && cut_start(w, c) > u) --c;
    return c;
}
// Where a unit leaves its part of a tile: it has at most one that begins inside a tile and one that begins a tile.
__device__ __forceinline__ int slot_of(int unit, bool begins) { return 2 * unit + begins; }

template <bool GROUPED>
__device__ __forceinline__ void tile_at(const MxArgs& a, int t, Seg& s) {
    if (GROUPED) {
        const int4 e = __ldg(a.tab + t / a.row_tiles);
        s.rt = t % a.row_tiles;
        s.expert = e.x; s.row0 = e.y; s.n = e.z; s.group = e.w;
    } else {
        s.rt = t / a.tiles_m;
        s.expert = 0;
        s.row0 = (t % a.tiles_m) * a.tile_w;
        s.group = (t % a.tiles_m) * a.tile_groups;
        s.n = min(a.tile_w, a.M - s.row0);
    }
}
// A unit's work piece by piece, in the order in which every role walks it.
template <bool GROUPED>
struct Walk {
    const MxArgs& a;
    const Work w;
    long long u, u1;
    int next;
    __device__ __forceinline__ Walk(const MxArgs& args, const Work& work) : a(args), w(work) {
        const int c = blockIdx.x / 2;
        u = c < w.ctas ? cut_start(w, c) : 0;
        u1 = c < w.ctas ? cut_start(w, c + 1) : 0;
        next = w.cut + c;
    }
    __device__ __forceinline__ bool operator()(Seg& s) {
        if (u < u1) {
            const int t = static_cast<int>(u / a.kts);
            const long long base = static_cast<long long>(t) * a.kts;
            tile_at<GROUPED>(a, t, s);
            s.k0 = static_cast<int>(u - base);
            s.k1 = static_cast<int>(min(u1 - base, static_cast<long long>(a.kts)));
            s.cut = s.k0 == 0 && s.k1 == a.kts ? -1 : t;
            u = base + s.k1;
            return true;
        }
        if (next >= w.tiles) return false;
        tile_at<GROUPED>(a, next, s);
        s.k0 = 0; s.k1 = a.kts; s.cut = -1;
        next += gridDim.x / 2;
        return true;
    }
};

// Whether any thread of the barrier's says so; all of them learn the same.
template <int THREADS>
__device__ __forceinline__ bool any_of(int bar, bool mine) {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbarrier.cta.red.or.pred q, %2, %3, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
                 : "=r"(r) : "r"(static_cast<uint32_t>(mine)), "r"(bar), "n"(THREADS) : "memory");
    return r != 0;
}

template <bool GROUPED>
__global__ void __launch_bounds__(THREADS, 1) mx_pair_kernel(const __grid_constant__ CUtensorMap map, const MxArgs a) {
    using L = Lay;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t sb = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* smem = smem_raw + (sb - smem_u32(smem_raw));
    volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::ABORT);
    const int warp = threadIdx.x >> 5, rank = static_cast<int>(pair_rank());
    if (threadIdx.x == 0) {
        for (int i = 0; i < L::STAGES; ++i) { mbar_init(sb + L::FULL + 8 * i, 2 - rank); mbar_init(sb + L::EMPTY + 8 * i, 1); }      // the even CTA's: its own copies and word of the other's
        mbar_init(sb + L::TFULL, 1);
        mbar_init(sb + L::TEMPTY, 2 * DRAIN / 32);
        *abort_flag = 0;
        fence_barrier_init();
        asm volatile("prefetch.tensormap [%0];" :: "l"(&map) : "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" :: "r"(sb + L::PTR), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    fence_before();
    __syncthreads();
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");        // both CTAs' barriers are there before either arrives on them
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    fence_after();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(smem + L::PTR);
    // Experts: the table of token tiles is made by the kernels before this one. One matrix: the weights may be copied meanwhile; the quantizer
    // before this kernel lets it start only after it has itself waited for what is before it in the stream, weights' writers included.
    if (GROUPED || warp != 0) asm volatile("griddepcontrol.wait;" ::: "memory");
    const int3 cut = GROUPED ? make_int3(a.work->x, a.work->y, a.work->z) : make_int3(a.dense.tiles, a.dense.cut, a.dense.ctas);
    const Work w{cut.x, cut.y, cut.z, static_cast<long long>(cut.y) * a.kts};

    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");       // 128 x 64 + 256 x 216 of 384 x 168 registers
    if (warp == 0 && elect_one()) {
        // of this CTA: its row tile (of an odd number the last one twice, the second time for nothing), its part of the tokens
        auto tile_of = [&](const Seg& s, int kt) { return (static_cast<size_t>(s.expert) * a.rts + min(s.rt * 2 + rank, a.rts - 1)) * a.kts + kt; };
        auto rows_of = [&](const Seg& s, int& first) {
            const int n8 = (s.n + 7) & ~7, half = ((s.n + 31) & ~31) / 2;
            first = rank * half;
            return rank ? max(n8 - half, 0) : min(n8, half);
        };
        auto weights = [&](int st, const Seg& s, int kt) {
            int first;
            const int groups = (s.n + 127) >> 7;
            const uint32_t bar = sb + L::FULL + 8 * st;
            mbar_expect_tx(bar, Q_TILE + SF_TILE + rows_of(s, first) * 128 + groups * SF_TILE);
            const size_t tile = tile_of(s, kt);
            tma_load_2d(sb + L::A + st * A_STAGE, &map, 0, static_cast<int>(tile * 128), bar);
            bulk_g2s(sb + L::SFA + st * SF_TILE, a.sfa + tile * SF_TILE, SF_TILE, bar);
        };
        auto tokens = [&](int st, const Seg& s, int kt) {
            int first;
            const int rows = rows_of(s, first), groups = (s.n + 127) >> 7;
            const uint32_t bar = sb + L::FULL + 8 * st;
            if (rows) bulk_g2s(sb + L::B + st * L::B_STAGE, a.img + (static_cast<size_t>(kt) * a.img_rows + s.row0 + first) * 128, rows * 128, bar);
            bulk_g2s(sb + L::SFB + st * L::GROUPS * SF_TILE, a.sfb + (static_cast<size_t>(kt) * a.groups + s.group) * SF_TILE, groups * SF_TILE, bar);
        };
        int early = 0;
        if (!GROUPED) {
            Walk<GROUPED> walk(a, w);
            Seg s;
            while (early < L::STAGES && walk(s))
                for (int kt = s.k0; kt < s.k1 && early < L::STAGES; ++kt) weights(early++, s, kt);
            asm volatile("griddepcontrol.wait;" ::: "memory");
        }
        Walk<GROUPED> walk(a, w);
        Seg s;
        int it = 0;
        bool ok = true;
        while (ok && walk(s))
            for (int kt = s.k0; kt < s.k1; ++kt, ++it) {
                const int st = it % L::STAGES, round = it / L::STAGES;
                if (round && !wait_or_abort<false>(sb + L::EMPTY + 8 * st, (round - 1) & 1, abort_flag, a.err, DEV_TIMEOUT_EMPTY)) { ok = false; break; }
                if (it >= early) weights(st, s, kt);
                tokens(st, s, kt);
            }
        if (!ok)                                        // what is in flight lands before the CTA goes
            for (int i = 0; i < 1000; ++i) __nanosleep(1000);
    } else if (warp == 1 && rank == 0 && elect_one()) {
        Walk<GROUPED> walk(a, w);
        Seg s;
        int it = 0;
        bool ok = true;
        for (int seg = 0; ok && walk(s); ++seg) {
            const int n = (s.n + 31) & ~31, groups = (s.n + 127) >> 7;
            if (seg && !wait_pair(sb + L::TEMPTY, (seg - 1) & 1, abort_flag, a.err, DEV_TIMEOUT_TMEM)) { ok = false; break; }
            fence_after();
            for (int kt = s.k0; kt < s.k1; ++kt, ++it) {
                const int st = it % L::STAGES;
                if (!wait_pair(sb + L::FULL + 8 * st, (it / L::STAGES) & 1, abort_flag, a.err, DEV_TIMEOUT_FULL)) { ok = false; break; }
                fence_after();
                const uint32_t sfa = tmem + SF_COL + 16 * (it & 1), sfb = sfa + 4;
                copy_scales<2>(sfa, sb + L::SFA + st * SF_TILE);
                for (int g = 0; g < groups; ++g) copy_scales<2>(sfb + 4 * g, sb + L::SFB + (st * L::GROUPS + g) * SF_TILE);
                const uint64_t ad = smem_desc_sw128(sb + L::A + st * A_STAGE), bd = smem_desc_sw128(sb + L::B + st * L::B_STAGE);
#pragma unroll
                for (int ks = 0; ks < 4; ++ks) mma_mx<2>(tmem, ad + 2 * ks, bd + 2 * ks, idesc_mx<2>(n, ks), sfa, sfb, kt != s.k0 || ks);
                commit_pair(sb + L::EMPTY + 8 * st);
            }
            if (ok) commit_pair(sb + L::TFULL);
        }
        if (!ok)                                        // what has been issued ends before the CTA goes
            for (int i = 0; i < 1000; ++i) __nanosleep(1000);
    } else if (warp == 1 && rank == 1 && elect_one()) {      // (elect takes the whole warp: no lane of the even CTA's may come here)
        // the odd CTA: tells the even one of its stages as they fill
        Walk<GROUPED> walk(a, w);
        Seg s;
        int it = 0;
        bool ok = true;
        while (ok && walk(s))
            for (int kt = s.k0; kt < s.k1; ++kt, ++it) {
                const int st = it % L::STAGES;
                if (!wait_or_abort<true>(sb + L::FULL + 8 * st, (it / L::STAGES) & 1, abort_flag, a.err, DEV_TIMEOUT_FULL)) { ok = false; break; }
                arrive_cluster(map_to_rank(sb + L::FULL + 8 * st, 0));
            }
    }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
        Walk<GROUPED> walk(a, w);
        Seg s;
        const int lane = threadIdx.x & 31, id = threadIdx.x - 128, half = id >> 7, r = id & 127;      // r: weight row of the tile
        const uint32_t quadrant = static_cast<uint32_t>(warp & 3) * 32u << 16;
        volatile int* say = reinterpret_cast<volatile int*>(smem + L::SAY);
        for (int seg = 0; walk(s); ++seg) {
            const bool ok = wait_or_abort<false>(sb + L::TFULL, seg & 1, abort_flag, a.err, DEV_TIMEOUT_MMA);
            // the warps meet at cut tiles (which come first): they leave together or not at all
            if (s.cut >= 0 ? any_of<DRAIN>(1, !ok) : !ok) break;
            __syncwarp();
            fence_after();
            const int rt = s.rt * 2 + rank, col = rt * 128 + r, unit = blockIdx.x / 2;
            // Columns 32 half + 64 j .. + 31: all into registers first, so that the next tile's products do not wait for what follows.
            constexpr int J = NT / 64;
            float v[J][32];
#pragma unroll
            for (int j = 0; j < J; ++j)
                if (32 * half + 64 * j < s.n) ld32(tmem + quadrant + 32 * half + 64 * j, v[j]);
            wait_ld();
            fence_before();
            __syncwarp();
            if (lane == 0) {
                if (rank == 0) mbar_arrive(sb + L::TEMPTY);
                else arrive_cluster(map_to_rank(sb + L::TEMPTY, 0));
            }
            const int full = half ? max(0, s.n - 32) : s.n;      // (columns of the tile from this half's first on)
            if (s.cut >= 0) {
                const long long u = static_cast<long long>(s.cut) * a.kts;
                const int first = cut_owner(w, u), pieces = cut_owner(w, u + a.kts - 1) - first + 1;
                unsigned* count = a.counters + 2 * (s.cut * 2 + rank);      // {arrived, written}
                auto part = [&](int c, bool begins) { return a.part + static_cast<size_t>(slot_of(c, begins) * 2 + rank) * (NT * 128) + (half * (8 * 128) + r) * 4; };      // [column / 4][row][4 columns]
                if (id == 0) *say = atomicAdd(count, 1u) == static_cast<unsigned>(pieces - 1);
                named_bar_sync(1, DRAIN);
                const bool last = *say;
                if (!last) {
                    float* q = part(unit, s.k0 == 0);
#pragma unroll
                    for (int j = 0; j < J; ++j)
#pragma unroll
                        for (int i = 0; i < 32; i += 4)
                            if (64 * j + i < full) __stcg(reinterpret_cast<float4*>(q + (64 * j + i) * 128), make_float4(v[j][i], v[j][i + 1], v[j][i + 2], v[j][i + 3]));
                    named_bar_sync(1, DRAIN);
                    if (id == 0) { __threadfence(); atomicAdd(count + 1, 1u); }
                    continue;
                }
                bool there = true;
                if (id == 0) {
                    there = false;
                    for (int i = 0; i < 1 << 22 && !there; ++i) {
                        uint32_t c;
                        asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(c) : "l"(count + 1) : "memory");
                        there = c == static_cast<unsigned>(pieces - 1);
                    }
                    if (!there) { *abort_flag = 1; report_status(a.err, DEV_TIMEOUT_DRAIN); }
                }
                if (any_of<DRAIN>(1, !there)) break;
#pragma unroll
                for (int j = 0; j < J; ++j) {
                    if (64 * j >= full) break;
                    float sum[32];
#pragma unroll
                    for (int i = 0; i < 32; ++i) sum[i] = 0.f;
#pragma unroll 1
                    for (int p = 0; p < pieces; ++p) {
                        if (first + p == unit) {
#pragma unroll
                            for (int i = 0; i < 32; ++i) sum[i] += v[j][i];
                        } else {
                            const float* q = part(first + p, p == 0) + j * (64 * 128);
                            float4 o[8];
#pragma unroll
                            for (int i = 0; i < 8; ++i) o[i] = 64 * j + 4 * i < full ? __ldcg(reinterpret_cast<const float4*>(q + i * 512)) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                            for (int i = 0; i < 8; ++i) { sum[4 * i] += o[i].x; sum[4 * i + 1] += o[i].y; sum[4 * i + 2] += o[i].z; sum[4 * i + 3] += o[i].w; }
                        }
                    }
#pragma unroll
                    for (int i = 0; i < 32; ++i) v[j][i] = sum[i];
                }
            }
#pragma unroll
            for (int j = 0; j < J; ++j) {
                const int c0 = 32 * half + 64 * j, here = min(32, s.n - c0);
                if (here <= 0) break;
                if (GROUPED) {
                    // lane: the row of y that column c0 + lane goes to, -1: to none
                    const int to = lane < here ? __ldg(a.out_row + s.row0 + c0 + lane) : 0;
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        const int m = __shfl_sync(0xffffffffu, to, i);
                        store_if(i < here && m >= 0 && col < a.N, a.y + static_cast<size_t>(m) * a.N + col, v[j][i]);
                    }
                } else if (col < a.N) {
                    float* q = a.y + static_cast<size_t>(s.row0 + c0) * a.N + col;
                    if (here == 32) {
#pragma unroll
                        for (int i = 0; i < 32; ++i) q[static_cast<size_t>(i) * a.N] = v[j][i];
                    } else {
#pragma unroll
                        for (int i = 0; i < 32; ++i)
                            if (i < here) q[static_cast<size_t>(i) * a.N] = v[j][i];
                    }
                }
                __syncwarp();
            }
        }
    }
    __syncwarp();
    fence_before();
    __syncthreads();
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");        // neither CTA leaves while the other may still reach into it
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (warp == 1) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" :: "r"(tmem), "r"(512u) : "memory");
    }
}

template <bool GROUPED>
int launch(const CUtensorMap& map, const MxArgs& a, cudaStream_t st) {
    static bool configured = false;
    if (!configured) {
        const int rc = cuda_check(cudaFuncSetAttribute(mx_pair_kernel<GROUPED>, cudaFuncAttributeMaxDynamicSharedMemorySize, Lay::BYTES), "mx_pair shared memory");
        if (rc) return rc;
        configured = true;
    }
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = 2; attr[1].val.clusterDim.y = 1; attr[1].val.clusterDim.z = 1;
    cfg.gridDim = dim3(ctx().sm_count / 2 * 2); cfg.blockDim = dim3(THREADS); cfg.dynamicSmemBytes = Lay::BYTES; cfg.stream = st; cfg.attrs = attr; cfg.numAttrs = 2;
    ctx().launches++;
    ctx().last_mx = KERNEL_PAIR + 16;
    return cuda_check(cudaLaunchKernelEx(&cfg, mx_pair_kernel<GROUPED>, map, a), "mx_pair launch");
}

}  // namespace

// Parts of cut tiles: two per CTA. Counters: two per cut tile and CTA of a pair, fewer than two tiles a pair.
size_t mx_pair_part_bytes() { return static_cast<size_t>(2 * ctx().sm_count) * NT * 128 * sizeof(float); }
int    mx_pair_counters() { return 4 * ctx().sm_count; }

int launch_mx_pair(const CUtensorMap& map, const MxArgs& a, bool grouped, cudaStream_t st) { return grouped ? launch<true>(map, a, st) : launch<false>(map, a, st); }

}  // namespace lp
