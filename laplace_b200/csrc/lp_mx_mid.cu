// lp_mx_mid.cu - products of packed MXFP4 weights and quantized rows, tiles of 128 weight rows x up to 128 tokens: 9 to 128 rows of one matrix, more where the model
// of its time is below that of the pairs of SMs (plan_of in lp_mx.cu), or experts with up to 128 pairs on average. Formats and layouts: lp_mx.cu, the instruction: lp_mx_mma.cuh.
//
// Bound by the weights' way from memory. A cluster of C CTAs takes tiles number cluster, cluster + clusters, ...; its CTAs share out k where there are
// fewer tiles than SMs, and C is 1 where there are enough. A CTA sends its part of a tile's results into the shared memory of their owners
// - CTA o owns the o-th run of the tokens -, which add the parts in the order of k and write y. (Parts through global memory with a
// counter, the last CTA adding up: 10,000 cycles from the last product to the end, most of it the fence behind the stores and the way
// back; 77 x 2816 x 8448 13.6 us.)
// In a graph over weights from cold memory, quantizer and all: 24 x 14336 x 4096 13.8 us, 77 x 2816 x 8448 10.5, 128 x 4096 x 14336 14.9, 512 x 4096 x 4096 14.9; a kernel that only copies 29 MB
// of weights into shared memory takes 7.5. 2,048 pairs of 128 experts 2048 x 1536 (214 MB) 42 us, 5 TB/s, 46 with grouping and quantizer, 47 to 49 call by call.
//
// Roles by warp: 0 copies, 1 MMA issue (owns the TMEM), 4-11 drain (lane = weight row), sums and output. All waits are bounded; a wait that
// gives up raises the status word and the roles leave their loops.
#include "lp_mx.cuh"
#include "lp_mx_mma.cuh"
#include "lp_tc.cuh"

namespace lp {
namespace {

using namespace mx;
using namespace tc;

constexpr int THREADS = 384;
constexpr int DRAIN_WARPS = 8;                 // two per quadrant of TMEM lanes
constexpr int MAX_STAGES = 10;
constexpr int A_STAGE = 128 * 128;             // 128 rows x 128 values, a byte each after the copy
constexpr uint32_t SF_COL = 256;               // TMEM columns of the scales, behind two accumulators: two sets of 8
constexpr size_t SMEM = 227 * 1024;

struct Fixed {
    uint64_t full[MAX_STAGES], empty[MAX_STAGES], tfull[2], tempty[2], recv, avail;
    uint32_t tmem;
    int      abort;
};
template <int NT> constexpr int stage_bytes() { return A_STAGE + NT * 128 + 2 * SF_TILE; }
// the receiving buffer: per CTA of the cluster its part of the owner's tokens, a multiple of four
template <int NT> constexpr int recv_bytes(int C) { return C == 1 ? 0 : (NT + 4 * C) * 512; }
template <int NT> constexpr int stages_of(int C) {
    const int s = static_cast<int>((SMEM - 1024 - sizeof(Fixed) - recv_bytes<NT>(C)) / stage_bytes<NT>());
    return s < MAX_STAGES ? s : MAX_STAGES;
}

// SPLIT: clusters of C > 1 CTAs. (A kernel of its own for C = 1: the code that either drags along is fetched by every SM of every launch, 0.4 us.)
template <int NT, bool GROUPED, bool SPLIT>
__global__ void __launch_bounds__(THREADS, 1) mx_mid_kernel(const __grid_constant__ CUtensorMap map, const MxArgs a, const int cluster_ctas, const int S) {
    const int C = SPLIT ? cluster_ctas : 1;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t sb = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* smem = smem_raw + (sb - smem_u32(smem_raw));
    const uint32_t off_b = S * A_STAGE, off_sfa = off_b + S * NT * 128, off_sfb = off_sfa + S * SF_TILE, off_recv = off_sfb + S * SF_TILE,
                   off_fixed = off_recv + (SPLIT ? (NT + 4 * C) * 512 : 0);
    Fixed& f = *reinterpret_cast<Fixed*>(smem + off_fixed);
    volatile int* abort_flag = &f.abort;
    auto bar = [&](const uint64_t& b) { return smem_u32(&b); };
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = SPLIT ? static_cast<int>(pair_rank()) : 0;
    if (threadIdx.x == 0) {
        for (int i = 0; i < S; ++i) { mbar_init(bar(f.full[i]), 1); mbar_init(bar(f.empty[i]), 1); }
        for (int i = 0; i < 2; ++i) { mbar_init(bar(f.tfull[i]), 1); mbar_init(bar(f.tempty[i]), DRAIN_WARPS); }
        mbar_init(bar(f.recv), DRAIN_WARPS * C);
        mbar_init(bar(f.avail), DRAIN_WARPS * C);
        f.abort = 0;
        fence_barrier_init();
        asm volatile("prefetch.tensormap [%0];" :: "l"(&map) : "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" :: "r"(smem_u32(&f.tmem)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    fence_before();
    __syncthreads();
    fence_after();
    if (SPLIT) cluster_arrive();                   // barriers are there for the other CTAs; waited for where they are used first
    const uint32_t tmem = f.tmem;
    // Experts: the table of token tiles is made by the kernels before this one. One matrix: the weights may be copied meanwhile; the quantizer
    // before this kernel lets it start only after it has itself waited for what is before it in the stream, weights' writers included.
    if (GROUPED || warp != 0) asm volatile("griddepcontrol.wait;" ::: "memory");
    const int tiles = GROUPED ? a.work->x : a.dense.tiles, clusters = gridDim.x / C, cluster = blockIdx.x / C;
    const int k0 = a.kts * rank / C, k1 = a.kts * (rank + 1) / C;      // every CTA has a step at least: kts >= C

    struct Tile { int expert, rt, row0, n, group; };
    auto tile_at = [&](int t) {
        if (GROUPED) {
            const int4 e = __ldg(a.tab + t / a.rts);
            return Tile{e.x, t % a.rts, e.y, e.z, e.w};
        }
        const int m = t % a.tiles_m, row0 = m * a.tile_w;
        return Tile{0, t / a.tiles_m, row0, min(a.tile_w, a.M - row0), m};      // (up to 128 tokens: a group of scales each)
    };

    if (warp == 0 && elect_one()) {
        auto weights = [&](int st, const Tile& s, int kt) {
            const uint32_t b = bar(f.full[st]);
            const size_t tile = (static_cast<size_t>(s.expert) * a.rts + s.rt) * a.kts + kt;
            mbar_expect_tx(b, Q_TILE + 2 * SF_TILE + ((s.n + 7) & ~7) * 128);
            tma_load_2d(sb + st * A_STAGE, &map, 0, static_cast<int>(tile * 128), b);
            bulk_g2s(sb + off_sfa + st * SF_TILE, a.sfa + tile * SF_TILE, SF_TILE, b);
        };
        int early = 0;
        if (!GROUPED) {
            for (int t = cluster; t < tiles && early < S; t += clusters) {
                const Tile s = tile_at(t);
                for (int kt = k0; kt < k1 && early < S; ++kt) weights(early++, s, kt);
            }
            asm volatile("griddepcontrol.wait;" ::: "memory");
        }
        int st = 0, parity = 1;
        bool ok = true;
        for (int t = cluster; ok && t < tiles; t += clusters) {
            const Tile s = tile_at(t);
            for (int kt = k0; kt < k1; ++kt) {
                if (!wait_or_abort<false>(bar(f.empty[st]), parity, abort_flag, a.err, DEV_TIMEOUT_EMPTY)) { ok = false; break; }
                if (early > 0) --early;            // the ring's first round: its weights are on their way
                else weights(st, s, kt);
                const uint32_t b = bar(f.full[st]);
                bulk_g2s(sb + off_b + st * (NT * 128), a.img + (static_cast<size_t>(kt) * a.img_rows + s.row0) * 128, ((s.n + 7) & ~7) * 128, b);
                bulk_g2s(sb + off_sfb + st * SF_TILE, a.sfb + (static_cast<size_t>(kt) * a.groups + s.group) * SF_TILE, SF_TILE, b);
                if (++st == S) { st = 0; parity ^= 1; }
            }
        }
        if (!ok)                                    // what is in flight lands before the CTA goes
            for (int i = 0; i < 1000; ++i) __nanosleep(1000);
        if (SPLIT) cluster_wait();
    } else if (warp == 1 && elect_one()) {
        int st = 0, parity = 0, i = 0, set = 0;      // set: of TMEM columns for the scales
        bool ok = true;
        for (int t = cluster; ok && t < tiles; t += clusters, ++i) {
            const int acc = i & 1, n = (tile_at(t).n + 15) & ~15;
            if (i >= 2 && !wait_or_abort<true>(bar(f.tempty[acc]), (i / 2 - 1) & 1, abort_flag, a.err, DEV_TIMEOUT_TMEM)) break;
            fence_after();
            for (int kt = k0; kt < k1; ++kt) {
                if (!wait_or_abort<true>(bar(f.full[st]), parity, abort_flag, a.err, DEV_TIMEOUT_FULL)) { ok = false; break; }
                fence_after();
                const uint32_t sfa = tmem + SF_COL + 8 * set, sfb = sfa + 4;
                set ^= 1;
                copy_scales<1>(sfa, sb + off_sfa + st * SF_TILE);
                copy_scales<1>(sfb, sb + off_sfb + st * SF_TILE);
                const uint64_t ad = smem_desc_sw128(sb + st * A_STAGE), bd = smem_desc_sw128(sb + off_b + st * (NT * 128));
#pragma unroll
                for (int ks = 0; ks < 4; ++ks) mma_mx<1>(tmem + acc * 128, ad + 2 * ks, bd + 2 * ks, idesc_mx<1>(n, ks), sfa, sfb, kt != k0 || ks);
                commit(bar(f.empty[st]));
                if (++st == S) { st = 0; parity ^= 1; }
            }
            if (ok) commit(bar(f.tfull[acc]));
        }
        if (SPLIT) cluster_wait();
    } else if (warp >= 4) {
        const int id = threadIdx.x - 128, half = id >> 7, r = id & 127;      // r: weight row of the tile
        const uint32_t quadrant = static_cast<uint32_t>(warp & 3) * 32u << 16;
        asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
        if (SPLIT) cluster_wait();
        int i = 0;
        for (int t = cluster; t < tiles; t += clusters, ++i) {
            const int acc = i & 1;
            const Tile s = tile_at(t);
            const int col = s.rt * 128 + r;
            if (!wait_or_abort<false>(bar(f.tfull[acc]), (i / 2) & 1, abort_flag, a.err, DEV_TIMEOUT_MMA)) break;
            __syncwarp();
            fence_after();
            // Columns 32 half + 64 j .. + 31: all into registers first, so that the products after the next tile's do not wait for what follows.
            constexpr int J = NT < 64 ? 1 : NT / 64;
            float v[J][32];
#pragma unroll
            for (int j = 0; j < J; ++j)
                if (32 * half + 64 * j < s.n) ld32(tmem + quadrant + acc * 128 + 32 * half + 64 * j, v[j]);
            wait_ld();
            fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(f.tempty[acc]));
            if constexpr (!SPLIT) {
#pragma unroll
                for (int j = 0; j < J; ++j) {
                    const int c0 = 32 * half + 64 * j, here = min(32, s.n - c0);
                    if (here <= 0) break;
                    if (GROUPED) {
                        // lane: the row of y that column c0 + lane goes to, -1: to none
                        const int to = lane < here ? __ldg(a.out_row + s.row0 + c0 + lane) : 0;
#pragma unroll
                        for (int k = 0; k < 32; ++k) {
                            const int m = __shfl_sync(0xffffffffu, to, k);
                            store_if(k < here && m >= 0 && col < a.N, a.y + static_cast<size_t>(m) * a.N + col, v[j][k]);
                        }
                    } else if (col < a.N) {
                        float* q = a.y + static_cast<size_t>(s.row0 + c0) * a.N + col;
#pragma unroll
                        for (int k = 0; k < 32; ++k)
                            if (k < here) q[static_cast<size_t>(k) * a.N] = v[j][k];
                    }
                    __syncwarp();
                }
            } else {
                // Owner o has tokens o * run .. of the tile; its buffer is [CTA of the cluster][token / 4][row][4 tokens].
                const int run = ((s.n + C - 1) / C + 3) & ~3;
                const uint32_t part = static_cast<uint32_t>(run) * 512;
                const float per_run = 1.0f / static_cast<float>(run);
                if (i && !wait_pair(bar(f.avail), (i - 1) & 1, abort_flag, a.err, DEV_TIMEOUT_DRAIN)) break;
                __syncwarp();
#pragma unroll
                for (int j = 0; j < J; ++j)
#pragma unroll
                    for (int k = 0; k < 32; k += 4) {
                        const int c = 32 * half + 64 * j + k;
                        if (c >= s.n) break;
                        const int o = static_cast<int>((static_cast<float>(c) + 0.5f) * per_run);       // c / run: half a token from either border at least, c < 128
                        st_cluster4(map_to_rank(sb + off_recv + rank * part + ((c - o * run) * 128 + r * 4) * 4, o), v[j][k], v[j][k + 1], v[j][k + 2], v[j][k + 3]);
                    }
                __syncwarp();
                if (lane < C) arrive_release(map_to_rank(bar(f.recv), lane));
                if (!wait_pair(bar(f.recv), i & 1, abort_flag, a.err, DEV_TIMEOUT_DRAIN)) break;
                __syncwarp();
                const int m0 = rank * run, mine = min(run, s.n - m0);
                for (int g0 = half; 4 * g0 < mine; g0 += 8) {      // four groups of four tokens at a time
                    const float4* p = reinterpret_cast<const float4*>(smem + off_recv) + g0 * 128 + r;
                    float4 sum[4] = {};
#pragma unroll 1
                    for (int c = 0; c < C; ++c) {
#pragma unroll
                        for (int u = 0; u < 4; ++u) {
                            if (4 * (g0 + 2 * u) >= mine) break;
                            const float4 o = p[(c * (run / 4) + 2 * u) * 128];
                            sum[u].x += o.x; sum[u].y += o.y; sum[u].z += o.z; sum[u].w += o.w;
                        }
                    }
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        if (4 * (g0 + 2 * u) >= mine) break;
                        const float e[4] = {sum[u].x, sum[u].y, sum[u].z, sum[u].w};
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const int at = 4 * (g0 + 2 * u) + k, m = m0 + at;
                            const int to = !GROUPED || at >= mine ? s.row0 + m : __ldg(a.out_row + s.row0 + m);
                            store_if(at < mine && to >= 0 && col < a.N, a.y + static_cast<size_t>(to) * a.N + col, e[k]);
                        }
                    }
                }
                if (t + clusters < tiles) {             // there is a next tile: the buffer is free for every CTA
                    __syncwarp();
                    if (lane < C) arrive_release(map_to_rank(bar(f.avail), lane));
                }
            }
        }
    } else if (SPLIT) {
        cluster_wait();
    }
    __syncwarp();
    fence_before();
    __syncthreads();
    // What the others send here has been waited for, and who this CTA sends to waits for that: it may go. After a wait that gave up it does not until
    // every CTA of the cluster is here or gone.
    if (SPLIT && *abort_flag) { cluster_arrive(); cluster_wait(); }
    if (warp == 1) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" :: "r"(tmem), "r"(512u) : "memory");
    }
}

cudaLaunchConfig_t config(int C, cudaLaunchAttribute (&attr)[2], cudaStream_t st) {
    cudaLaunchConfig_t cfg{};
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = static_cast<unsigned>(C); attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.blockDim = dim3(THREADS); cfg.dynamicSmemBytes = SMEM; cfg.stream = st; cfg.attrs = attr; cfg.numAttrs = 2;
    return cfg;
}
// Clusters of C CTAs that run side by side on this GPU; 0: none. i: log2 C
template <int NT, bool GROUPED>
int clusters_of(int i) {
    static int n[4] = {-1, -1, -1, -1};
    if (n[i] < 0) {
        cudaLaunchAttribute attr[2];
        cudaLaunchConfig_t cfg = config(1 << i, attr, nullptr);
        cfg.gridDim = dim3(1 << i);
        cfg.numAttrs = 1;
        int got = 0;
        const bool ok = cudaFuncSetAttribute(mx_mid_kernel<NT, GROUPED, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM) == cudaSuccess &&
                        cudaFuncSetAttribute(mx_mid_kernel<NT, GROUPED, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM) == cudaSuccess &&
                        (i == 0 || cudaOccupancyMaxActiveClusters(&got, mx_mid_kernel<NT, GROUPED, true>, &cfg) == cudaSuccess);
        n[i] = !ok ? 0 : i == 0 ? ctx().sm_count : got;
        cudaGetLastError();
    }
    return n[i];
}

// k over C CTAs, so that the time is least: rounds of tiles, each the steps of a CTA and an exchange by the tokens that it moves and the CTAs that meet.
// Measured, us with C = 1 / 2 / 4 / 8: 24 x 4096 x 4096 12.2 / 10.0 / 8.1 / 12.0, 24 x 14336 x 4096 31.7 / 19.4 / 13.7 / 17.0, 24 x 4096 x 14336
// 13.0 / 14.3 / 17.4 / 27.3, 48 x 4096 x 1024 12.0 / 9.8 / 8.1 / 7.3, 77 x 2816 x 8448 10.6 / 11.1 / 13.3 / 23.7, 128 x 4096 x 4096 13.4 / 13.3 / 11.5 / 20.0.
// tiles: of a grouped call as many as there would be with an even-handed router. Returns ns; best: log2 C.
template <int NT, bool GROUPED>
long long share_k(long long tiles, int kts, int tokens, int& best) {
    long long least = 1ll << 62;
    for (int i = 0; i < 4; ++i) {
        const int c = 1 << i, n = clusters_of<NT, GROUPED>(i);
        if (!n || kts < c) continue;
        const long long ns = (tiles + n - 1) / n * ((kts + c - 1) / c * (230ll + tokens / 2) + (c > 1 ? 900 + 240 * (tokens / 9 + c / 2) : 0));
        if (ns < least) { least = ns; best = i; }
    }
    return least;
}
template <int NT, bool GROUPED>
int launch_nt(const CUtensorMap& map, const MxArgs& a, long long tiles, cudaStream_t st) {
    int best = 0;
    share_k<NT, GROUPED>(tiles, a.kts, GROUPED ? NT / 2 : a.tile_w < a.M ? a.tile_w : a.M, best);
    const int C = 1 << best;
    cudaLaunchAttribute attr[2];
    cudaLaunchConfig_t cfg = config(C, attr, st);
    cfg.gridDim = dim3(clusters_of<NT, GROUPED>(best) * C);
    ctx().launches++;
    ctx().last_mx = KERNEL_SINGLE + 16 * C;
    return cuda_check(C > 1 ? cudaLaunchKernelEx(&cfg, mx_mid_kernel<NT, GROUPED, true>, map, a, C, stages_of<NT>(C))
                            : cudaLaunchKernelEx(&cfg, mx_mid_kernel<NT, GROUPED, false>, map, a, C, stages_of<NT>(C)), "mx_mid launch");
}

}  // namespace

// Time of the tiles of one matrix, `tokens` (65 to 128) each, on this kernel.
long long mx_mid_ns(long long tiles, int kts, int tokens) {
    int best;
    return share_k<128, false>(tiles, kts, tokens, best);
}

int launch_mx_mid(const CUtensorMap& map, const MxArgs& a, int nt, long long tiles, bool grouped, cudaStream_t st) {
    if (grouped) return nt == 32 ? launch_nt<32, true>(map, a, tiles, st) : nt == 64 ? launch_nt<64, true>(map, a, tiles, st) : launch_nt<128, true>(map, a, tiles, st);
    return nt == 32 ? launch_nt<32, false>(map, a, tiles, st) : nt == 64 ? launch_nt<64, false>(map, a, tiles, st) : launch_nt<128, false>(map, a, tiles, st);
}

}  // namespace lp
