// lp_mx_small.cu - products of packed MXFP4 weights with a handful of rows, in one launch: up to 8 activation rows of one matrix, or up to
// 32 (token, expert) pairs. Formats and layouts: lp_mx.cu, the instruction: lp_mx_mma.cuh.
//
// Bound by the weights' way from memory (0.53 bytes a value) and, where they are few, by latencies: a launch, the first copy, the last
// sums. So there is no quantizer launch - the rows are quantized by eight warps of every CTA, a 128-value step ahead of the tensor
// core, out of L2 (M x 512 bytes beside 8.7 KB of weights) - and no sum goes through memory: the CTAs of a cluster share out k, and each sends its
// part of a tile's results straight into the shared memory of the tile's owner, which adds them in the order of k and writes y.
//
// One row, in a graph over weights from cold memory: 4096 x 1024 3.4 us, 4096 x 4096 5.3, 4096 x 14336 9.8 us (31 MB, on 112 of 148 SMs; lp_gemv.cu streams 33 MB of Q4_K in
// 7.7, so it is the ring's bytes in flight that bound it), 28672 rows 12.5 us (5 TB/s); eight rows of 4096 x 14336 10.8. With quantizer launch and sums through global memory 8.2, 17.2 and, eight rows, 18.1. Two CTAs an SM, so that the next call's first copies and the
// last sums of this one overlap.
//
// A cluster of C CTAs takes tiles (128 weight rows x up to 8 tokens) number cluster, cluster + clusters, ...; the i-th of them is owned by CTA i % C.
// Roles by warp: 0 copies, 1 MMA issue (owns the TMEM), 2, 3, 8-13 quantizers (in pairs, four rows each), 4-7 drain (lane = weight row), sums and output. All waits are
// bounded; a wait that gives up raises the status word and the roles leave their loops.
#include "lp_mx.cuh"
#include "lp_mx_mma.cuh"
#include "lp_tc.cuh"

namespace lp {
namespace {

using namespace mx;
using namespace tc;

constexpr int THREADS = 448;
constexpr int QUANT = 4;                       // pairs of quantizer warps. At most the stages: a warp that waits for a stage must have seen the use before the last one end
constexpr int TOK = 8, MAX_PAIRS = 32;
constexpr int N_MMA = 16;                      // columns of the instruction; those from TOK on are not read
constexpr int ACCS = 8;                        // accumulators in TMEM
constexpr uint32_t SF_COL = ACCS * N_MMA, TMEM_COLS = 256;
constexpr int SLOTS = 2;                       // tiles that an owner may be receiving at once
constexpr int MAX_C = 8, MAX_STAGES = 12;
constexpr int A_STAGE = 128 * 128, B_STAGE = TOK * 128, STAGE = A_STAGE + B_STAGE + 2 * SF_TILE;

// Shared memory behind the ring (whose size goes by the number of stages) and the receiving slots: barriers, tables.
struct Fixed {
    uint64_t full[MAX_STAGES], empty[MAX_STAGES], tfull[ACCS], tempty[ACCS], recv[SLOTS], avail[MAX_C * SLOTS];
    uint32_t tmem;
    int      abort, n_tiles;
    int      expert[MAX_PAIRS], n[MAX_PAIRS];
    int      pair[MAX_PAIRS][TOK], row[MAX_PAIRS][TOK];
};

struct SmallArgs {
    const uint8_t* q;
    const uint8_t* sfa;
    const float*   x;
    float*         y;
    const int*     pair_expert;
    const int*     pair_row;
    int            M, N, K, kts, rts, experts, x_rows, stages, slot_tok;      // slot_tok: tokens that a receiving slot holds
    int*           err;
};

template <int C, bool GROUPED>
__global__ void __launch_bounds__(THREADS, 2) mx_small_kernel(const __grid_constant__ CUtensorMap map, const SmallArgs a) {
    extern __shared__ uint8_t smem_raw[];
    const uint32_t sb = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* smem = smem_raw + (sb - smem_u32(smem_raw));
    const int S = a.stages;
    const uint32_t off_b = S * A_STAGE, off_sfa = off_b + S * B_STAGE, off_sfb = off_sfa + S * SF_TILE, off_recv = off_sfb + S * SF_TILE,
                   slot_bytes = C * a.slot_tok * 512, off_fixed = off_recv + (C > 1 ? SLOTS * slot_bytes : 0);
    Fixed& f = *reinterpret_cast<Fixed*>(smem + off_fixed);
    volatile int* abort_flag = &f.abort;
    auto bar = [&](const uint64_t& b) { return smem_u32(&b); };
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = C > 1 ? static_cast<int>(pair_rank()) : 0;
    if (threadIdx.x == 0) {
        for (int i = 0; i < S; ++i) { mbar_init(bar(f.full[i]), 3); mbar_init(bar(f.empty[i]), 1); }
        for (int i = 0; i < ACCS; ++i) { mbar_init(bar(f.tfull[i]), 1); mbar_init(bar(f.tempty[i]), 4); }
        for (int i = 0; i < SLOTS; ++i) mbar_init(bar(f.recv[i]), 4 * C);
        for (int i = 0; i < C * SLOTS; ++i) mbar_init(bar(f.avail[i]), 4);
        f.abort = 0;
        fence_barrier_init();
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" :: "r"(smem_u32(&f.tmem)), "r"(TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (warp == 2) {
        if (lane == 0) asm volatile("prefetch.tensormap [%0];" :: "l"(&map) : "memory");
        if (GROUPED) {
            // Token tiles: the pairs of an expert in order, eight at a time; a tile's place is that of its first pair.
            asm volatile("griddepcontrol.wait;" ::: "memory");
            int e = -1, r = 0;
            if (lane < a.M) {
                e = __ldg(a.pair_expert + lane);
                r = a.pair_row ? __ldg(a.pair_row + lane) : lane;
                if (e >= 0 && (e >= a.experts || static_cast<unsigned>(r) >= static_cast<unsigned>(a.x_rows))) {
                    e = -1;
                    if (blockIdx.x == 0) atomicCAS(a.err, DEV_OK, DEV_BAD_INDEX);
                }
            }
            const unsigned same = __match_any_sync(0xffffffffu, e), before = (1u << lane) - 1;
            const int place = __popc(same & before), mine = place / TOK;
            const unsigned firsts = __ballot_sync(0xffffffffu, e >= 0 && place % TOK == 0);
            // the tile of a pair: the first whose expert and number among the expert's tiles are its own
            unsigned m = same & firsts;
            for (int i = 0; i < mine; ++i) m &= m - 1;
            if (e >= 0) {
                const int t = __popc(firsts & ((1u << (__ffs(m) - 1)) - 1));
                f.pair[t][place % TOK] = lane;
                f.row[t][place % TOK] = r;
                if (place % TOK == 0) { f.expert[t] = e; f.n[t] = min(TOK, __popc(same) - place); }
            }
            if (lane == 0) f.n_tiles = __popc(firsts);
        } else if (lane < TOK) {
            f.pair[0][lane] = lane; f.row[0][lane] = lane;
            if (lane == 0) { f.expert[0] = 0; f.n[0] = a.M; f.n_tiles = 1; }
        }
    }
    fence_before();
    __syncthreads();
    fence_after();
    if (C > 1) cluster_arrive();                   // barriers are there for the other CTAs; waited for where they are used first
    const uint32_t tmem = f.tmem;
    const int tiles = f.n_tiles * a.rts, clusters = gridDim.x / C, cluster = blockIdx.x / C;
    const int k0 = a.kts * rank / C, k1 = a.kts * (rank + 1) / C;      // every CTA has a step at least: kts >= C

    if (warp == 0 && elect_one()) {
        // One matrix: a ring of weights may be copied while the kernel before this one ends. Nothing is freed before it has (the quantizers wait for it), however
        // long that takes, so the bounded waits begin after it.
        int st = 0, parity = 1, early = GROUPED ? 0 : S;
        bool ok = true;
        for (int t = cluster; ok && t < tiles; t += clusters) {
            const size_t tile0 = (static_cast<size_t>(f.expert[t / a.rts]) * a.rts + t % a.rts) * a.kts;
            for (int kt = k0; kt < k1; ++kt) {
                if (!GROUPED && early-- == 0) asm volatile("griddepcontrol.wait;" ::: "memory");
                if (!wait_or_abort<false>(bar(f.empty[st]), parity, abort_flag, a.err, DEV_TIMEOUT_EMPTY)) { ok = false; break; }
                const uint32_t b = bar(f.full[st]);
                mbar_expect_tx(b, Q_TILE + SF_TILE);
                tma_load_2d(sb + st * A_STAGE, &map, 0, static_cast<int>((tile0 + kt) * 128), b);
                bulk_g2s(sb + off_sfa + st * SF_TILE, a.sfa + (tile0 + kt) * SF_TILE, SF_TILE, b);
                if (++st == S) { st = 0; parity ^= 1; }
            }
        }
        if (!ok)                                    // what is in flight lands before the CTA goes
            for (int i = 0; i < 1000; ++i) __nanosleep(1000);
        if (C > 1) cluster_wait();
    } else if (warp == 1 && elect_one()) {
        int st = 0, parity = 0, i = 0, set = 0;      // set: of TMEM columns for the scales
        bool ok = true;
        if (!GROUPED) asm volatile("griddepcontrol.wait;" ::: "memory");
        for (int t = cluster; ok && t < tiles; t += clusters, ++i) {
            const int acc = i % ACCS;
            if (i >= ACCS && !wait_or_abort<true>(bar(f.tempty[acc]), (i / ACCS - 1) & 1, abort_flag, a.err, DEV_TIMEOUT_TMEM)) break;
            fence_after();
            for (int kt = k0; kt < k1; ++kt) {
                if (!wait_or_abort<true>(bar(f.full[st]), parity, abort_flag, a.err, DEV_TIMEOUT_FULL)) { ok = false; break; }
                fence_after();
                const uint32_t sfa = tmem + SF_COL + 8 * set, sfb = sfa + 4;
                set ^= 1;
                copy_scales<1>(sfa, sb + off_sfa + st * SF_TILE);
                copy_scales<1>(sfb, sb + off_sfb + st * SF_TILE);
                const uint64_t ad = smem_desc_sw128(sb + st * A_STAGE), bd = smem_desc_sw128(sb + off_b + st * B_STAGE);
#pragma unroll
                for (int ks = 0; ks < 4; ++ks) mma_mx<1>(tmem + acc * N_MMA, ad + 2 * ks, bd + 2 * ks, idesc_mx<1>(N_MMA, ks), sfa, sfb, kt != k0 || ks);
                commit(bar(f.empty[st]));
                if (++st == S) { st = 0; parity ^= 1; }
            }
            if (ok) commit(bar(f.tfull[acc]));
        }
        if (C > 1) cluster_wait();
    } else if (warp == 2 || warp == 3 || warp >= 8) {
        // 16 lanes a row: a step is 128 values of two rows, 8 values a lane, a 32-value block per four lanes; the second warp of a pair has rows 4 to 7
        const int w = warp < 4 ? warp - 2 : warp - 6, which = w >> 1, m0 = (w & 1) * (TOK / 2) + (lane >> 4), k8 = (lane & 15) * 8;
        asm volatile("griddepcontrol.wait;" ::: "memory");
        int st = 0, parity = 1, turn = 0;
        bool ok = true;
        for (int t = cluster; ok && t < tiles; t += clusters) {
            const int tt = t / a.rts, n = f.n[tt];
            for (int kt = k0; kt < k1; ++kt) {
                if (turn == which) {
                    const int k = kt * 128 + k8;
                    float v[TOK / 4][8];
#pragma unroll
                    for (int j = 0; j < TOK / 4; ++j) {            // loads of all rows before the wait and the first use
                        const int m = m0 + 2 * j;
                        if (m < n && k < a.K) load8(a.x + static_cast<size_t>(f.row[tt][m]) * a.K + k, v[j]);
                        else
#pragma unroll
                            for (int i = 0; i < 8; ++i) v[j][i] = 0.f;
                    }
                    if (!wait_or_abort<false>(bar(f.empty[st]), parity, abort_flag, a.err, DEV_TIMEOUT_EMPTY)) { ok = false; break; }
                    uint8_t* img = smem + off_b + st * B_STAGE;
                    uint8_t* sf = smem + off_sfb + st * SF_TILE;
#pragma unroll
                    for (int j = 0; j < TOK / 4; ++j) {
                        const int m = m0 + 2 * j;
                        if (m - (lane >> 4) >= n) break;
                        uint32_t sc;
                        const uint2 q = mxfp8_block8(v[j], lane, sc);
                        if (m < n) {
                            *reinterpret_cast<uint2*>(img + m * 128 + ((((lane & 15) >> 1) ^ m) << 4) + (lane & 1) * 8) = q;
                            if ((lane & 15) == 0) *reinterpret_cast<uint32_t*>(sf + m * 16) = sc;
                        }
                    }
                    fence_proxy_async();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(bar(f.full[st]));
                }
                if (++turn == QUANT) turn = 0;
                if (++st == S) { st = 0; parity ^= 1; }
            }
        }
        if (C > 1) cluster_wait();
    } else if (warp >= 4 && warp < 8) {
        const int r = threadIdx.x - 128;                // weight row of the tile
        const uint32_t quadrant = static_cast<uint32_t>(warp & 3) * 32u << 16;
        asm volatile("griddepcontrol.wait;" ::: "memory");
        asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
        if (C > 1) cluster_wait();
        int i = 0;
        for (int t = cluster; t < tiles; t += clusters, ++i) {
            const int acc = i % ACCS, tt = t / a.rts, n = f.n[tt], col = (t % a.rts) * 128 + r;
            if (!wait_or_abort<true>(bar(f.tfull[acc]), (i / ACCS) & 1, abort_flag, a.err, DEV_TIMEOUT_MMA)) break;
            __syncwarp();
            fence_after();
            float v[TOK];
            ld8(tmem + quadrant + acc * N_MMA, v);
            wait_ld();
            fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(f.tempty[acc]));
            if (C == 1) {
#pragma unroll
                for (int m = 0; m < TOK; ++m)
                    if (m < n && col < a.N) a.y[static_cast<size_t>(f.pair[tt][m]) * a.N + col] = v[m];
                continue;
            }
            const int owner = i % C, slot = i / C % SLOTS, use = i / C / SLOTS;
            const uint32_t at = sb + off_recv + slot * slot_bytes;
            if (use && !wait_pair(bar(f.avail[owner * SLOTS + slot]), (use - 1) & 1, abort_flag, a.err, DEV_TIMEOUT_DRAIN)) break;
            const uint32_t there = map_to_rank(at + static_cast<uint32_t>(rank * a.slot_tok) * 512 + r * 4, owner);
#pragma unroll
            for (int m = 0; m < TOK; ++m)
                if (m < n) st_cluster(there + m * 512, v[m]);
            __syncwarp();
            if (lane == 0) arrive_release(map_to_rank(bar(f.recv[slot]), owner));
            if (owner != rank) continue;
            if (!wait_pair(bar(f.recv[slot]), use & 1, abort_flag, a.err, DEV_TIMEOUT_DRAIN)) break;
            __syncwarp();
            const float* p = reinterpret_cast<const float*>(smem + off_recv + slot * slot_bytes) + r;
#pragma unroll
            for (int m = 0; m < TOK; ++m) {
                if (m >= n) break;
                float sum = 0.f;
#pragma unroll
                for (int c = 0; c < C; ++c) sum += p[(c * a.slot_tok + m) * 128];
                if (col < a.N) a.y[static_cast<size_t>(f.pair[tt][m]) * a.N + col] = sum;
            }
            if (t + C * SLOTS * clusters < tiles) {     // the slot has a next tile: free for every CTA
                __syncwarp();
                if (lane < C) arrive_release(map_to_rank(bar(f.avail[rank * SLOTS + slot]), lane));
            }
        }
    } else if (C > 1) {
        cluster_wait();
    }
    __syncwarp();
    fence_before();
    __syncthreads();
    // What the others send here has been waited for, and who this CTA sends to waits for that: it may go. After a wait that gave up it does not until
    // every CTA of the cluster is here or gone.
    if (C > 1 && *abort_flag) { cluster_arrive(); cluster_wait(); }
    if (warp == 1) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" :: "r"(tmem), "r"(TMEM_COLS) : "memory");
    }
}

constexpr size_t SMEM = 113 * 1024;
int slot_tokens(int M) { return M < TOK ? M : TOK; }
int stages_of(int C, int M) {
    const size_t left = SMEM - 1024 - sizeof(Fixed) - (C > 1 ? static_cast<size_t>(SLOTS) * C * slot_tokens(M) * 512 : 0);
    const int s = static_cast<int>(left / STAGE);
    return s < MAX_STAGES ? s : MAX_STAGES;
}

// Clusters of C CTAs that run side by side on this GPU; 0: none.
template <int C, bool GROUPED>
int clusters_at_once(cudaLaunchConfig_t cfg) {
    static int n = -1;
    if (n < 0) {
        cfg.gridDim = dim3(C);
        int got = 0;
        n = cudaFuncSetAttribute(mx_small_kernel<C, GROUPED>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM) == cudaSuccess &&
                    (C == 1 || cudaOccupancyMaxActiveClusters(&got, mx_small_kernel<C, GROUPED>, &cfg) == cudaSuccess)
                ? (C == 1 ? 2 * ctx().sm_count : got) : 0;
        cudaGetLastError();
    }
    return n;
}
template <int C, bool GROUPED>
int clusters_of() {
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim = {C, 1, 1};
    cfg.blockDim = dim3(THREADS); cfg.dynamicSmemBytes = SMEM; cfg.attrs = attr; cfg.numAttrs = C > 1 ? 1 : 0;
    return clusters_at_once<C, GROUPED>(cfg);
}

template <int C, bool GROUPED>
int launch_c(const CUtensorMap& map, SmallArgs a, int tiles, cudaStream_t st) {
    const int most = clusters_of<C, GROUPED>();
    a.stages = stages_of(C, a.M);
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim = {C, 1, 1};
    cfg.gridDim = dim3((tiles < most ? tiles : most) * C); cfg.blockDim = dim3(THREADS); cfg.dynamicSmemBytes = SMEM; cfg.stream = st; cfg.attrs = attr; cfg.numAttrs = C > 1 ? 2 : 1;
    ctx().launches++;
    ctx().last_mx = KERNEL_SMALL + 16 * C;
    return cuda_check(cudaLaunchKernelEx(&cfg, mx_small_kernel<C, GROUPED>, map, a), "mx_small launch");
}

template <bool GROUPED>
int launch_small(const CUtensorMap& map, const SmallArgs& a, int tiles, cudaStream_t st) {
    // k over C CTAs, so that the time is least: rounds of tiles, each the steps of a CTA (200 ns, or more where so many CTAs are at work that memory is
    // what they wait for: 470 with all of them) and an exchange. Measured, one row, us with C = 1 / 2 / 4 / 8 (with a barrier at the end, 0.3 us): 4096 x 1024 8.6 / 5.5 / 4.1 / 3.6, 4096 x 4096
    // 8.8 / 6.1 / 5.9 / 7.5, 4096 x 14336 9.8 / 10.6 / 11.1 / 14.4, 14336 x 4096 25.5 / 14.7 / 9.8 / 12.6, eight experts 2048 x 1536 6.7 / 7.7 / 7.9 / 6.6.
    const int n[4] = {clusters_of<1, GROUPED>(), clusters_of<2, GROUPED>(), clusters_of<4, GROUPED>(), clusters_of<8, GROUPED>()};
    int best = 0;
    long long least = 1ll << 62;
    for (int i = 0; i < 4; ++i) {
        const int c = 1 << i;
        if (!n[i] || a.kts < c || stages_of(c, a.M) < QUANT) continue;
        const long long active = static_cast<long long>(tiles < n[i] ? tiles : n[i]) * c, step = active * 470 / (2 * ctx().sm_count);
        const long long ns = (tiles + n[i] - 1) / n[i] * ((a.kts + c - 1) / c * (step > 200 ? step : 200) + (c > 1 ? 900 + 100 * c : 0));
        if (ns < least) { least = ns; best = i; }
    }
    switch (best) {
        case 0: return launch_c<1, GROUPED>(map, a, tiles, st);
        case 1: return launch_c<2, GROUPED>(map, a, tiles, st);
        case 2: return launch_c<4, GROUPED>(map, a, tiles, st);
        default: return launch_c<8, GROUPED>(map, a, tiles, st);
    }
}

}  // namespace

// Whether a call goes here: rows of one matrix, or pairs, and few enough.
bool mx_small_takes(int rows, bool grouped) { return rows <= (grouped ? MAX_PAIRS : TOK); }

int launch_mx_small(const float* x, int x_rows, const uint8_t* packed, const int* pair_expert, const int* pair_row, int rows, int experts, float* y, int K, int N, cudaStream_t st) {
    SmallArgs a{};
    a.kts = (K + 127) / 128; a.rts = (N + 127) / 128;
    const size_t tiles = static_cast<size_t>(experts) * a.rts * a.kts;
    a.q = packed; a.sfa = packed + tiles * Q_TILE; a.x = x; a.y = y; a.pair_expert = pair_expert; a.pair_row = pair_row;
    a.M = rows; a.N = N; a.K = K; a.experts = experts; a.x_rows = x_rows; a.slot_tok = slot_tokens(rows); a.err = ctx().d_err;
    CUtensorMap map;
    if (!mx_weights_map(&map, packed, tiles)) return LAPLACE_ERR_CUDA;
    const int most = pair_expert ? (rows < experts ? rows : experts) : 1;       // token tiles, were no expert chosen by more than eight
    return pair_expert ? launch_small<true>(map, a, most * a.rts, st) : launch_small<false>(map, a, a.rts, st);
}

}  // namespace lp
