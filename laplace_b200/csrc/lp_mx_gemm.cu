// lp_mx_gemm.cu - products of packed MXFP4 weights and MXFP8 activations on the block-scaled tensor core instruction
// (tcgen05.mma kind::mxf8f6f4): D[128 weight rows][up to NT tokens] += A * B, 32 values a step, both scaled by a power of two per 32 values.
// Formats and layouts: lp_mx.cu. The instruction takes the 4-bit weights and their scale bytes as they lie in memory: no thread
// touches a weight. TMA spreads the 8 bytes of 16 values over 16 bytes of shared memory on the way in, the form that the instruction reads.
//
// Work. Tiles of 128 weight rows x NT tokens, k in steps of 128. Of T tiles and G CTAs (one per SM) the last T - T % G go to the CTAs
// one after the other, whole; the T % G before them are cut: their k steps, in tile order, in equal runs to the CTAs. A CTA that has a part
// of a tile leaves its sums in the workspace; the last of a tile's CTAs to arrive (a counter) adds them up in the order of k, so that the
// result does not depend on who was last. Few rows (decode) are all cut: every SM streams the same share of the weights.
//
// Roles by warp: 0 copies, 1 MMA issue (owns the TMEM), 4-11 drain (lane = weight row). All waits are bounded; a wait that gives up
// raises the status word and the roles leave their loops.
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

template <int NT> struct Lay {
    static constexpr int GROUPS = (NT + 127) / 128;       // 128-row groups of scales
    static constexpr int STAGE = A_STAGE + NT * 128 + SF_TILE + GROUPS * SF_TILE;
    static constexpr int STAGES = (226 * 1024 - 1024) / STAGE;
    static constexpr int ACCS = NT == 256 ? 1 : 2;
    static constexpr uint32_t A = 0, B = A + STAGES * A_STAGE, SFA = B + STAGES * NT * 128, SFB = SFA + STAGES * SF_TILE, BAR = SFB + STAGES * GROUPS * SF_TILE;
    static constexpr uint32_t FULL = BAR, EMPTY = FULL + 8 * STAGES, TFULL = EMPTY + 8 * STAGES, TEMPTY = TFULL + 16, PTR = TEMPTY + 16, ABORT = PTR + 4, LAST = ABORT + 4,
                              BYTES = LAST + 8 + 1024;
    static_assert(BYTES <= 227 * 1024, "shared memory");
    static_assert(ACCS * NT <= SF_COL, "TMEM columns");
};

struct Seg { int expert, rt, row0, n, group, k0, k1, cut; };      // group: first 128-row group of its scales; cut: number of the cut tile, -1 for a whole one
struct Work { int tiles, cut, ctas; long long units; };

__host__ __device__ __forceinline__ Work work_of(long long tiles, int kts, int grid) {
    Work w;
    w.tiles = static_cast<int>(tiles);
    w.cut = w.tiles % grid;
    w.units = static_cast<long long>(w.cut) * kts;
    const long long most = w.units / MIN_STEPS;
    w.ctas = most < 1 ? (w.units ? 1 : 0) : most < grid ? static_cast<int>(most) : grid;
    return w;
}
__device__ __forceinline__ long long cut_start(const Work& w, int c) { return w.units * c / w.ctas; }
// the CTA whose run holds unit u
__device__ __forceinline__ int cut_owner(const Work& w, long long u) {
    int c = static_cast<int>(u * w.ctas / w.units);
    while (c + 1 < w.ctas && cut_start(w, c + 1) <= u) ++c;
    while (c > 0 && cut_start(w, c) > u) --c;
    return c;
}

template <bool GROUPED>
__device__ __forceinline__ void tile_at(const MxArgs& a, int t, Seg& s) {
    if (GROUPED) {
        const int4 e = __ldg(a.tab + t / a.rts);
        s.rt = t % a.rts;
        s.expert = e.x; s.row0 = e.y; s.n = e.z; s.group = e.w;
    } else {
        s.rt = t / a.tiles_m;
        s.expert = 0;
        s.row0 = (t % a.tiles_m) * a.tile_w;
        s.group = (t % a.tiles_m) * a.tile_groups;
        s.n = min(a.tile_w, a.M - s.row0);
    }
}
// A CTA's work piece by piece, in the order in which every role walks it.
template <bool GROUPED>
struct Walk {
    const MxArgs& a;
    const Work w;
    long long u, u1;
    int next;
    __device__ __forceinline__ Walk(const MxArgs& args, const Work& work) : a(args), w(work) {
        const int c = blockIdx.x;
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
        next += gridDim.x;
        return true;
    }
};

template <int NT, bool GROUPED>
__global__ void __launch_bounds__(THREADS, 1) mx_gemm_kernel(const __grid_constant__ CUtensorMap map, const MxArgs a) {
    using L = Lay<NT>;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t sb = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* smem = smem_raw + (sb - smem_u32(smem_raw));
    volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::ABORT);
    const int warp = threadIdx.x >> 5;
    if (threadIdx.x == 0) {
        for (int i = 0; i < L::STAGES; ++i) { mbar_init(sb + L::FULL + 8 * i, 1); mbar_init(sb + L::EMPTY + 8 * i, 1); }
        for (int i = 0; i < 2; ++i) { mbar_init(sb + L::TFULL + 8 * i, 1); mbar_init(sb + L::TEMPTY + 8 * i, DRAIN / 32); }
        *abort_flag = 0;
        fence_barrier_init();
        asm volatile("prefetch.tensormap [%0];" :: "l"(&map) : "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" :: "r"(sb + L::PTR), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(smem + L::PTR);
    // Experts: the table of token tiles is made by the kernels before this one. One matrix: the weights may be copied meanwhile; the quantizer
    // before this kernel lets it start only after it has itself waited for what is before it in the stream, weights' writers included.
    if (GROUPED || warp != 0) asm volatile("griddepcontrol.wait;" ::: "memory");
    const Work w = work_of(GROUPED ? static_cast<long long>(*a.n_tiles) * a.rts : static_cast<long long>(a.tiles_m) * a.rts, a.kts, gridDim.x);

    if (warp == 0 && elect_one()) {
        auto tile_of = [&](const Seg& s, int kt) { return (static_cast<size_t>(s.expert) * a.rts + s.rt) * a.kts + kt; };
        auto weights = [&](int st, const Seg& s, int kt) {
            const int n8 = (s.n + 7) & ~7, groups = (s.n + 127) >> 7;
            const uint32_t bar = sb + L::FULL + 8 * st;
            mbar_expect_tx(bar, Q_TILE + SF_TILE + n8 * 128 + groups * SF_TILE);
            const size_t tile = tile_of(s, kt);
            tma_load_2d(sb + L::A + st * A_STAGE, &map, 0, static_cast<int>(tile * 128), bar);
            bulk_g2s(sb + L::SFA + st * SF_TILE, a.sfa + tile * SF_TILE, SF_TILE, bar);
        };
        auto tokens = [&](int st, const Seg& s, int kt) {
            const int n8 = (s.n + 7) & ~7, groups = (s.n + 127) >> 7;
            const uint32_t bar = sb + L::FULL + 8 * st;
            bulk_g2s(sb + L::B + st * NT * 128, a.img + (static_cast<size_t>(kt) * a.img_rows + s.row0) * 128, n8 * 128, bar);
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
    } else if (warp == 1 && elect_one()) {
        Walk<GROUPED> walk(a, w);
        Seg s;
        int it = 0;
        bool ok = true;
        for (int seg = 0; ok && walk(s); ++seg) {
            const int acc = seg % L::ACCS, n = (s.n + 15) & ~15, groups = (s.n + 127) >> 7;
            const uint32_t d = tmem + acc * NT;
            if (seg >= L::ACCS && !wait_or_abort<true>(sb + L::TEMPTY + 8 * acc, (seg / L::ACCS - 1) & 1, abort_flag, a.err, DEV_TIMEOUT_TMEM)) break;
            fence_after();
            for (int kt = s.k0; kt < s.k1; ++kt, ++it) {
                const int st = it % L::STAGES;
                if (!wait_or_abort<true>(sb + L::FULL + 8 * st, (it / L::STAGES) & 1, abort_flag, a.err, DEV_TIMEOUT_FULL)) { ok = false; break; }
                fence_after();
                const uint32_t sfa = tmem + SF_COL + 16 * (it & 1), sfb = sfa + 4;
                copy_scales(sfa, sb + L::SFA + st * SF_TILE);
                for (int g = 0; g < groups; ++g) copy_scales(sfb + 4 * g, sb + L::SFB + (st * L::GROUPS + g) * SF_TILE);
                const uint64_t ad = smem_desc_sw128(sb + L::A + st * A_STAGE), bd = smem_desc_sw128(sb + L::B + st * NT * 128);
#pragma unroll
                for (int ks = 0; ks < 4; ++ks) mma_mx(d, ad + 2 * ks, bd + 2 * ks, idesc_mx(n, ks), sfa, sfb, kt != s.k0 || ks);
                commit(sb + L::EMPTY + 8 * st);
            }
            if (ok) commit(sb + L::TFULL + 8 * acc);
        }
    } else if (warp >= 4) {
        Walk<GROUPED> walk(a, w);
        Seg s;
        const int lane = threadIdx.x & 31, id = threadIdx.x - 128, half = id >> 7, r = id & 127;      // r: weight row of the tile
        const uint32_t quadrant = static_cast<uint32_t>(warp & 3) * 32u << 16;
        volatile int* last = reinterpret_cast<volatile int*>(smem + L::LAST);
        for (int seg = 0; walk(s); ++seg) {
            const int acc = seg % L::ACCS;
            if (!wait_or_abort<false>(sb + L::TFULL + 8 * acc, (seg / L::ACCS) & 1, abort_flag, a.err, DEV_TIMEOUT_MMA)) break;
            __syncwarp();
            fence_after();
            const int col = s.rt * 128 + r;
            float* part = a.part + static_cast<size_t>(blockIdx.x + max(s.cut, 0)) * (NT * 128) + r;
            for (int c0 = 32 * half; c0 < s.n; c0 += 64) {
                float v[32];
                const int here = min(32, s.n - c0);
                int to = 0;                             // lane: the row of y that column c0 + lane goes to
                if (GROUPED && s.cut < 0 && lane < here) to = __ldg(a.out_row + s.row0 + c0 + lane);
                __syncwarp();
                ld32(tmem + quadrant + acc * NT + c0, v);
                wait_ld();
                if (s.cut >= 0) {
                    float* q = part + c0 * 128;
                    if (here == 32) {
#pragma unroll
                        for (int i = 0; i < 32; ++i) __stcg(q + i * 128, v[i]);
                    } else {
#pragma unroll
                        for (int i = 0; i < 32; ++i)
                            if (i < here) __stcg(q + i * 128, v[i]);
                    }
                } else if (GROUPED) {
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        const int m = __shfl_sync(0xffffffffu, to, i);
                        if (i < here && col < a.N) a.y[static_cast<size_t>(m) * a.N + col] = v[i];
                    }
                } else {
                    float* q = a.y + static_cast<size_t>(s.row0 + c0) * a.N + col;
                    if (here == 32 && col < a.N) {
#pragma unroll
                        for (int i = 0; i < 32; ++i) q[static_cast<size_t>(i) * a.N] = v[i];
                    } else if (col < a.N) {
#pragma unroll
                        for (int i = 0; i < 32; ++i)
                            if (i < here) q[static_cast<size_t>(i) * a.N] = v[i];
                    }
                }
            }
            fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(sb + L::TEMPTY + 8 * acc);
            if (s.cut < 0) continue;
            const long long u = static_cast<long long>(s.cut) * a.kts;
            const int first = cut_owner(w, u), pieces = cut_owner(w, u + a.kts - 1) - first + 1;
            __threadfence();
            named_bar_sync(1, DRAIN);
            if (id == 0) *last = atomicAdd(a.counters + s.cut, 1u) == static_cast<unsigned>(pieces - 1);
            named_bar_sync(1, DRAIN);
            if (!*last) continue;
            __threadfence();
            // four rows of a column a thread, eight columns at a time; parts in the order of k
            const int r4 = (id & 31) * 4, col4 = s.rt * 128 + r4;
            const float* p0 = a.part + static_cast<size_t>(first + s.cut) * (NT * 128) + r4;
            const bool vec = (a.N & 3) == 0 && (reinterpret_cast<uintptr_t>(a.y) & 15) == 0;
            for (int c0 = id >> 5; c0 < s.n; c0 += 32) {
                float4 sum[4] = {};
                for (int p = 0; p < pieces; p += 4) {
                    float4 v[4][4];
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            v[i][j] = p + i < pieces && c0 + 8 * j < s.n ? __ldcg(reinterpret_cast<const float4*>(p0 + static_cast<size_t>(p + i) * (NT * 128) + (c0 + 8 * j) * 128))
                                                                          : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int j = 0; j < 4; ++j) { sum[j].x += v[i][j].x; sum[j].y += v[i][j].y; sum[j].z += v[i][j].z; sum[j].w += v[i][j].w; }
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int m = c0 + 8 * j;
                    if (m >= s.n) break;
                    float* q = a.y + static_cast<size_t>(GROUPED ? __ldg(a.out_row + s.row0 + m) : s.row0 + m) * a.N + col4;
                    if (vec) {
                        if (col4 < a.N) *reinterpret_cast<float4*>(q) = sum[j];
                    } else {
                        const float e[4] = {sum[j].x, sum[j].y, sum[j].z, sum[j].w};
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (col4 + i < a.N) q[i] = e[i];
                    }
                }
            }
        }
    }
    __syncwarp();
    fence_before();
    __syncthreads();
    if (warp == 1) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" :: "r"(tmem), "r"(512u) : "memory");
    }
}

template <int NT, bool GROUPED>
int launch_nt(const CUtensorMap& map, const MxArgs& a, cudaStream_t st) {
    static bool configured = false;
    if (!configured) {
        const int rc = cuda_check(cudaFuncSetAttribute(mx_gemm_kernel<NT, GROUPED>, cudaFuncAttributeMaxDynamicSharedMemorySize, Lay<NT>::BYTES), "mx_gemm shared memory");
        if (rc) return rc;
        configured = true;
    }
    ctx().launches++;
    return launch_early(mx_gemm_kernel<NT, GROUPED>, dim3(ctx().sm_count), THREADS, Lay<NT>::BYTES, st, map, a);
}

}  // namespace

// Partial sums: the c-th CTA's part of the t-th cut tile is number c + t.
size_t mx_gemm_part_bytes(int nt, int cut_tiles) { return static_cast<size_t>(ctx().sm_count + cut_tiles) * nt * 128 * sizeof(float); }

int launch_mx_gemm(const MxArgs& a, int nt, long long tiles, bool grouped, cudaStream_t st) {
    CUtensorMap map;
    if (!mx_weights_map(&map, a.q, static_cast<size_t>(tiles))) return LAPLACE_ERR_CUDA;
    if (grouped) switch (nt) {
        case 32: return launch_nt<32, true>(map, a, st);
        case 64: return launch_nt<64, true>(map, a, st);
        case 128: return launch_nt<128, true>(map, a, st);
        default: return launch_nt<256, true>(map, a, st);
    }
    switch (nt) {
        case 32: return launch_nt<32, false>(map, a, st);
        case 64: return launch_nt<64, false>(map, a, st);
        case 128: return launch_nt<128, false>(map, a, st);
        default: return launch_nt<256, false>(map, a, st);
    }
}

}  // namespace lp
