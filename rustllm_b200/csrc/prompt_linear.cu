// Projections of prompts (tmllm_prompt_linear): out = residual + act(x W + bias) for any number
// of rows, the matrix product on the 5th-generation tensor cores and everything behind it in
// its epilogue, so the product never makes a round trip through memory.
//
// A persistent grid walks the output tiles: one warp feeds x and W tiles through a ring by TMA,
// one issues the products into one of two accumulators in tensor memory, eight empty the other
// one, so the epilogue runs under the next tile's products.  Bound by the tensor pipe (92 % active
// at 8191 x 4096 x 4096 with bias and residual, 178 us = 1.54 PFLOP/s at first, 232 us back to back
// under the power limit, where a library product alone takes 237) and by latency for few rows
// (33 x 768 x 2048: 6.4 us in a graph, 9.4 with bias, 10 us a call), where K is split over the CTAs
// of a cluster if it is long (33 x 4096 x 64: 6.0 us instead of 17.2, library product 6.7; 33 x 4096
// x 4096: 10.7 instead of 17.7, library 8.5).
//
// F16 x [rows, k], W [k, n] row-major (nn/linear.rs:26-27), F32 accumulation and F32 all the
// way through bias, activation (kernels/silu.metal:38-46 for SwiGLU) and residual, one
// rounding to F16 at the store.
#include <atomic>
#include <type_traits>

#include "common.cuh"
#include "tc.cuh"

namespace tmllm {
namespace {

constexpr int kM = 128;        // rows of an output tile (the tensor-memory lanes)
constexpr int kK = 64;         // K columns per stage: one 128-byte swizzle row
constexpr int kEpiWarps = 8;
constexpr int kThreads = 64 + 32 * kEpiWarps;  // warp 0: TMA, warp 1: MMA, the rest: epilogue

__device__ int g_linear_status;

enum Act : int { ACT_NONE = 0, ACT_RELU = 1, ACT_SILU = 2, ACT_GELU = 3, ACT_SWIGLU = 4 };

struct LinArgs {
    const __half* bias;
    const __half* residual;
    __half* out;
    int64_t ld_res, ld_out;
    int32_t rows, k, n, act;
    int32_t m_tiles, n_tiles, tiles, group_m;
};

__device__ __forceinline__ float silu(float x) { return __fdividef(x, 1.f + __expf(-x)); }
// x Phi(x).  Phi(-|x|) = exp(-x^2 / 2) g(|x|): g falls slowly and is fitted by a polynomial in
// t = 1 / (1 + 0.42 |x| / sqrt 2) (the form Hastings gave for erfc; the coefficients are a
// least-squares fit reweighted to an even relative error, 1.1e-6 up to |x| = 6.2), so the left
// tail keeps its relative accuracy.  Two MUFU operations and about 14 others, a third of what
// erfcf takes.
__device__ __forceinline__ float gelu(float x) {
    constexpr float GC0 = 0.11946170f, GC1 = 0.10668742f, GC2 = 0.16564545f, GC3 = -0.05811026f,
                    GC4 = 0.25197804f, GC5 = -0.08566288f;
    const float t = __fdividef(1.f, fmaf(0.29698485f, fabsf(x), 1.f));
    float g = fmaf(t, GC5, GC4);
    g = fmaf(t, g, GC3);
    g = fmaf(t, g, GC2);
    g = fmaf(t, g, GC1);
    g = fmaf(t, g, GC0) * t;
    const float tail = __expf(-0.5f * x * x) * g;
    return x * (x < 0.f ? tail : 1.f - tail);
}
__device__ __forceinline__ float relu(float x) { return x > 0.f ? x : (x <= 0.f ? 0.f : x); }  // NaN stays

// BN: accumulator columns of a tile; with GATED half of them are gate and half up columns.
// PAIR: the two CTAs of a cluster share a tile of 256 rows, each with its 128 rows of A and half
// the columns of W in shared memory.
// SPLIT > 1: the SPLIT CTAs of a cluster take a part of K of one tile each; every CTA then gets
// the others' sums of its share of the columns and stores those.
template <int BN, bool GATED, bool PAIR = false, int SPLIT = 1>
struct LinCfg {
    static constexpr int ON = GATED ? BN / 2 : BN;  // output columns of a tile
    static constexpr int A_BYTES = kM * kK * 2;
    static constexpr int BC = PAIR ? BN / 2 : BN;  // columns of W in this CTA
    static constexpr int B_BYTES = BC * kK * 2;
    static constexpr int STAGE = A_BYTES + B_BYTES;
    // output staging: every epilogue warp has two buffers of 32 rows x 32 columns; with a split K
    // the sums of this CTA's share of the columns from every other CTA instead
    static constexpr int OUT_BYTES =
        SPLIT > 1 ? kM * (BN / SPLIT) * 4 * (SPLIT - 1) : kEpiWarps * 2 * 2048;
    static constexpr int RING = 229376 - OUT_BYTES;
    static constexpr int STAGES = RING / STAGE < 8 ? RING / STAGE : 8;
    static constexpr int OFF_OUT = STAGES * STAGE;
    static constexpr int OFF_BIAS = OFF_OUT + OUT_BYTES;
    // bias as F16: 32 columns (and the 32 up columns of a gated tile) of each epilogue warp
    static constexpr int OFF_BAR = OFF_BIAS + kEpiWarps * 64 * 2;
    static constexpr int SMEM = OFF_BAR + 512 + 1024;  // + alignment
    static constexpr int ACC = BN <= 64 ? 64 : BN <= 128 ? 128 : 256;  // columns apart
    static constexpr int TMEM_COLS = 2 * ACC;                          // two accumulators
    static_assert(SMEM <= 227 * 1024, "shared memory of one CTA");
    static constexpr int SHARE = ON / SPLIT;  // output columns of a CTA
    static_assert(SHARE % 8 == 0, "16 bytes of a row");
    // 8 accumulator columns 8 i .. among those of the CTA that stores them
    static __device__ __forceinline__ int chunk(int i) {
        const int up = GATED && i * 8 >= ON;
        return up * (SHARE / 8) + (i - up * (ON / 8)) % (SHARE / 8);
    }
};

// Tile `t`: groups of group_m row tiles sweep the columns together, so a wave's A and W tiles
// stay in L2.
__device__ __forceinline__ void tile_of(const LinArgs& a, int t, int& m, int& n) {
    const int per = a.group_m * a.n_tiles;
    const int g = t / per, first = g * a.group_m;
    const int gm = a.m_tiles - first < a.group_m ? a.m_tiles - first : a.group_m;
    const int r = t - g * per;
    m = first + r % gm;
    n = r / gm;
}

template <int BN, bool GATED, bool PAIR, int SPLIT>
__global__ void __launch_bounds__(kThreads, 1)
    prompt_linear_kernel(const __grid_constant__ CUtensorMap xmap,
                         const __grid_constant__ CUtensorMap wmap,
                         const __grid_constant__ CUtensorMap omap,
                         const __grid_constant__ CUtensorMap rmap, const LinArgs a) {
    using Cfg = LinCfg<BN, GATED, PAIR, SPLIT>;
    static_assert(!PAIR || SPLIT == 1, "one use of the cluster");
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    const uint32_t sbase = smem_u32(smem);
    const int tid = threadIdx.x, lane = tid & 31;
    const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);  // uniform for the compiler too
    const uint32_t bars = sbase + Cfg::OFF_BAR;
    auto full = [&](int i) { return bars + 8u * i; };
    auto empty = [&](int i) { return bars + 8u * (Cfg::STAGES + i); };
    auto acc_full = [&](int i) { return bars + 8u * (2 * Cfg::STAGES + i); };
    auto acc_empty = [&](int i) { return bars + 8u * (2 * Cfg::STAGES + 2 + i); };
    const uint32_t done = bars + 8u * (2 * Cfg::STAGES + 4);
    auto res_full = [&](int w, int b) { return bars + 8u * (2 * Cfg::STAGES + 5 + 2 * w + b); };
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(
        smem + Cfg::OFF_BAR + 8 * (2 * Cfg::STAGES + 5 + 2 * kEpiWarps));
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

    if (tid == 0) {
        for (int i = 0; i < Cfg::STAGES; ++i) {
            mbar_init(full(i), 1);
            mbar_init(empty(i), 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(acc_full(i), 1);
            mbar_init(acc_empty(i), kEpiWarps * (PAIR ? 2 : 1));
        }
        mbar_init(done, 1);
        for (int i = 0; i < 2 * kEpiWarps; ++i) mbar_init(res_full(i >> 1, i & 1), 1);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        if (PAIR) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                             smem_u32(tmem_slot)),
                         "r"(Cfg::TMEM_COLS)
                         : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        } else {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                             smem_u32(tmem_slot)),
                         "r"(Cfg::TMEM_COLS)
                         : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        }
    }
    tc_fence_before();
    if (PAIR || SPLIT > 1) cluster_sync_all();  // the other CTAs' barriers are ready too
    else __syncthreads();
    tc_fence_after();
    // the pair walks the tiles together; this CTA has the rows from `row_of` on
    const int rank = PAIR ? static_cast<int>(cluster_rank()) : 0;
    const int share = SPLIT > 1 ? static_cast<int>(cluster_rank()) : 0;  // of K and the columns
    const int tile_first = blockIdx.x / (PAIR ? 2 : SPLIT);
    const int tile_step = gridDim.x / (PAIR ? 2 : SPLIT);
    auto row_of = [&](int m) { return PAIR ? (2 * m + rank) * kM : m * kM; };
    const uint32_t tmem = *tmem_slot;
    const int k_steps = (a.k + kK - 1) / kK;  // this CTA's are [k_lo, k_lo + nk)
    const int k_lo = static_cast<int>(static_cast<int64_t>(k_steps) * share / SPLIT);
    const int nk = static_cast<int>(static_cast<int64_t>(k_steps) * (share + 1) / SPLIT) - k_lo;

    if (warp == 0) {
        if (lane == 0) {
            int g = 0;
            bool ok = true;
            for (int t = tile_first; ok && t < a.tiles; t += tile_step) {
                int m, n;
                tile_of(a, t, m, n);
                for (int kb = 0; kb < nk; ++kb, ++g) {
                    const int st = g % Cfg::STAGES, use = g / Cfg::STAGES;
                    if (use > 0) {
                        ok = mbar_wait_bounded(empty(st), (use - 1) & 1, abort_flag, &g_linear_status);
                        if (!ok) break;
                    }
                    const uint32_t sa = sbase + st * Cfg::STAGE, sb = sa + Cfg::A_BYTES;
                    // both CTAs' copies count on the first one's barrier, where the products wait
                    if (!PAIR || rank == 0) mbar_arrive_tx(full(st), Cfg::STAGE * (PAIR ? 2 : 1));
                    const uint32_t fb = PAIR ? cluster_addr(full(st), 0) : full(st);
                    auto load = [&](uint32_t dst, const CUtensorMap* map, int x, int y) {
                        if (PAIR) tma_load_2d_pair(dst, map, x, y, fb);
                        else tma_load_2d(dst, map, x, y, fb);
                    };
                    load(sa, &xmap, (k_lo + kb) * kK, row_of(m));
#pragma unroll
                    for (int c = 0; c < Cfg::BC / 64; ++c) {
                        const int tc = rank * Cfg::BC + c * 64;  // accumulator column
                        const int col = GATED ? (tc < Cfg::ON ? n * Cfg::ON + tc
                                                              : a.n + n * Cfg::ON + tc - Cfg::ON)
                                              : n * BN + tc;
                        load(sb + c * (64 * kK * 2), &wmap, col, (k_lo + kb) * kK);
                    }
                }
            }
            // every copy has landed before the CTA gives its memory back, also when this warp
            // got through and another one gave up
            for (int i = g < Cfg::STAGES ? 0 : g - Cfg::STAGES; rank == 0 && i < g; ++i)
                mbar_drain(full(i % Cfg::STAGES), (i / Cfg::STAGES) & 1);
        }
    } else if (warp == 1 && rank == 0) {
        // The whole warp walks this code and one elected lane issues, so that the descriptors
        // stay in uniform registers.
        constexpr uint32_t IDESC = f16_idesc(PAIR ? 2 * kM : kM, BN, true);
        auto commit = [](uint32_t bar) {
            if (PAIR) tc_commit_pair(bar);
            else tc_commit(bar);
        };
        const bool leader = elect_one();
        const uint32_t abort_addr = smem_u32(const_cast<int*>(abort_flag));
        int st = 0, phase = 0, it = 0;
        for (int t = tile_first; t < a.tiles && !*abort_flag; t += tile_step, ++it) {
            const int ab = it & 1;
            if (it >= 2) {
                mbar_wait_uniform(acc_empty(ab), ((it >> 1) - 1) & 1, abort_addr, &g_linear_status);
                tc_fence_after();
            }
            const uint32_t d = tmem + ab * Cfg::ACC;
            for (int kb = 0; kb < nk; ++kb) {
                mbar_wait_uniform(full(st), phase, abort_addr, &g_linear_status);
                tc_fence_after();
                const uint32_t sa = sbase + st * Cfg::STAGE;
                const uint64_t ad = sw128_desc(sa, 16, 1024);
                const uint64_t bd = sw128_desc(sa + Cfg::A_BYTES, 64 * kK * 2, 1024);
                if (leader) {
#pragma unroll
                    for (int kk = 0; kk < kK / 16; ++kk) {
                        const uint64_t ak = ad + kk * (32 >> 4), bk = bd + kk * (2048 >> 4);
                        if (PAIR) tc_mma_pair(d, ak, bk, IDESC, kb > 0 || kk > 0);
                        else tc_mma(d, ak, bk, IDESC, kb > 0 || kk > 0);
                    }
                    commit(empty(st));
                }
                __syncwarp();
                if (++st == Cfg::STAGES) st = 0, phase ^= 1;
            }
            if (leader) commit(acc_full(ab));
            __syncwarp();
        }
        if (leader) {  // every product has completed before the CTA frees its memory
            commit(done);
            mbar_drain(done, 0);
        }
        __syncwarp();
    } else if (SPLIT > 1 && warp > 1) {
        // ---- the sums of the others' columns go to them, 8 columns and 32 rows at a time:
        // [CTA][8 columns][4 of them][row] of 16 bytes
        const int row = (warp & 3) * 32 + lane;
        const uint32_t acc = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
        mbar_wait_uniform(acc_full(0), 0, smem_u32(const_cast<int*>(abort_flag)), &g_linear_status);
        tc_fence_after();
#pragma unroll 1
        for (int i = (warp - 2) >> 2; i < BN / 8; i += 2) {  // 8 columns of the tile
            const int o = i * 8 % Cfg::ON, to = o / Cfg::SHARE;  // output column, its CTA
            if (to == share) continue;
            float y[8];
            tmem_ld8(acc + i * 8, y);
            const int from = share < to ? share : share - 1;  // among the CTAs that send there
            const uint32_t slot = static_cast<uint32_t>(
                Cfg::OFF_OUT + ((from * (BN / 8 / SPLIT) + Cfg::chunk(i)) * 2 * kM + row) * 16);
            const uint32_t dst = cluster_addr(sbase + slot, to);
            st_cluster(dst, y[0], y[1], y[2], y[3]);
            st_cluster(dst + kM * 16, y[4], y[5], y[6], y[7]);
        }
    } else if (warp > 1) {
        // ---- epilogue: a warp owns 32 rows and every other 32 columns of the tile.  It works
        // alone: its rows leave through its own two buffers and bulk stores; the residual
        // arrives the same way in the buffer it leaves by, 32 columns ahead, and the bias by a
        // load a lane, 32 columns ahead too.  No barrier joins the warps: one that gave up a wait
        // leaves by itself, and a barrier has no limit.
        const int quarter = warp & 3, part = (warp - 2) >> 2;
        __half* bias = reinterpret_cast<__half*>(smem + Cfg::OFF_BIAS) + (warp - 2) * 64;
        unsigned char* stage = smem + Cfg::OFF_OUT + (warp - 2) * 4096;
        const uint32_t stage_addr = smem_u32(stage);
        const uint32_t lane_base = static_cast<uint32_t>(quarter * 32) << 16;
        const uint32_t abort_addr = smem_u32(const_cast<int*>(abort_flag));
        int it = 0, ob = 0;
        uint32_t phases[2] = {0u, 0u};
        uint32_t sent = 0;  // bit b: an odd number of residual loads went to buffer b
        for (int t = tile_first; t < a.tiles && !*abort_flag; t += tile_step, ++it) {
            int m, n;
            tile_of(a, t, m, n);
            const int ab = it & 1;
            __half bias_next[2] = {__half(0.f), __half(0.f)};  // this lane's of the next columns
            auto load_bias = [&](int c0) {
                const int col = n * Cfg::ON + c0 + lane;
                if (!a.bias || c0 >= Cfg::ON || col >= a.n) return;
                bias_next[0] = a.bias[col];
                if (GATED) bias_next[1] = a.bias[a.n + col];
            };
            // columns c0 .. of the tile into buffer b, once its last store has been read
            auto load_res = [&](int c0, int b) {
                const int col = n * Cfg::ON + c0;
                if (!a.residual || c0 >= Cfg::ON || col >= a.n || lane != 0) return;
                if (*abort_flag) return;  // the buffer's last load may still be in flight
                bulk_wait_read<0>();
                mbar_arrive_tx(res_full(warp - 2, b), 2048);
                sent ^= 1u << b;
                tma_load_2d(stage_addr + b * 2048, &rmap, col, row_of(m) + quarter * 32,
                            res_full(warp - 2, b));
            };
            load_res(part * 32, ob);
            load_bias(part * 32);
            mbar_wait_uniform(acc_full(ab), (it >> 1) & 1, abort_addr, &g_linear_status);
            tc_fence_after();
            const uint32_t acc = tmem + ab * Cfg::ACC + lane_base;
#pragma unroll 1
            for (int c0 = part * 32; c0 < Cfg::ON; c0 += 64, ob ^= 1) {
                const int col0 = n * Cfg::ON + c0;
                if (col0 >= a.n) break;  // uniform: the rest of the tile is outside
                if (a.bias) {
                    bias[lane] = bias_next[0];
                    if (GATED) bias[32 + lane] = bias_next[1];
                    __syncwarp();
                    load_bias(c0 + 64);
                }
                float y[32];
                tmem_ld32(acc + c0, y);
                if (a.bias) {
#pragma unroll
                    for (int i = 0; i < 32; ++i) y[i] += __half2float(bias[i]);
                }
                if (GATED) {
                    float u[32];
                    tmem_ld32(acc + Cfg::ON + c0, u);
                    if (a.bias) {
#pragma unroll
                        for (int i = 0; i < 32; ++i) u[i] += __half2float(bias[32 + i]);
                    }
#pragma unroll
                    for (int i = 0; i < 32; ++i) y[i] = silu(y[i]) * u[i];
                } else if (a.act == ACT_GELU) {
#pragma unroll
                    for (int i = 0; i < 32; ++i) y[i] = gelu(y[i]);
                } else if (a.act == ACT_SILU) {
#pragma unroll
                    for (int i = 0; i < 32; ++i) y[i] = silu(y[i]);
                } else if (a.act == ACT_RELU) {
#pragma unroll
                    for (int i = 0; i < 32; ++i) y[i] = relu(y[i]);
                }
                unsigned char* srow = stage + ob * 2048 + lane * 64;  // 64-byte swizzle
                if (a.residual) {
                    load_res(c0 + 64, ob ^ 1);
                    mbar_wait_uniform(res_full(warp - 2, ob), phases[ob], abort_addr,
                                      &g_linear_status);
                    phases[ob] ^= 1;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        float f[8];
                        Chunk<__half>::unpack(*reinterpret_cast<const uint4*>(
                                                  srow + ((j ^ (lane >> 1 & 3)) << 4)),
                                              f);
#pragma unroll
                        for (int e = 0; e < 8; ++e) y[8 * j + e] += f[e];
                    }
                } else {
                    // the buffer of two stores ago has been read
                    if (lane == 0) bulk_wait_read<1>();
                    __syncwarp();
                }
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    *reinterpret_cast<uint4*>(srow + ((j ^ (lane >> 1 & 3)) << 4)) =
                        make_uint4(pack_half2(y[8 * j], y[8 * j + 1]),
                                   pack_half2(y[8 * j + 2], y[8 * j + 3]),
                                   pack_half2(y[8 * j + 4], y[8 * j + 5]),
                                   pack_half2(y[8 * j + 6], y[8 * j + 7]));
                fence_async_smem();
                __syncwarp();
                if (lane == 0) {
                    tma_store_2d(&omap, col0, row_of(m) + quarter * 32, stage_addr + ob * 2048);
                    bulk_commit();
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                if (PAIR) mbar_arrive_cluster(cluster_addr(acc_empty(ab), 0));
                else mbar_arrive(acc_empty(ab));
            }
        }
        if (lane == 0) {
            bulk_wait<0>();
            // a residual tile that nobody waited for (a wait was given up) has landed, too
            for (int b = 0; b < 2; ++b) mbar_drain(res_full(warp - 2, b), (sent >> b & 1u) ^ 1u);
        }
        __syncwarp();
    }
    __syncwarp();
    if (SPLIT > 1) {
        cluster_sync_all();  // all sums have arrived
        // ---- this CTA's columns: a thread has one row of every other 8 of them
        int m, n;
        tile_of(a, tile_first, m, n);
        const int row = (warp & 3) * 32 + lane, grow = m * kM + row;
        const uint32_t acc = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
#pragma unroll 1
        for (int c = (warp - 2) >> 2; warp > 1 && c < Cfg::SHARE / 8; c += 2) {
            const int o = share * Cfg::SHARE + c * 8, col = n * Cfg::ON + o;
            if (col >= a.n) break;  // n is a multiple of 8
            auto sum = [&](int i, float (&y)[8]) {  // columns 8 i .. of the tile
                float own[8];
                tmem_ld8(acc + i * 8, own);
#pragma unroll
                for (int q = 0; q < SPLIT; ++q) {  // in order of K, whichever CTA adds
                    float x[8];
                    if (q == share) {
#pragma unroll
                        for (int e = 0; e < 8; ++e) x[e] = own[e];
                    } else {
                        const int from = q < share ? q : q - 1;
                        const float4* part =
                            reinterpret_cast<const float4*>(smem + Cfg::OFF_OUT) +
                            (from * (BN / 8 / SPLIT) + Cfg::chunk(i)) * 2 * kM + row;
                        const float4 lo = part[0], hi = part[kM];
                        x[0] = lo.x, x[1] = lo.y, x[2] = lo.z, x[3] = lo.w;
                        x[4] = hi.x, x[5] = hi.y, x[6] = hi.z, x[7] = hi.w;
                    }
#pragma unroll
                    for (int e = 0; e < 8; ++e) y[e] = q == 0 ? x[e] : y[e] + x[e];
                }
                if (a.bias) {
                    const __half* b = a.bias + (GATED && i * 8 >= Cfg::ON ? a.n + col : col);
#pragma unroll
                    for (int e = 0; e < 8; ++e) y[e] += __half2float(b[e]);
                }
            };
            float y[8];
            sum(o / 8, y);
            if (GATED) {
                float u[8];
                sum((Cfg::ON + o) / 8, u);
#pragma unroll
                for (int e = 0; e < 8; ++e) y[e] = silu(y[e]) * u[e];
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    y[e] = a.act == ACT_GELU   ? gelu(y[e])
                           : a.act == ACT_SILU ? silu(y[e])
                           : a.act == ACT_RELU ? relu(y[e])
                                               : y[e];
            }
            if (grow < a.rows) {
                if (a.residual) {
                    float f[8];
                    Chunk<__half>::unpack(
                        *reinterpret_cast<const uint4*>(a.residual + grow * a.ld_res + col), f);
#pragma unroll
                    for (int e = 0; e < 8; ++e) y[e] += f[e];
                }
                *reinterpret_cast<uint4*>(a.out + grow * a.ld_out + col) =
                    make_uint4(pack_half2(y[0], y[1]), pack_half2(y[2], y[3]),
                               pack_half2(y[4], y[5]), pack_half2(y[6], y[7]));
            }
            __syncwarp();
        }
    }
    tc_fence_before();
    if (PAIR) cluster_sync_all();  // neither CTA leaves while the other one uses its memory
    else __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        if (PAIR)
            asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem),
                         "r"(Cfg::TMEM_COLS)
                         : "memory");
        else
            asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem),
                         "r"(Cfg::TMEM_COLS)
                         : "memory");
    }
}

// Time of a whole product in units of a 128 x 1 column of accumulators over 16 of K: waves of the
// grid times a tile's.  `weight` is a tile's time a K step against 256 for a 128 x 256 tile, which
// falls more slowly than its columns, because A's part of the shared-memory and L2 traffic stays
// (measured at 8191 x 4096 x 4096, time a wave: 256 columns 31.1 us, 192 24.7, 128 20.0, 64 15.6;
// a pair of CTAs, which holds half of W each, 27.2); 1500 is what a tile costs beside its products.
inline int64_t time_of(int64_t m_tiles, int64_t n_tiles, int units, int weight, int64_t ksteps) {
    return (m_tiles * n_tiles + units - 1) / units * (weight * ksteps + 1500);
}

// Which kernel takes a product: accumulator columns of a tile, CTAs that share one (a pair or one),
// CTAs that share its K.
struct Form {
    int columns, ctas, split;
    bool gated;
};

// The fastest tile by that model: few or ragged tiles take narrow ones, large products a pair of CTAs
// (8191 x 4096 x 4096: 190 us against 218 alone, back to back under the power limit).  Few tiles with
// a long K: the split of K over a cluster with the shortest time, if that is shorter.  Handing the
// sums round costs 6 units a column and CTA, and the first 6 to 8 K steps of a CTA are in flight
// together, so shorter parts gain nothing (33 x 4096 x 512: 17.3 us in one part, 10.6, 7.6, 6.2 in
// 2, 4, 8).
inline Form choose(int64_t rows, int64_t k, int64_t n, bool gated, int sms) {
    const int64_t mt = (rows + kM - 1) / kM, mp = (rows + 2 * kM - 1) / (2 * kM);
    const int64_t ksteps = (k + 15) / 16;
    // output columns of a tile: half of a gated one's are gate columns
    auto tiles = [&](int columns) {
        const int on = gated ? columns / 2 : columns;
        return (n + on - 1) / on;
    };
    struct Tile {
        int columns, weight, max_split;
    };
    constexpr Tile kTiles[4] = {{64, 130, 8}, {128, 170, 8}, {192, 210, 2}, {256, 256, 2}};
    Form best{};
    int64_t time = INT64_MAX;
    auto offer = [&](int64_t t, int columns, int ctas, int split) {
        if (t < time) time = t, best = {columns, ctas, split, gated};
    };
    for (const Tile& c : kTiles) {
        if (gated && (c.columns == 64 || c.columns == 192)) continue;
        offer(time_of(mt, tiles(c.columns), sms, c.weight, ksteps), c.columns, 1, 1);
    }
    offer(time_of(mp, tiles(256), sms / 2, 224, ksteps), 256, 2, 1);
    for (const Tile& c : kTiles) {
        if (gated && (c.columns == 64 || c.columns == 192)) continue;
        for (int split = 2; split <= c.max_split; split *= 2) {
            // 148 SMs hold 74 clusters of 2, 33 of 4, 15 of 8 at once
            const int64_t held = split == 2 ? 74 : split == 4 ? 33 : 15;
            if (mt * tiles(c.columns) * 148 > sms * held ||
                (k + kK - 1) / kK < (c.columns == 64 ? 6 : 8) * split)
                continue;
            offer(time_of(1, 1, 1, c.weight, (ksteps + split - 1) / split) + 400 +
                      int64_t{6} * c.columns * (split - 1),
                  c.columns, 1, split);
        }
    }
    return best;
}

template <int BN, bool GATED, bool PAIR = false, int SPLIT = 1>
int launch(const void* x, int64_t ldx, const void* w, int64_t ldw, void* out, int64_t ldo,
           LinArgs a, cudaStream_t s) {
    using Cfg = LinCfg<BN, GATED, PAIR, SPLIT>;
    CUtensorMap xmap, wmap, omap;
    if (int st = make_map(&xmap, x, a.k, a.rows, ldx * 2, kM)) return st;
    if (int st = make_map(&wmap, w, GATED ? 2 * static_cast<int64_t>(a.n) : a.n, a.k, ldw * 2, kK))
        return st;
    if (int st = make_store_map(&omap, out, a.n, a.rows, ldo * 2)) return st;
    CUtensorMap rmap = omap;
    if (a.residual)
        if (int st = make_store_map(&rmap, a.residual, a.n, a.rows, a.ld_res * 2)) return st;
    a.m_tiles = PAIR ? (a.rows + 2 * kM - 1) / (2 * kM) : (a.rows + kM - 1) / kM;
    a.n_tiles = (a.n + Cfg::ON - 1) / Cfg::ON;
    int64_t tiles;
    if (!mul_ok(a.m_tiles, a.n_tiles, &tiles) || tiles > INT32_MAX)
        return fail(TMLLM_INVALID_SHAPE, "too many output tiles");
    a.tiles = static_cast<int32_t>(tiles);
    a.group_m = PAIR ? 8 : 16;
    static std::atomic<uint64_t> opted{0};
    int dev = 0;
    TMLLM_CUDA_TRY(cudaGetDevice(&dev));
    const uint64_t bit = dev < 64 ? (1ull << dev) : 0;
    if (!bit || !(opted.load(std::memory_order_relaxed) & bit)) {
        TMLLM_CUDA_TRY(cudaFuncSetAttribute(prompt_linear_kernel<BN, GATED, PAIR, SPLIT>,
                                            cudaFuncAttributeMaxDynamicSharedMemorySize,
                                            Cfg::SMEM));
        opted.fetch_or(bit, std::memory_order_relaxed);
    }
    const int sms = device_sm_count();
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute attr[1];
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = Cfg::SMEM;
    cfg.stream = s;
    if (PAIR || SPLIT > 1) {
        const int64_t pairs = tiles < sms / 2 ? tiles : sms / 2;
        cfg.gridDim = dim3(static_cast<unsigned>(PAIR ? 2 * pairs : SPLIT * tiles));
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = PAIR ? 2 : SPLIT;
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
    } else {
        cfg.gridDim = dim3(static_cast<unsigned>(tiles < sms ? tiles : sms));
    }
    TMLLM_CUDA_TRY(cudaLaunchKernelEx(&cfg, prompt_linear_kernel<BN, GATED, PAIR, SPLIT>, xmap, wmap, omap,
                                      rmap, a));
    TMLLM_LAUNCH_TRY();
    return TMLLM_OK;
}

}  // namespace

int take_linear_wait_status(int* out) { return take_status(g_linear_status, out); }

}  // namespace tmllm

using namespace tmllm;

extern "C" {

int tmllm_prompt_linear(const void* x, int64_t ldx, const void* w, int64_t ldw, const void* bias,
                        int32_t activation, const void* residual, int64_t ldr, void* out,
                        int64_t ldo, int32_t rows, int32_t k, int32_t n, tmllm_stream stream) {
    clear_error();
    if (rows < 0 || k <= 0 || n <= 0)
        return fail(TMLLM_INVALID_SHAPE, "prompt_linear dimensions must be positive");
    if (k % 8 || n % 8) return fail(TMLLM_INVALID_SHAPE, "prompt_linear needs k and n in multiples of 8");
    if (activation < ACT_NONE || activation > ACT_SWIGLU)
        return fail(TMLLM_INVALID_ARGUMENT, "unknown activation %d", activation);
    const int64_t wide = activation == ACT_SWIGLU ? 2 * static_cast<int64_t>(n) : n;
    if (rows > INT32_MAX - 1024 || k > INT32_MAX - 1024 || wide > INT32_MAX - 1024)
        return fail(TMLLM_INVALID_SHAPE, "prompt_linear dimensions must fit 31 bits");
    if (rows == 0) return TMLLM_OK;
    if (!x || !w || !out) return fail(TMLLM_INVALID_ARGUMENT, "null tensor pointer");
    int64_t span;
    for (int64_t ld : {ldx, ldw, ldo, ldr})
        if (ld % 8 || ld > (int64_t{1} << 38))  // the tensor maps' stride limit is 2^40 bytes
            return fail(TMLLM_INVALID_SHAPE, "row strides must be multiples of 8 elements");
    if (ldx < k || ldw < wide || ldo < n || (residual && ldr < n))
        return fail(TMLLM_INVALID_SHAPE, "row strides must cover a row");
    for (int64_t ld : {ldx, ldo, residual ? ldr : 0})
        if (!mul_ok(rows, ld, &span) || span > INT64_MAX / 8)
            return fail(TMLLM_INVALID_SHAPE, "rows and row strides must fit 60 bits");
    if (!mul_ok(k, ldw, &span) || span > INT64_MAX / 8)
        return fail(TMLLM_INVALID_SHAPE, "rows and row strides must fit 60 bits");
    for (const void* p : {x, w, residual, static_cast<const void*>(out)})
        if (!aligned16(p))
            return fail(TMLLM_INVALID_ARGUMENT, "x, w, residual and out must be 16-byte aligned");
    if (reinterpret_cast<uintptr_t>(bias) % 2)
        return fail(TMLLM_INVALID_ARGUMENT, "bias must be aligned to its element size");
    // tiles are stored while others are still read: out may be the residual itself only
    if (overlaps({out, ldo, n}, {x, ldx, k}, rows, 2) ||
        (residual && !(residual == out && ldr == ldo) &&
         overlaps({out, ldo, n}, {residual, ldr, n}, rows, 2)))
        return fail(TMLLM_INVALID_ARGUMENT, "out overlaps x, or the residual without being it");
    const uintptr_t o0 = reinterpret_cast<uintptr_t>(out), w0 = reinterpret_cast<uintptr_t>(w);
    const uintptr_t o1 = o0 + 2 * static_cast<uintptr_t>((rows - 1) * ldo + n);
    const uintptr_t w1 = w0 + 2 * static_cast<uintptr_t>((k - 1) * ldw + wide);
    if (o0 < w1 && w0 < o1) return fail(TMLLM_INVALID_ARGUMENT, "out overlaps W");
    if (inside(bias, 2 * wide, {out, ldo, n}, rows, 2))
        return fail(TMLLM_INVALID_ARGUMENT, "out overlaps the bias");
    LinArgs a{};
    a.bias = static_cast<const __half*>(bias);
    a.residual = static_cast<const __half*>(residual);
    a.out = static_cast<__half*>(out);
    a.ld_res = ldr;
    a.ld_out = ldo;
    a.rows = rows;
    a.k = k;
    a.n = n;
    a.act = activation;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    const Form f = choose(rows, k, n, activation == ACT_SWIGLU, device_sm_count());
    auto go = [&](auto bn, auto gated, auto pair, auto split) {
        return launch<bn(), gated(), pair(), split()>(x, ldx, w, ldw, out, ldo, a, s);
    };
    std::integral_constant<int, 64> c64;
    std::integral_constant<int, 128> c128;
    std::integral_constant<int, 192> c192;
    std::integral_constant<int, 256> c256;
    std::integral_constant<int, 1> s1;
    std::integral_constant<int, 2> s2;
    std::integral_constant<int, 4> s4;
    std::integral_constant<int, 8> s8;
    std::true_type yes;
    std::false_type no;
    if (f.gated) {
        if (f.ctas == 2) return go(c256, yes, yes, s1);
        if (f.columns == 256) return f.split == 1 ? go(c256, yes, no, s1) : go(c256, yes, no, s2);
        switch (f.split) {
            case 1: return go(c128, yes, no, s1);
            case 2: return go(c128, yes, no, s2);
            case 4: return go(c128, yes, no, s4);
            default: return go(c128, yes, no, s8);
        }
    }
    if (f.ctas == 2) return go(c256, no, yes, s1);
    if (f.columns == 256) return f.split == 1 ? go(c256, no, no, s1) : go(c256, no, no, s2);
    if (f.columns == 192) return f.split == 1 ? go(c192, no, no, s1) : go(c192, no, no, s2);
    if (f.columns == 128) switch (f.split) {
            case 1: return go(c128, no, no, s1);
            case 2: return go(c128, no, no, s2);
            case 4: return go(c128, no, no, s4);
            default: return go(c128, no, no, s8);
        }
    switch (f.split) {
        case 1: return go(c64, no, no, s1);
        case 2: return go(c64, no, no, s2);
        case 4: return go(c64, no, no, s4);
        default: return go(c64, no, no, s8);
    }
}

int tmllm_prompt_linear_form(int32_t rows, int32_t k, int32_t n, int32_t activation, int32_t sms,
                             int32_t* form) {
    clear_error();
    if (!form) return fail(TMLLM_INVALID_ARGUMENT, "null output");
    if (rows <= 0 || k <= 0 || n <= 0 || sms < 0)
        return fail(TMLLM_INVALID_SHAPE, "prompt_linear dimensions must be positive");
    if (activation < ACT_NONE || activation > ACT_SWIGLU)
        return fail(TMLLM_INVALID_ARGUMENT, "unknown activation %d", activation);
    const Form f = choose(rows, k, n, activation == ACT_SWIGLU, sms ? sms : device_sm_count());
    form[0] = f.columns;
    form[1] = f.ctas;
    form[2] = f.split;
    return TMLLM_OK;
}

}  // extern "C"
