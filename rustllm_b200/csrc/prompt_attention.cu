// Causal attention over whole packed prompts (tmllm_prompt_attention): sequences of different
// lengths back to back, grouped query heads, no cache.
//
//   o_i = sum_{j <= i} p_ij v_j,  p_ij = exp(scale q_i . k_j - lse_i),
//   lse_i = ln sum_{j <= i} exp(scale q_i . k_j)
//
// per sequence and query head, keys and values of KV head h / (Hq / Hkv)
// (nn/attention.rs:216-247 with start = 0).  One pass over the keys with the running maximum
// m and sum l of each row (O and l are rescaled by 2^(m_old - m_new) when m grows), so the
// score matrix never leaves the SM.
#include <atomic>
#include <cmath>

#include "common.cuh"
#include "tc.cuh"

namespace tmllm {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

struct PromptArgs {
    const void* q;
    const void* k;
    const void* v;
    void* out;
    float* lse;  // [rows, q_heads] or null
    const int32_t* q_start;
    int64_t rows;
    int64_t q_stride, kv_stride, out_stride;
    int32_t num_seqs, max_rows, q_heads, kv_heads, group, head_dim, out_f32;
    int32_t pairs;  // tensor-core form: a unit is 0 one item, 1 two heads, 2 two row tiles
    float scale_log2;
};

__device__ int g_attention_status;

// First row and row count of sequence s, clipped to the packed rows that exist.
__device__ __forceinline__ int seq_rows(const PromptArgs& a, int s, int64_t* row0) {
    int64_t lo = a.q_start[s], hi = a.q_start[s + 1];
    if (hi > a.rows) hi = a.rows;
    if (lo < 0 || lo >= hi) return 0;
    *row0 = lo;
    return static_cast<int>(hi - lo);
}

// ---- CUDA-core form: any type and head size up to 256 -----------------------------------
// One CTA per (TT / 16 RT query rows, query head, sequence), which goes on to the rows a launch's
// worth behind them in a sequence longer than the launch was sized for; TEAMS teams of TT threads that take
// every TEAMS-th tile of keys each and are joined at the end.  Thread (ty, tx) of a team holds RT
// rows from RT ty on of S (columns tx + 16 c of a tile of 64 keys) and of O (columns 4 tx + 64 c
// on).  DP: head size rounded up to 64 / 128 / 256.  Both products run on packed F32 pairs (two
// multiply-adds an instruction) out of 16-byte shared-memory reads: 8 RT multiply-add pairs for
// RT + 4 reads of 4 cycles each, which is what bounds it at long prompts (4096 tokens, 8 / 2 heads
// of 128: 928 us, 37 TFLOP/s; 64 x 700 tokens, 9 / 3 heads of 64: 1080 us, 33), so few threads with
// many rows each; at short ones the chain of a CTA's tiles does, so a second team.  With F32 rows
// on the 16-byte grid K and V are copied asynchronously, and a single team (DP <= 128) copies the
// next tile while this one is computed.
constexpr int kFmaTile = 64;  // keys

template <int DP, int RT, int TT, int TEAMS>
struct FmaCfg {
    static constexpr int ROWS = TT / 16 * RT;
    static constexpr int LD = DP + 4;  // pitch of Q and K: rows 16 bytes apart in the banks
    static constexpr int BUFS = TEAMS == 1 && DP <= 128 ? 2 : 1;  // of each team
    static constexpr int KV = kFmaTile * (LD + DP);  // floats of a K and a V tile
    static constexpr int LP = kFmaTile + 4;
    static constexpr int PS = ROWS * LP;
    static constexpr int SMEM = (ROWS * LD + TEAMS * (BUFS * KV + PS)) * 4;
    // a team's results fit where its tiles were
    static_assert(TT * RT * (DP / 16 + 2) <= BUFS * KV, "merge");
};

// Barrier `id` of `threads` threads, and whether one of them has x.
template <int THREADS>
__device__ __forceinline__ bool barrier_or(int id, bool x) {
    uint32_t any;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.u32 p, %1, 0;\n\t"
        "barrier.cta.red.or.pred q, %2, %3, p;\n\t"
        "selp.u32 %0, 1, 0, q;\n\t}"
        : "=r"(any)
        : "r"(static_cast<uint32_t>(x)), "r"(id), "n"(THREADS)
        : "memory");
    return any != 0;
}

// Rows q_lo .. of query head h of the sequence of n rows from row0 on.
template <typename T, int DP, int RT, int TT, int TEAMS>
__device__ __forceinline__ void fma_rows(const PromptArgs& a, float* fsm, int h, int64_t row0, int n,
                                         int q_lo, int async) {
    using Cfg = FmaCfg<DP, RT, TT, TEAMS>;
    constexpr int ROWS = Cfg::ROWS, LD = Cfg::LD, LP = Cfg::LP, CG = DP / 64;
    float* qs = fsm;                          // [ROWS][LD]
    const int team = TEAMS == 1 ? 0 : threadIdx.x / TT;
    float* kv0 = qs + ROWS * LD + team * (Cfg::BUFS * Cfg::KV + Cfg::PS);  // [BUFS]: K [64][LD],
                                                                           // V [64][DP]
    float* ps = kv0 + Cfg::BUFS * Cfg::KV;                                 // [ROWS][LP]
    const int kvh = h / a.group, D = a.head_dim;
    const int tid = threadIdx.x % TT, tx = tid & 15, ty = tid >> 4;
    const T* qg = static_cast<const T*>(a.q) + (row0 + q_lo) * a.q_stride +
                  static_cast<int64_t>(h) * D;
    const T* kg = static_cast<const T*>(a.k) + row0 * a.kv_stride + static_cast<int64_t>(kvh) * D;
    const T* vg = static_cast<const T*>(a.v) + row0 * a.kv_stride + static_cast<int64_t>(kvh) * D;
    const int q_hi = q_lo + ROWS < n ? q_lo + ROWS : n;  // keys [0, q_hi) are visible
    // rows j0 .. of K and V (zeros past the last visible key and the head size)
    auto load = [&](int j0, int buf) {
        float* ks = kv0 + buf * Cfg::KV;
        float* vs = ks + kFmaTile * LD;
        if (async) {
            for (int i = tid; i < kFmaTile * (DP / 4); i += TT) {
                const int r = i / (DP / 4), c = (i % (DP / 4)) * 4;
                const bool in = j0 + r < q_hi && c < D;  // D is a multiple of 4 here
                const int64_t off = in ? static_cast<int64_t>(j0 + r) * a.kv_stride + c : 0;
                cp_async16(ks + r * LD + c, kg + off, in ? 16 : 0);
                cp_async16(vs + r * DP + c, vg + off, in ? 16 : 0);
            }
            cp_async_commit();
        } else {
            for (int i = tid; i < kFmaTile * DP; i += TT) {
                const int r = i / DP, c = i % DP;
                const bool in = j0 + r < q_hi && c < D;
                const int64_t off = static_cast<int64_t>(j0 + r) * a.kv_stride + c;
                ks[r * LD + c] = in ? to_f32<T>(kg[off]) : 0.f;
                vs[r * DP + c] = in ? to_f32<T>(vg[off]) : 0.f;
            }
        }
    };
    constexpr int STRIDE = TEAMS * kFmaTile;  // between a team's tiles
    if (team * kFmaTile < q_hi) load(team * kFmaTile, 0);
    for (int i = threadIdx.x; i < ROWS * DP; i += TT * TEAMS) {
        const int r = i / DP, c = i % DP;
        qs[r * LD + c] = (q_lo + r < n && c < D) ? to_f32<T>(qg[r * a.q_stride + c]) : 0.f;
    }
    float2 o[RT][2 * CG];
    float m[RT], l[RT];
#pragma unroll
    for (int i = 0; i < RT; ++i) {
        m[i] = -INFINITY;
        l[i] = 0.f;
#pragma unroll
        for (int c = 0; c < 2 * CG; ++c) o[i][c] = make_float2(0.f, 0.f);
    }
    if (TEAMS > 1) __syncthreads();  // Q
    auto team_sync = [&]() {
        if (TEAMS == 1) __syncthreads();
        else asm volatile("barrier.cta.sync %0, %1;" ::"r"(1 + team), "n"(TT) : "memory");
    };
    int buf = 0;
    for (int j0 = team * kFmaTile; j0 < q_hi; j0 += STRIDE) {
        const bool ahead = Cfg::BUFS == 2 && async && j0 + STRIDE < q_hi;
        if (ahead) {
            load(j0 + STRIDE, buf ^ 1);
            cp_async_wait<1>();
        } else {
            cp_async_wait<0>();
        }
        team_sync();
        const float* ks = kv0 + buf * Cfg::KV;
        const float* vs = ks + kFmaTile * LD;
        const bool diag = j0 + kFmaTile > q_lo;
        // 0 * inf is not 0: a diagonal tile with non-finite values takes the masked product
        bool odd = false;
        if (diag) {
            for (int i = tid; i < kFmaTile * DP; i += TT) odd |= !(fabsf(vs[i]) < INFINITY);
            odd = TEAMS == 1 ? __syncthreads_or(odd) != 0 : barrier_or<TT>(1 + team, odd);
        }
        float2 s2[RT][4];
#pragma unroll
        for (int i = 0; i < RT; ++i)
#pragma unroll
            for (int c = 0; c < 4; ++c) s2[i][c] = make_float2(0.f, 0.f);
#pragma unroll 4
        for (int d = 0; d < D; d += 4) {  // rows are zero past D
            float4 qv[RT], kv[4];
#pragma unroll
            for (int i = 0; i < RT; ++i)
                qv[i] = *reinterpret_cast<const float4*>(qs + (RT * ty + i) * LD + d);
#pragma unroll
            for (int c = 0; c < 4; ++c)
                kv[c] = *reinterpret_cast<const float4*>(ks + (tx + 16 * c) * LD + d);
#pragma unroll
            for (int i = 0; i < RT; ++i)
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    s2[i][c] = __ffma2_rn(make_float2(qv[i].x, qv[i].y),
                                          make_float2(kv[c].x, kv[c].y), s2[i][c]);
                    s2[i][c] = __ffma2_rn(make_float2(qv[i].z, qv[i].w),
                                          make_float2(kv[c].z, kv[c].w), s2[i][c]);
                }
        }
#pragma unroll
        for (int i = 0; i < RT; ++i) {
            const int qi = q_lo + RT * ty + i;
            float sc[4], mt = -INFINITY;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                sc[c] = j0 + tx + 16 * c <= qi ? (s2[i][c].x + s2[i][c].y) * a.scale_log2 : -INFINITY;
                mt = fmaxf(mt, sc[c]);
            }
#pragma unroll
            for (int w = 8; w > 0; w >>= 1) mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, w));
            const float mn = fmaxf(m[i], mt);
            const float base = mn == -INFINITY ? 0.f : mn;  // nothing visible yet: exp2(-inf)
            const float corr = exp2f(m[i] - base);
            float ls = 0.f;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const float p = exp2f(sc[c] - base);
                ps[(RT * ty + i) * LP + tx + 16 * c] = p;
                ls += p;
            }
#pragma unroll
            for (int w = 8; w > 0; w >>= 1) ls += __shfl_xor_sync(0xffffffffu, ls, w);
            l[i] = l[i] * corr + ls;
            m[i] = mn;
#pragma unroll
            for (int c = 0; c < 2 * CG; ++c)
                o[i][c] = make_float2(o[i][c].x * corr, o[i][c].y * corr);
        }
        __syncwarp();  // the rows of ps a warp reads are the ones its own lanes wrote
        if (!odd) {
#pragma unroll 2
            for (int j = 0; j < kFmaTile; j += 4) {  // P is zero for keys that are not there
                float4 pv[RT];
#pragma unroll
                for (int i = 0; i < RT; ++i)
                    pv[i] = *reinterpret_cast<const float4*>(ps + (RT * ty + i) * LP + j);
#pragma unroll
                for (int c = 0; c < CG; ++c)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float4 vv =
                            *reinterpret_cast<const float4*>(vs + (j + e) * DP + 64 * c + 4 * tx);
#pragma unroll
                        for (int i = 0; i < RT; ++i) {
                            const float p = e == 0 ? pv[i].x : e == 1 ? pv[i].y : e == 2 ? pv[i].z : pv[i].w;
                            const float2 p2 = make_float2(p, p);
                            o[i][2 * c] = __ffma2_rn(p2, make_float2(vv.x, vv.y), o[i][2 * c]);
                            o[i][2 * c + 1] = __ffma2_rn(p2, make_float2(vv.z, vv.w), o[i][2 * c + 1]);
                        }
                    }
            }
        } else {
            const int nk = q_hi - j0 < kFmaTile ? q_hi - j0 : kFmaTile;
            for (int j = 0; j < nk; ++j)
                for (int i = 0; i < RT; ++i) {
                    if (j0 + j > q_lo + RT * ty + i) continue;
                    const float p = ps[(RT * ty + i) * LP + j];
#pragma unroll
                    for (int c = 0; c < CG; ++c) {
                        const float* vv = vs + j * DP + 64 * c + 4 * tx;
                        o[i][2 * c].x = fmaf(p, vv[0], o[i][2 * c].x);
                        o[i][2 * c].y = fmaf(p, vv[1], o[i][2 * c].y);
                        o[i][2 * c + 1].x = fmaf(p, vv[2], o[i][2 * c + 1].x);
                        o[i][2 * c + 1].y = fmaf(p, vv[3], o[i][2 * c + 1].y);
                    }
                }
        }
        team_sync();  // the tiles are done with
        if (ahead) {
            buf ^= 1;
        } else if (j0 + STRIDE < q_hi) {
            load(j0 + STRIDE, buf);
        }
    }
    if (TEAMS > 1) {  // the first team joins the others' rows to its own
        float2* part = reinterpret_cast<float2*>(kv0);  // [RT (2 CG + 1)][TT]
        constexpr int W = 2 * CG + 1;
        if (team > 0) {
#pragma unroll
            for (int i = 0; i < RT; ++i) {
#pragma unroll
                for (int c = 0; c < 2 * CG; ++c) part[(i * W + c) * TT + tid] = o[i][c];
                part[(i * W + 2 * CG) * TT + tid] = make_float2(m[i], l[i]);
            }
        }
        __syncthreads();
        if (team > 0) return;
#pragma unroll
        for (int t = 1; t < TEAMS; ++t) {
            part = reinterpret_cast<float2*>(kv0 + t * (Cfg::BUFS * Cfg::KV + Cfg::PS));
#pragma unroll
            for (int i = 0; i < RT; ++i) {
                const float2 ml = part[(i * W + 2 * CG) * TT + tid];
                const float mn = fmaxf(m[i], ml.x), base = mn == -INFINITY ? 0.f : mn;
                const float own = exp2f(m[i] - base), its = exp2f(ml.x - base);
                l[i] = l[i] * own + ml.y * its;
                m[i] = mn;
#pragma unroll
                for (int c = 0; c < 2 * CG; ++c) {
                    const float2 x = part[(i * W + c) * TT + tid];
                    o[i][c] = make_float2(fmaf(x.x, its, o[i][c].x * own),
                                          fmaf(x.y, its, o[i][c].y * own));
                }
            }
        }
    }
    bool none = false;
#pragma unroll
    for (int i = 0; i < RT; ++i) none |= l[i] == 0.f;
    if (none) {  // every score of a row -inf: zeros, whatever the values are (0 * inf is not 0)
#pragma unroll
        for (int i = 0; i < RT; ++i) {
            if (l[i] != 0.f) continue;
#pragma unroll
            for (int c = 0; c < 2 * CG; ++c) o[i][c] = make_float2(0.f, 0.f);
        }
    }
#pragma unroll
    for (int i = 0; i < RT; ++i) {
        const int r = q_lo + RT * ty + i;
        if (r >= n) continue;
        const float inv = l[i] == 0.f ? 0.f : 1.f / l[i];
        const int64_t off = (row0 + r) * a.out_stride + static_cast<int64_t>(h) * D;
#pragma unroll
        for (int c = 0; c < CG; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int d = 64 * c + 4 * tx + e;
                if (d >= D) continue;
                const float2 x = o[i][2 * c + (e >> 1)];
                const float y = ((e & 1) ? x.y : x.x) * inv;
                if (a.out_f32) static_cast<float*>(a.out)[off + d] = y;
                else static_cast<T*>(a.out)[off + d] = from_f32<T>(y);
            }
        if (a.lse && tx == 0)
            a.lse[(row0 + r) * a.q_heads + h] =
                ((m[i] == -INFINITY ? 0.f : m[i]) + log2f(l[i])) * kLn2;
    }
}

// The same out of line, for the rows past the launch's.  One team of up to 128 columns: as a loop
// around the code above the usual single pass was slower (F32, 64 x 700 tokens, 9/3 heads of 64:
// 1115 us against 1081; 4096 tokens, 8/2 heads of 128: 934 against 928); the others are better off
// with the loop (prompts of 50, 3 and 100 tokens, 9/3 heads of 64: 8.6 us against 9.8; 4 x 1000,
// 8/2 heads of 256: 472 against 475).
template <typename T, int DP, int RT, int TT, int TEAMS>
__device__ __noinline__ void fma_more_rows(const PromptArgs& a, float* fsm, int h, int64_t row0,
                                           int n, int q_lo, int async) {
    __syncthreads();  // the rows before are done with the shared memory
    fma_rows<T, DP, RT, TT, TEAMS>(a, fsm, h, row0, n, q_lo, async);
}

template <typename T, int DP, int RT, int TT, int TEAMS>
__global__ void __launch_bounds__(TT * TEAMS) prompt_fma_kernel(const __grid_constant__ PromptArgs a,
                                                                 int row_tiles, int async) {
    constexpr int ROWS = FmaCfg<DP, RT, TT, TEAMS>::ROWS;
    extern __shared__ __align__(16) float fsm[];
    const int64_t hb = static_cast<int64_t>(a.q_heads) * a.num_seqs;
    const int tile = row_tiles - 1 - static_cast<int>(blockIdx.x / hb);
    const int h = static_cast<int>(blockIdx.x % hb) % a.q_heads;
    const int s = static_cast<int>(blockIdx.x % hb) / a.q_heads;
    int64_t row0 = 0;
    const int n = seq_rows(a, s, &row0);
    const int64_t step = static_cast<int64_t>(row_tiles) * ROWS;
    int64_t q_lo = static_cast<int64_t>(tile) * ROWS;
    if constexpr (TEAMS == 1 && DP <= 128) {
        if (q_lo >= n) return;
        fma_rows<T, DP, RT, TT, TEAMS>(a, fsm, h, row0, n, static_cast<int>(q_lo), async);
        for (q_lo += step; q_lo < n; q_lo += step)
            fma_more_rows<T, DP, RT, TT, TEAMS>(a, fsm, h, row0, n, static_cast<int>(q_lo), async);
    } else {
        while (q_lo < n) {
            fma_rows<T, DP, RT, TT, TEAMS>(a, fsm, h, row0, n, static_cast<int>(q_lo), async);
            q_lo += step;
            if (q_lo < n) __syncthreads();  // the rows are done with the shared memory
        }
    }
}

template <typename T, int DP, int RT, int TT, int TEAMS>
int launch_fma_rows(const PromptArgs& a, cudaStream_t s) {
    const int row_tiles = (a.max_rows + FmaCfg<DP, RT, TT, TEAMS>::ROWS - 1) / FmaCfg<DP, RT, TT, TEAMS>::ROWS;
    int64_t ctas;
    if (!mul_ok(static_cast<int64_t>(row_tiles) * a.q_heads, a.num_seqs, &ctas) ||
        ctas > INT32_MAX)
        return fail(TMLLM_INVALID_SHAPE, "too many prompt tiles");
    constexpr int smem = FmaCfg<DP, RT, TT, TEAMS>::SMEM;
    static_assert(smem <= 227 * 1024, "shared memory of one CTA");
    const int async = sizeof(T) == 4 && a.head_dim % 4 == 0 && a.kv_stride % 4 == 0 &&
                      aligned16(a.k) && aligned16(a.v);
    TMLLM_CUDA_TRY(cudaFuncSetAttribute(prompt_fma_kernel<T, DP, RT, TT, TEAMS>,
                                        cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    prompt_fma_kernel<T, DP, RT, TT, TEAMS>
        <<<static_cast<unsigned>(ctas), TT * TEAMS, smem, s>>>(a, row_tiles, async);
    TMLLM_LAUNCH_TRY();
    return TMLLM_OK;
}

// 64 query rows a CTA read K and V half as often; 32 spread a small batch over more SMs, and two
// teams halve its longest CTA (F32, 2 x 500 tokens, 8 / 2 heads of 128: 49 us against 65 with one
// team of 256 threads; but 512 CTAs over 4096 tokens, heads of 128: 1016 against 928, and 64 x 700
// tokens, 9 / 3 heads of 64: 1187 against 1082).
template <typename T, int DP>
int launch_fma(const PromptArgs& a, cudaStream_t s) {
    const bool small = (a.rows / 64 + a.num_seqs) * a.q_heads < 2 * device_sm_count();
    if constexpr (DP <= 128) {
        if (small) return launch_fma_rows<T, DP, 4, 128, 2>(a, s);
        return DP == 64 ? launch_fma_rows<T, 64, 8, 128, 1>(a, s)
                        : launch_fma_rows<T, DP, 4, 256, 1>(a, s);
    } else {  // one tile of K and V fills the shared memory
        return small ? launch_fma_rows<T, DP, 2, 256, 1>(a, s)
                     : launch_fma_rows<T, DP, 4, 256, 1>(a, s);
    }
}

template <typename T>
int launch_fma_d(const PromptArgs& a, cudaStream_t s) {
    if (a.head_dim <= 64) return launch_fma<T, 64>(a, s);
    if (a.head_dim <= 128) return launch_fma<T, 128>(a, s);
    return launch_fma<T, 256>(a, s);
}


// ---- tensor-core form: F16, head size a multiple of 8 up to 128 -------------------------
// Tiles are cut from the packed rows, not from the sequences: an item is 128 packed rows (whatever
// sequences they belong to) of one query head, and a row sees the keys from its own sequence's
// first row to itself.  So 500 prompts of one token are four row tiles, not 500.  Keys are tiled
// on the same grid: the tile of the item's own rows is the last one it reads, the tile holding
// the first row's sequence start the first one.
// A unit is two items that stream the same K and V tiles: two heads of a KV group over the same
// rows, or (odd groups) two neighbouring row tiles of one head.  Per CTA:
//   warps 0-3, 4-7  softmax of item 0 / 1, one thread a query row
//   warp 8          TMA producer: Q tiles, then K and V tiles through a ring
//   warps 9, 10     MMA issuers of item 0 / 1
//   warp 11         scrub (below)
// K and V arrive in tiles of 128 keys and are used in steps of KS: 64 above head size 64, where the
// accumulators leave less tensor memory, and for short prompts, whose masked steps cost more than
// a step's fixed part (9/3 heads of 64: 512 prompts of 300 tokens, 345 us in steps of 128 and 260 in
// steps of 64; 16 of 2048 tokens 126 and 136), else 128.  S = Q K^T of a step sits in tensor memory;
// its rows are read to registers (and the next step's S is computed over it), exponentiated, and P
// is written to columns of its own as F16, from where it is the A operand of O += P V, so only V
// crosses shared memory for the second product.
//   tensor memory: S_i at [KS i, + KS), P_i at [2 KS + KS / 2 i, + KS / 2), O_i at
//   [512 - DP (2 - i), + DP)
//
// Bound by the softmax groups' own chain of waits, loads, maximum, exponentials and stores: a step
// of 64 keys of two items of head size 128 takes about 1,850 cycles, of which the tensor pipe needs
// 1,024 and the exponentials 768 of the MUFU's (1,024 without the quarter that goes to the
// multiply-add pipe); 54 % of the issue slots are used.  16384 rows of 32/8 heads of 128: 1.75 ms,
// 1.26 PFLOP/s; 4 x 4096 rows of 32/8 heads of 64: 359 us, 766 TFLOP/s; 64 prompts of 1 to 2048
// tokens (39,424 rows), 15/5 heads of 64: 221 us in a graph, 450 TFLOP/s.
//
// Masked places never reach a result: scores that a row does not see are replaced by -inf before
// the maximum, and since 0 * inf is not 0, the non-finite entries of every V tile that some row
// of the unit does not see whole are zeroed in shared memory before the product and added
// afterwards to the rows that see them ("scrubbed" tiles: the diagonal, the tile where the
// sequence starts, all tiles of an item whose rows belong to several sequences).  The mask of the
// units that had some leaves out keys of no sequence, so that NaN in padding costs nothing.
constexpr int kTile = 128;
constexpr int kTcThreads = 384;
constexpr int kWindow = 1024;    // row tiles a launch schedules (131,072 packed rows)

template <int DP, int KSV>
struct AttCfg {
    static constexpr int BLK = 16384;          // 64 columns x 128 rows, swizzled
    static constexpr int TILE = DP / 64 * BLK; // Q, K or V tile
    static constexpr int QBUF = DP == 64 ? 2 : 1;
    static constexpr int STAGES = DP == 64 ? 8 : 4;
    static constexpr int OFF_KV = 2 * QBUF * TILE;
    static constexpr int OFF_SEQ = OFF_KV + STAGES * TILE;      // int32 see AttSched::tile_seq
    static constexpr int OFF_FIRST = OFF_SEQ + kWindow * 4;     // uint32 see AttSched::tile_first
    static constexpr int OFF_HIST = OFF_FIRST + kWindow * 4;    // int32 row tiles of each cost
    static constexpr int OFF_COST = OFF_HIST + kWindow * 4;     // uint16 key tiles of an entry
    static constexpr int OFF_LIST = OFF_COST + kWindow * 2;     // uint16 entries, longest first
    static constexpr int OFF_OUT = OFF_LIST + kWindow * 2;      // a warp's 32 rows x 64 bytes, x 8
    static constexpr int OFF_BAR = OFF_OUT + 8 * 2048;
    static constexpr int KS = KSV;        // keys of a step
    static constexpr int SPT = 128 / KS;  // steps of a key tile
    static_assert(3 * KS + 2 * DP <= 512, "tensor memory");
    static constexpr int SMEM = OFF_BAR + 512 + 1024;  // + alignment
    static_assert(SMEM <= 227 * 1024, "shared memory of one CTA");
};

// Barriers: QF/QE Q tile full / empty, KF/KE ring full / empty, SB V tile of a ring stage ready for
// the product; of each item: S scores ready, F scores read, P probabilities written, O product done, E
// accumulator read; DONE all products.  Both MMA warps give back every K and V tile, whether their
// item uses it or not, so no role falls more than a phase behind the ring.
template <int DP, int KSV>
struct AttBar {
    using Cfg = AttCfg<DP, KSV>;
    static constexpr int QF = 0, QE = QF + 2 * Cfg::QBUF, KF = QE + 2 * Cfg::QBUF,
                         KE = KF + Cfg::STAGES, S = KE + Cfg::STAGES, F = S + 2, P = F + 2,
                         O = P + 2, E = O + 2, SB = E + 2, DONE = SB + Cfg::STAGES,
                         COUNT = DONE + 1;
    static_assert(COUNT * 8 + 64 <= 512, "barrier area");
};

// Last sequence whose first row is <= row, among [lo, hi].
__device__ __forceinline__ int seq_at(const PromptArgs& a, int row, int lo, int hi) {
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (__ldg(a.q_start + mid) <= row) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

struct AttUnit {
    int kvh, jlo, jhi;         // key tiles the unit streams
    int head[2], tile[2];      // query head and row tile of each item
    int lo[2], hi[2];          // its steps (lo > hi: no such item)
    bool several[2];           // its rows belong to more than one sequence
    bool any_several;
    int first;                 // first visible key of the unit's first row
    __device__ __forceinline__ bool on(int i) const { return lo[i] <= hi[i]; }
    // the same values in every lane, and known to be
    __device__ __forceinline__ void make_uniform() {
        auto bc = [](int x) { return __shfl_sync(0xffffffffu, x, 0); };
        kvh = bc(kvh), jlo = bc(jlo), jhi = bc(jhi), first = bc(first);
        any_several = bc(any_several);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            head[i] = bc(head[i]), tile[i] = bc(tile[i]), lo[i] = bc(lo[i]), hi[i] = bc(hi[i]);
            several[i] = bc(several[i]);
        }
    }
    // some row of the unit does not see key tile j whole
    __device__ __forceinline__ bool ragged(int j) const {
        return any_several || j == tile[0] || j == tile[1] || j * kTile < first;
    }
};

// The work list every role of every CTA walks in the same order: row tiles with the longest key
// range first, heads innermost (they share K and V in L2), dealt to the CTAs in a snake so their
// sums come out alike.
struct AttSched {
    const int32_t* tile_seq;     // of each row tile of the window: sequence of its first row,
    const uint32_t* tile_first;  // that sequence's first row, and kSeveral if it ends in the tile
    const uint16_t* list;
    int row_lo, row_hi;          // live rows
    int tile0, tile_end;         // the window's first tile; its live ones end here (relative)
    int per, total, k;           // units of a list entry
    static constexpr uint32_t kSeveral = 1u << 31;

    // first row of the sequence of a row of (absolute) tile t
    __device__ __forceinline__ int row_first(const PromptArgs& a, int t, int row) const {
        t -= tile0;
        const uint32_t f = tile_first[t];
        if (!(f & kSeveral)) return static_cast<int>(f);
        const int hi = t + 1 < tile_end ? tile_seq[t + 1] : a.num_seqs - 1;
        return max(__ldg(a.q_start + seq_at(a, row, tile_seq[t], hi)), 0);
    }

    template <int KS>
    __device__ __forceinline__ bool next(const PromptArgs& a, AttUnit& u) {
        const int G = gridDim.x;
        int idx;
        do {
            const int64_t base = static_cast<int64_t>(k) * G;
            if (base >= total) return false;
            const int64_t at = (k & 1) ? base + G - 1 - blockIdx.x : base + blockIdx.x;
            ++k;
            idx = at < total ? static_cast<int>(at) : -1;
        } while (idx < 0);
        const int rank = idx / per;
        int rem = idx - rank * per;
        const int np = per / a.kv_heads;
        u.kvh = rem / np;
        rem -= u.kvh * np;
        u.any_several = false;
        const int st = list[rank];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            int tile = st, g = rem;
            bool in = true;
            if (a.pairs == 1) g = 2 * rem + i;     // two heads of the group
            else if (a.pairs == 2) tile = 2 * st + i;  // two row tiles of one head
            else in = i == 0;
            const int r0 = (tile0 + tile) * kTile;
            in = in && r0 < row_hi && r0 + kTile > row_lo;
            u.head[i] = u.kvh * a.group + g;
            u.tile[i] = tile0 + tile;
            u.lo[i] = 1;
            u.hi[i] = 0;
            u.several[i] = false;
            if (!in) continue;
            const uint32_t f = tile_first[tile];
            const int end = r0 + kTile < row_hi ? r0 + kTile : row_hi;
            u.several[i] = f >> 31;
            u.any_several |= u.several[i];
            const int first = static_cast<int>(f & ~kSeveral);
            u.lo[i] = first / KS;
            u.hi[i] = (end - 1) / KS;
            if (i == 0 || !u.on(0)) u.first = first;
        }
        u.jlo = (u.on(0) ? u.lo[0] : u.lo[1]) / (kTile / KS);
        u.jhi = (u.on(1) ? u.hi[1] : u.hi[0]) / (kTile / KS);
        return true;
    }
};

__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// 2^x of two numbers on the multiply-add pipe: x = n + f with n the nearest integer (it appears in
// the low bits of x + 1.5 2^23), 2^f by a polynomial on [-1/2, 1/2] (degree 4, least-squares fit
// reweighted to an even relative error of 2.6e-6; P is rounded to 2^-11 behind it) and 2^n put
// together as a float.  -127 and below give 0, NaN stays.  The softmax's time is the MUFU unit's,
// which does 4 exponentials a cycle and quarter of an SM, so every fourth pair is computed here
// (4 x 4096 tokens, 32/8 heads of 64: 375 us without, 358 with every eighth, 359 every fourth,
// 377 every third).
__device__ __forceinline__ float2 exp2_fma(float2 x) {
    constexpr float C0 = 0.999999285f, C1 = 0.693121791f, C2 = 0.240247443f, C3 = 0.0559178367f,
                    C4 = 0.00957007986f;
    float a, b;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(a) : "f"(x.x), "f"(-127.f));
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(b) : "f"(x.y), "f"(-127.f));
    const float2 xc = make_float2(a, b);
    const float2 t = __fadd2_rn(xc, make_float2(12582912.f, 12582912.f));
    const float2 n = __fadd2_rn(t, make_float2(-12582912.f, -12582912.f));
    const float2 f = __ffma2_rn(n, make_float2(-1.f, -1.f), xc);
    float2 p = __ffma2_rn(f, make_float2(C4, C4), make_float2(C3, C3));
    p = __ffma2_rn(p, f, make_float2(C2, C2));
    p = __ffma2_rn(p, f, make_float2(C1, C1));
    p = __ffma2_rn(p, f, make_float2(C0, C0));
    const float2 two_n = make_float2(__int_as_float((__float_as_int(t.x) << 23) + 0x3F800000),
                                     __int_as_float((__float_as_int(t.y) << 23) + 0x3F800000));
    return __fmul2_rn(p, two_n);
}
__device__ __forceinline__ float max3(float x, float y, float z) {
    float m;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(m) : "f"(x), "f"(y), "f"(z));
    return m;
}
__device__ __forceinline__ bool odd_half(uint32_t bits) { return (bits & 0x7C00u) == 0x7C00u; }

// What a stored row lacks (rare, and out of line: the mere code of it cost instruction fetches in
// the hot loop; 512 prompts of 300 tokens, 9/3 heads of 64: 290 us inline, 272 without, when it was
// taken out).  The
// non-finite values that the scrub took out of V (`vg`: column 0 of the KV head) are added to a row
// that sees keys first .. row.  A row without a key (`none`: every score -inf) becomes zeros, since
// the product made NaN of 0 * inf in the tiles that were not scrubbed.
__device__ __noinline__ void finish_row(const __half* vg, int64_t kv_stride, void* out, int out_f32,
                                        int head_dim, int first, int row, bool any_several,
                                        int tile0, int tile1, int unit_first, bool none) {
    if (none) {
        for (int i = 0; i < head_dim; ++i) {
            if (out_f32) static_cast<float*>(out)[i] = 0.f;
            else static_cast<__half*>(out)[i] = __half(0.f);
        }
        return;
    }
    for (int key = first; key <= row; ++key) {
        const int t = key / 128;
        if (!(any_several || t == tile0 || t == tile1 || t * 128 < unit_first)) {
            key |= 127;  // a tile that was not scrubbed: to its end
            continue;
        }
        for (int i = 0; i < head_dim; ++i) {
            const __half hv = vg[key * kv_stride + i];
            if (!odd_half(__half_as_ushort(hv))) continue;
            if (out_f32) {
                static_cast<float*>(out)[i] += __half2float(hv);
            } else {
                __half* o = static_cast<__half*>(out) + i;
                *o = __float2half(__half2float(*o) + __half2float(hv));
            }
        }
    }
}

template <int DP, int KS>
__global__ void __launch_bounds__(kTcThreads, 1)
    prompt_tc_kernel(const __grid_constant__ CUtensorMap qmap,
                     const __grid_constant__ CUtensorMap kmap,
                     const __grid_constant__ CUtensorMap vmap, const PromptArgs a, int tile0) {
    using Cfg = AttCfg<DP, KS>;
    using B = AttBar<DP, KS>;
    constexpr int SPT = Cfg::SPT;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    const uint32_t sbase = smem_u32(smem);
    const int tid = threadIdx.x, lane = tid & 31;
    const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);  // uniform for the compiler too
    const uint32_t bars = sbase + Cfg::OFF_BAR;
    auto bar = [&](int i) { return bars + 8u * static_cast<uint32_t>(i); };
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + Cfg::OFF_BAR + B::COUNT * 8);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    // bit k % 32: the scrub took visible values out of the tiles of this CTA's unit k
    volatile uint32_t* odd_units = tmem_slot + 2;
    int* top_cost = reinterpret_cast<int*>(tmem_slot + 3);
    constexpr unsigned FULL = 0xffffffffu;

    if (tid == 0) {
        for (int i = 0; i < B::COUNT; ++i) {
            const bool group = (i >= B::F && i < B::O) || (i >= B::E && i < B::SB);
            const bool both = i == B::DONE || (i >= B::KE && i < B::KE + Cfg::STAGES);
            mbar_init(bar(i), group ? 128u : both ? 2u : 1u);
        }
        *abort_flag = 0;
        *odd_units = 0;
        *top_cost = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 9) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                         smem_u32(tmem_slot)),
                     "r"(512)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    // ---- the work list
    int32_t* tile_seq = reinterpret_cast<int32_t*>(smem + Cfg::OFF_SEQ);
    uint32_t* tile_first = reinterpret_cast<uint32_t*>(smem + Cfg::OFF_FIRST);
    int32_t* hist = reinterpret_cast<int32_t*>(smem + Cfg::OFF_HIST);
    uint16_t* list = reinterpret_cast<uint16_t*>(smem + Cfg::OFF_LIST);
    uint16_t* cost = reinterpret_cast<uint16_t*>(smem + Cfg::OFF_COST);
    AttSched sched{tile_seq, tile_first, list, 0, 0, tile0, 0, 0, 0, 0};
    {
        const int q0 = __ldg(a.q_start), q1 = __ldg(a.q_start + a.num_seqs);
        sched.row_lo = q0 > 0 ? q0 : 0;
        sched.row_hi = q1 < a.rows ? q1 : static_cast<int>(a.rows);
        const int span = a.pairs == 2 ? 2 : 1;  // row tiles of a list entry
        // live tiles of the window, relative to its first
        int ta = sched.row_lo / kTile - tile0, tb = (sched.row_hi + kTile - 1) / kTile - tile0;
        ta = ta > 0 ? ta : 0;
        tb = tb < kWindow ? tb : kWindow;
        sched.tile_end = tb;
        const int ea = ta / span, eb = (tb + span - 1) / span;
        const int count = sched.row_hi > sched.row_lo && eb > ea ? eb - ea : 0;
        sched.per = a.kv_heads * (a.pairs == 1 ? a.group / 2 : a.group);
        sched.total = count * sched.per;
        const bool sorted = sched.total > static_cast<int>(gridDim.x);
        for (int i = tid; i < kWindow; i += kTcThreads) hist[i] = 0;
        for (int t = ta + tid; t < tb; t += kTcThreads) {
            const int row = (tile0 + t) * kTile;
            const int s = seq_at(a, row > sched.row_lo ? row : sched.row_lo, 0, a.num_seqs - 1);
            const int end = row + kTile < sched.row_hi ? row + kTile : sched.row_hi;
            tile_seq[t] = s;
            tile_first[t] = static_cast<uint32_t>(max(__ldg(a.q_start + s), 0)) |
                            (__ldg(a.q_start + s + 1) < end ? AttSched::kSeveral : 0u);
        }
        __syncthreads();
        if (!sorted) {
            for (int i = tid; i < count; i += kTcThreads) list[i] = static_cast<uint16_t>(ea + i);
        } else {
            int top = 0;
            for (int i = tid; i < count; i += kTcThreads) {
                const int t0 = max((ea + i) * span, ta), t1 = min((ea + i) * span + span, tb) - 1;
                const int first = static_cast<int>(tile_first[t0] & ~AttSched::kSeveral);
                const int c = tile0 + t1 - first / kTile;
                cost[i] = static_cast<uint16_t>(c < kWindow ? c : kWindow - 1);
                atomicAdd(hist + cost[i], 1);
                top = max(top, static_cast<int>(cost[i]));
            }
            __syncwarp();
            top = __reduce_max_sync(FULL, top);
            if (lane == 0 && top > 0) atomicMax(top_cost, top);
            __syncthreads();
            if (warp == 0) {
                int above = 0;  // entries of a higher cost
                for (int c0 = *top_cost; c0 >= 0; c0 -= 32) {
                    const int c = c0 - lane, own = c >= 0 ? hist[c] : 0;
                    int sum = own;
#pragma unroll
                    for (int o = 1; o < 32; o <<= 1) {
                        const int x = __shfl_up_sync(FULL, sum, o);
                        if (lane >= o) sum += x;
                    }
                    if (c >= 0) hist[c] = above + sum - own;
                    above += __shfl_sync(FULL, sum, 31);
                }
                __syncwarp();
                // in order within a cost, so every CTA has the same list
                for (int i0 = 0; i0 < count; i0 += 32) {
                    const int i = i0 + lane;
                    const int c = i < count ? cost[i] : -1;
                    const unsigned same = __match_any_sync(FULL, c);
                    const int before = __popc(same & ((1u << lane) - 1u));
                    const int at = c >= 0 ? hist[c] : 0;
                    __syncwarp();
                    if (c >= 0) {
                        list[at + before] = static_cast<uint16_t>(ea + i);
                        if (before == 0) hist[c] = at + __popc(same);
                    }
                    __syncwarp();
                }
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    auto tmem_s = [&](int i) { return tmem + static_cast<uint32_t>(KS * i); };
    auto tmem_p = [&](int i) { return tmem + static_cast<uint32_t>(2 * KS + KS / 2 * i); };
    auto tmem_o = [&](int i) { return tmem + static_cast<uint32_t>(512 - DP * (2 - i)); };
    auto wait = [&](int b, uint32_t parity) {
        return mbar_wait_bounded(bar(b), parity & 1u, abort_flag, &g_attention_status);
    };
    AttUnit u{};

    // A row of S takes 128 registers: the softmax groups get 200 each out of the launch's 168,
    // the others' warpgroup 96 (2 x 200 + 96 <= 3 x 168 in each quarter of the SM).
    if (warp < 8) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 200;");
        // ---- softmax: thread r of group w owns row r of item w
        const int w = warp >> 2, r = tid & 127;
        const uint32_t lane_base = static_cast<uint32_t>((warp & 3) * 32) << 16;
        const uint32_t ts = tmem_s(w) + lane_base, tp = tmem_p(w) + lane_base,
                       to = tmem_o(w) + lane_base;
        unsigned char* stage = smem + Cfg::OFF_OUT + warp * 2048;
        const uint32_t abort_addr = smem_u32(const_cast<int*>(abort_flag));
        int step = 0;
        auto await = [&](int b, int phase) {
            mbar_wait_uniform(bar(b), phase & 1, abort_addr, &g_attention_status);
        };
        const float2 sc2 = make_float2(a.scale_log2, a.scale_log2);
        struct Row {  // this thread's row of a unit: keys `first` .. row are visible
            int lo, hi, head, row, first;
            bool live;
        } x, y{};  // the current unit's and the next one's, found before the epilogue's wait
        auto next = [&]() {
            if (!sched.template next<Cfg::KS>(a, u)) return false;
            const int tile = w ? u.tile[1] : u.tile[0];
            y.lo = w ? u.lo[1] : u.lo[0], y.hi = w ? u.hi[1] : u.hi[0];
            y.head = w ? u.head[1] : u.head[0];
            y.row = tile * kTile + r;
            y.live = y.lo <= y.hi && y.row >= sched.row_lo && y.row < sched.row_hi;
            y.first = y.live ? sched.row_first(a, tile, y.row) : INT32_MAX;
            return true;
        };
        bool more = next();
        while (more && !*abort_flag) {
            x = y;
            const AttUnit now = u;
            const uint32_t unit_bit = 1u << ((sched.k - 1) & 31);
            const int lo = x.lo, hi = x.hi, row = x.row, first = x.first, head = x.head;
            const bool live = x.live;
            float m = -INFINITY, l = 0.f;
            for (int n = lo; n <= hi; ++n) {
                const bool ragged = now.ragged(n / SPT);
                await(B::S + w, step);
                tc_fence_after();
                float v[KS];
                tmem_ld_row(ts, v);
                tc_fence_before();
                mbar_arrive(bar(B::F + w));
                // of each 32 columns: every row of the warp sees all of them (mask without
                // work), none sees any (no exponentials either), or something between
                uint32_t dark = 0;  // bit c: 32 columns from 32 c on are dark
                if (ragged) {
                    // columns c_lo .. c_hi of this row are visible
                    const int c_lo = live ? first - n * KS : KS;
                    const int c_hi = live ? row - n * KS : -1;
                    const int some_lo = __reduce_min_sync(FULL, c_lo);
                    const int some_hi = __reduce_max_sync(FULL, c_hi);
                    const int all_lo = __reduce_max_sync(FULL, c_lo);
                    const int all_hi = __reduce_min_sync(FULL, c_hi);
#pragma unroll
                    for (int c = 0; c < KS / 32; ++c) {
                        if (c * 32 > some_hi || c * 32 + 31 < some_lo) dark |= 1u << c;
                        if (c * 32 < all_lo || c * 32 + 31 > all_hi) {
                            auto below = [](int x) {  // bits 0 .. x - 1
                                return x <= 0 ? 0u : x >= 32 ? ~0u : (1u << x) - 1u;
                            };
                            const uint32_t see = below(c_hi + 1 - c * 32) & ~below(c_lo - c * 32);
#pragma unroll
                            for (int i = 0; i < 32; ++i)
                                v[c * 32 + i] = (see & (1u << i)) ? v[c * 32 + i] : -INFINITY;
                        }
                    }
                }
                float mx[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
                for (int i = 4; i < KS - 4; i += 8)
#pragma unroll
                    for (int e = 0; e < 4; ++e) mx[e] = max3(mx[e], v[i + e], v[i + 4 + e]);
                const float mt = fmaxf(max3(mx[0], mx[1], fmaxf(v[KS - 4], v[KS - 3])),
                                       max3(mx[2], mx[3], fmaxf(v[KS - 2], v[KS - 1]))) *
                                 a.scale_log2;
                // The running maximum m follows only when a row's grew by more than 2^8 (then O and
                // l are rescaled); else P stays below 2^8 and 1 / l makes up for it.  A row's first
                // visible step (m = -inf: its l and O are zero) takes its maximum.
                float alpha = 1.f;
                const bool fresh = m == -INFINITY, grow = mt > m + 8.f;
                if (grow) {
                    if (!fresh) {
                        alpha = exp2_approx(m - mt);
                        l *= alpha;
                    }
                    m = mt;
                }
                const bool rescale = __any_sync(FULL, grow && !fresh);
                // P goes to F16 (the MMA's A operand has V's type): 2^-11 of each probability, as
                // much as the output's own rounding; kept to 11 bits it lies in tensor memory at
                // half the columns.  The sum l takes the unrounded ones and stays in F32.
                // -inf (nothing visible yet): exp2(-inf - 0) = 0
                const float sub = m == -INFINITY ? 0.f : -m;
                const float2 sub2 = make_float2(sub, sub);
                float2 l2[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
                for (int c = 0; c < KS / 32; ++c) {
                    uint32_t pk[16];
                    // 32 columns no row of the warp sees: zeros without exponentials
                    if (!(dark >> c & 1u)) {
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            const int i = c * 32 + 2 * e;
                            const float2 x = __ffma2_rn(make_float2(v[i], v[i + 1]), sc2, sub2);
                            const float2 p = (e & 3) == 2
                                                 ? exp2_fma(x)
                                                 : make_float2(exp2_approx(x.x), exp2_approx(x.y));
                            l2[e & 1] = __fadd2_rn(l2[e & 1], p);
                            pk[e] = pack_half2(p.x, p.y);
                        }
                    } else {
#pragma unroll
                        for (int e = 0; e < 16; ++e) pk[e] = 0u;
                    }
                    if (c == 0 && step > 0) {  // the last product has read P
                        await(B::O + w, step - 1);
                        tc_fence_after();
                    }
                    tmem_st16_bits(tp + 16 * c, pk);
                }
                l += (l2[0].x + l2[0].y) + (l2[1].x + l2[1].y);
                if (rescale) {  // O is to hold the products before this step
#pragma unroll 1
                    for (int c = 0; c < DP / 32; ++c) {
                        float o[32];
                        tmem_ld32(to + c * 32, o);
#pragma unroll
                        for (int i = 0; i < 32; ++i) o[i] *= alpha;
                        tmem_st32(to + c * 32, o);
                    }
                }
                tmem_wait_st();
                tc_fence_before();
                mbar_arrive(bar(B::P + w));
                ++step;
            }
            more = next();  // while the last product runs
            if (lo > hi) continue;
            // ---- epilogue
            await(B::O + w, step - 1);
            tc_fence_after();
            const bool none = l == 0.f;  // every score -inf
            const float inv = none ? 0.f : 1.f / l;
            const int64_t orow = (live ? row : 0) * a.out_stride +
                                 static_cast<int64_t>(head) * a.head_dim;
#pragma unroll 1
            for (int c = 0; c < DP / 32; ++c) {
                if (c * 32 >= a.head_dim) break;
                float o[32];
                tmem_ld32(to + c * 32, o);
#pragma unroll
                for (int i = 0; i < 32; ++i) o[i] *= inv;
                if (a.out_f32) {
                    if (!live) continue;
#pragma unroll
                    for (int i = 0; i < 32; i += 8) {
                        if (c * 32 + i >= a.head_dim) break;
                        float4* dst = reinterpret_cast<float4*>(static_cast<float*>(a.out) + orow +
                                                                c * 32 + i);
                        dst[0] = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
                        dst[1] = make_float4(o[i + 4], o[i + 5], o[i + 6], o[i + 7]);
                    }
                    continue;
                }
                // through shared memory, so that four lanes write a row's 64 bytes together
                // (straight from the registers every store would touch 32 rows)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    *reinterpret_cast<uint4*>(stage + lane * 64 + ((i ^ (lane >> 1 & 3)) << 4)) =
                        make_uint4(pack_half2(o[8 * i], o[8 * i + 1]),
                                   pack_half2(o[8 * i + 2], o[8 * i + 3]),
                                   pack_half2(o[8 * i + 4], o[8 * i + 5]),
                                   pack_half2(o[8 * i + 6], o[8 * i + 7]));
                __syncwarp();
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int sr = i * 8 + (lane >> 2), sc = lane & 3;  // row and 16-byte chunk
                    const int srow = row - lane + sr;
                    const uint4 x = *reinterpret_cast<const uint4*>(
                        stage + sr * 64 + ((sc ^ (sr >> 1 & 3)) << 4));
                    if (srow >= sched.row_lo && srow < sched.row_hi &&
                        c * 32 + sc * 8 < a.head_dim)
                        *reinterpret_cast<uint4*>(static_cast<__half*>(a.out) +
                                                  srow * a.out_stride +
                                                  static_cast<int64_t>(head) * a.head_dim + c * 32 +
                                                  sc * 8) = x;
                }
                __syncwarp();
            }
            tc_fence_before();
            mbar_arrive(bar(B::E + w));
            if (a.lse && live)
                a.lse[static_cast<int64_t>(row) * a.q_heads + head] =
                    ((m == -INFINITY ? 0.f : m) + log2f(l)) * kLn2;
            if (__any_sync(FULL, live && (none || (*odd_units & unit_bit)))) {
                // (rows were stored by any lane: the vote and the barriers before it order that)
                if (live)
                    finish_row(static_cast<const __half*>(a.v) +
                                   static_cast<int64_t>(now.kvh) * a.head_dim,
                               a.kv_stride,
                               static_cast<unsigned char*>(a.out) + orow * (a.out_f32 ? 4 : 2),
                               a.out_f32, a.head_dim, first, row, now.any_several, now.tile[0],
                               now.tile[1], now.first, none);
                __syncwarp();
            }
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 96;");
        if (warp == 8 && lane == 0) {
            constexpr int NB = DP / 64;
            int ring = 0, cnt[2] = {0, 0};
            bool ok = true;
            auto load_q = [&](int i) {
                const int qb = cnt[i] % Cfg::QBUF, round = cnt[i] / Cfg::QBUF;
                const int b = qb * 2 + i;
                if (round > 0) ok = wait(B::QE + b, round - 1);
                if (!ok) return;
                ++cnt[i];
                mbar_arrive_tx(bar(B::QF + b), static_cast<uint32_t>(Cfg::TILE));
                for (int c = 0; c < NB; ++c)
                    tma_load_3d(sbase + b * Cfg::TILE + c * Cfg::BLK, &qmap, c * 64, u.head[i],
                                u.tile[i] * kTile, bar(B::QF + b));
            };
            auto load_kv = [&](const CUtensorMap* map, int j) {
                const int st = ring % Cfg::STAGES, round = ring / Cfg::STAGES;
                if (round > 0) ok = wait(B::KE + st, round - 1);
                if (!ok) return;
                ++ring;
                mbar_arrive_tx(bar(B::KF + st), static_cast<uint32_t>(Cfg::TILE));
                for (int c = 0; c < NB; ++c)
                    tma_load_3d(sbase + Cfg::OFF_KV + st * Cfg::TILE + c * Cfg::BLK, map, c * 64,
                                u.kvh, j * kTile, bar(B::KF + st));
            };
            while (ok && sched.template next<Cfg::KS>(a, u)) {
                for (int j = u.jlo; ok && j <= u.jhi; ++j) {
                    if (u.on(0) && j == u.lo[0] / SPT) load_q(0);
                    if (ok) load_kv(&kmap, j);
                    if (ok && u.on(1) && j == u.lo[1] / SPT) load_q(1);
                    if (ok) load_kv(&vmap, j);
                }
            }
            // every copy has landed before the CTA gives its memory back, also when this warp got
            // through and another one gave up
            for (int i = ring < Cfg::STAGES ? 0 : ring - Cfg::STAGES; i < ring; ++i)
                mbar_drain(bar(B::KF + i % Cfg::STAGES), (i / Cfg::STAGES) & 1);
            for (int i = 0; i < 2; ++i)
                for (int n = cnt[i] < Cfg::QBUF ? 0 : cnt[i] - Cfg::QBUF; n < cnt[i]; ++n)
                    mbar_drain(bar(B::QF + (n % Cfg::QBUF) * 2 + i), (n / Cfg::QBUF) & 1);
        } else if (warp == 9 || warp == 10) {
            // One MMA warp an item: while one waits for its softmax group the other one's
            // products run.  The whole warp walks this code and one elected lane issues: with
            // uniform control flow the descriptors stay in uniform registers (issued from a
            // divergent lane, an MMA took about 100 cycles, against 32 to 64 to execute).
            constexpr uint32_t IDESC_QK = f16_idesc(128, KS, false);
            constexpr uint32_t IDESC_PV = f16_idesc(128, DP, true);
            const int i = warp - 9;
            const bool leader = elect_one();
            const int ksteps = (a.head_dim + 15) / 16;
            const uint32_t abort_addr = smem_u32(const_cast<int*>(abort_flag));
            int ring0 = 0, units = 0, scores = 0, prods = 0;
            auto await = [&](int b, int phase) {
                mbar_wait_uniform(bar(b), phase & 1, abort_addr, &g_attention_status);
            };
            auto stage_of = [&](int x) { return x % Cfg::STAGES; };
            auto await_full = [&](int x) { await(B::KF + stage_of(x), x / Cfg::STAGES); };
            int lo = 0, hi = 0;  // this item's steps
            // S = Q K^T of step n, if the item has it, over scores that were read.  Every K tile is
            // given back once, by both warps.
            auto qk = [&](int n) {
                const int sub = n % SPT;
                const int x = ring0 + 2 * (n / SPT - u.jlo), qb = units % Cfg::QBUF;
                const bool mine = n >= lo && n <= hi;
                if (sub == 0) await_full(x);  // each tile, to stay in step with the other warp
                if (mine) {
                    if (n == lo) await(B::QF + qb * 2 + i, units / Cfg::QBUF);
                    if (scores > 0) await(B::F + i, scores - 1);
                    tc_fence_after();
                }
                const uint32_t qa = sbase + (qb * 2 + i) * Cfg::TILE;
                const uint32_t ka = sbase + Cfg::OFF_KV + stage_of(x) * Cfg::TILE + sub * KS * 128;
                const uint64_t qd = sw128_desc(qa, 16, 1024), kd = sw128_desc(ka, 16, 1024);
                const uint32_t d = tmem_s(i);
                if (leader) {
                    if (mine) {
#pragma unroll
                        for (int kk = 0; kk < DP / 16; ++kk) {
                            const uint32_t off = ((kk >> 2) * Cfg::BLK + (kk & 3) * 32) >> 4;
                            if (kk < ksteps) tc_mma(d, qd + off, kd + off, IDESC_QK, kk > 0);
                        }
                        tc_commit(bar(B::S + i));
                        if (n == hi) tc_commit(bar(B::QE + qb * 2 + i));
                    }
                    if (sub == SPT - 1) tc_commit(bar(B::KE + stage_of(x)));
                }
                __syncwarp();
                if (mine) ++scores;
            };
            auto pv = [&](int n) {
                const int sub = n % SPT;
                const int x = ring0 + 2 * (n / SPT - u.jlo) + 1;
                const bool mine = n >= lo && n <= hi;
                if (sub == 0) await(B::SB + stage_of(x), x / Cfg::STAGES);
                if (mine) {
                    await(B::P + i, prods);
                    // the accumulator still holds this item's previous unit
                    if (n == lo && units > 0) await(B::E + i, units - 1);
                    tc_fence_after();
                }
                const uint32_t va = sbase + Cfg::OFF_KV + stage_of(x) * Cfg::TILE + sub * KS * 128;
                const uint64_t vd = sw128_desc(va, Cfg::BLK, 1024);
                const uint32_t d = tmem_o(i), p = tmem_p(i);
                if (leader) {
                    if (mine) {
#pragma unroll
                        for (int kk = 0; kk < KS / 16; ++kk)
                            tc_mma_ts(d, p + 8u * kk, vd + kk * (2048 >> 4), IDESC_PV,
                                      n > lo || kk > 0);
                        tc_commit(bar(B::O + i));
                    }
                    if (sub == SPT - 1) tc_commit(bar(B::KE + stage_of(x)));
                }
                __syncwarp();
                if (mine) ++prods;
            };
            while (sched.template next<Cfg::KS>(a, u) && !*abort_flag) {
                u.make_uniform();
                lo = i ? u.lo[1] : u.lo[0];
                hi = i ? u.hi[1] : u.hi[0];
                const int n0 = u.jlo * SPT, n1 = u.jhi * SPT + SPT - 1;
                qk(n0);
                for (int n = n0; n <= n1; ++n) {
                    if (n < n1) qk(n + 1);
                    pv(n);
                }
                ring0 += 2 * (u.jhi - u.jlo + 1);
                if (lo <= hi) ++units;
            }
            __syncwarp();
            if (leader) {  // every product is done before the CTA frees its memory
                tc_commit(bar(B::DONE));
                mbar_drain(bar(B::DONE), 0);
            }
        } else if (warp == 11) {
            // ---- scrub: a V tile that some row of the unit does not see whole loses its
            // non-finite entries (and the unit's bit says that a sequence's key had some) before
            // the products read it, while the softmax groups are at its scores
            const uint32_t abort_addr = smem_u32(const_cast<int*>(abort_flag));
            int x = 1;  // ring index of the V tile
            while (sched.template next<Cfg::KS>(a, u) && !*abort_flag) {
                for (int j = u.jlo; j <= u.jhi; ++j, x += 2) {
                    const int st = x % Cfg::STAGES;
                    mbar_wait_uniform(bar(B::KF + st), (x / Cfg::STAGES) & 1, abort_addr,
                                      &g_attention_status);
                    if (u.ragged(j)) {
                        unsigned char* v = smem + Cfg::OFF_KV + st * Cfg::TILE + lane * 16;
                        __half2 probe[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) probe[e] = __floats2half2_rn(0.f, 0.f);
                        const __half2 zero = probe[0];
#pragma unroll 8
                        for (int c = 0; c < Cfg::TILE / 512; ++c) {
                            const uint4 y = *reinterpret_cast<const uint4*>(v + 512 * c);
                            const __half2* h = reinterpret_cast<const __half2*>(&y);
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                probe[e] = __hfma2(h[e], zero, probe[e]);  // 0 or NaN
                        }
                        const __half2 sum = __hadd2(__hadd2(probe[0], probe[1]),
                                                    __hadd2(probe[2], probe[3]));
                        if (!(__low2float(sum) == 0.f && __high2float(sum) == 0.f)) {
                            bool any = false;
                            for (int c = 0; c < Cfg::TILE / 512; ++c) {
                                uint16_t* b = reinterpret_cast<uint16_t*>(v + 512 * c);
                                // 16 bytes a lane of rows of 128, 128 rows a block of columns
                                const int key = j * kTile + (lane / 8 + 4 * c) % kTile;
                                for (int e = 0; e < 8; ++e) {
                                    if (!odd_half(b[e])) continue;
                                    b[e] = 0;
                                    any |= key >= sched.row_lo && key < sched.row_hi;
                                }
                            }
                            if (any)
                                atomicOr(const_cast<uint32_t*>(odd_units),
                                         1u << ((sched.k - 1) & 31));
                            fence_async_smem();
                        }
                    }
                    __syncwarp();
                    if (lane == 0) mbar_arrive(bar(B::SB + st));
                    __syncwarp();
                }
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 9) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512)
                     : "memory");
    }
}

template <int DP, int KS>
int launch_tc(PromptArgs a, cudaStream_t s) {
    using Cfg = AttCfg<DP, KS>;
    CUtensorMap qmap, kmap, vmap;
    if (int st = make_map_heads(&qmap, a.q, a.head_dim, a.q_heads, a.rows, a.q_stride * 2, kTile))
        return st;
    if (int st = make_map_heads(&kmap, a.k, a.head_dim, a.kv_heads, a.rows, a.kv_stride * 2, kTile))
        return st;
    if (int st = make_map_heads(&vmap, a.v, a.head_dim, a.kv_heads, a.rows, a.kv_stride * 2, kTile))
        return st;
    static std::atomic<uint64_t> opted{0};
    int dev = 0;
    TMLLM_CUDA_TRY(cudaGetDevice(&dev));
    const uint64_t bit = dev < 64 ? (1ull << dev) : 0;
    if (!bit || !(opted.load(std::memory_order_relaxed) & bit)) {
        TMLLM_CUDA_TRY(cudaFuncSetAttribute(prompt_tc_kernel<DP, KS>,
                                            cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::SMEM));
        opted.fetch_or(bit, std::memory_order_relaxed);
    }
    const int sms = device_sm_count();
    const int64_t tiles = (a.rows + kTile - 1) / kTile;
    for (int64_t t0 = 0; t0 < tiles; t0 += kWindow) {
        const int64_t n = tiles - t0 < kWindow ? tiles - t0 : kWindow;
        const int64_t items = n * a.q_heads;
        if (items > INT32_MAX) return fail(TMLLM_INVALID_SHAPE, "too many prompt tiles");
        // one item a unit while that still leaves SMs idle
        a.pairs = items <= sms ? 0 : a.group % 2 == 0 ? 1 : 2;
        const int64_t ctas = items < sms ? items : sms;
        prompt_tc_kernel<DP, KS><<<static_cast<unsigned>(ctas), kTcThreads, Cfg::SMEM, s>>>(
            qmap, kmap, vmap, a, static_cast<int>(t0));
        TMLLM_LAUNCH_TRY();
    }
    return TMLLM_OK;
}

}  // namespace
}  // namespace tmllm

using namespace tmllm;

namespace tmllm {
int take_linear_wait_status(int* out);  // prompt_linear.cu
}

extern "C" {

int tmllm_prompt_status(int32_t* status) {
    clear_error();
    if (!status) return fail(TMLLM_INVALID_ARGUMENT, "null status pointer");
    int linear = 0, attention = 0;
    if (int st = take_linear_wait_status(&linear)) return st;
    if (int st = take_status(g_attention_status, &attention)) return st;
    *status = linear ? linear : attention;
    return TMLLM_OK;
}

int tmllm_prompt_attention(tmllm_dtype dtype, const void* q, int64_t q_stride, const void* k,
                           const void* v, int64_t kv_stride, const int32_t* q_start,
                           int32_t num_seqs, int64_t rows, int32_t max_rows, int32_t q_heads,
                           int32_t kv_heads, int32_t head_dim, float scale, void* out,
                           int32_t out_f32, float* lse, tmllm_stream stream) {
    clear_error();
    if (!valid_dtype(dtype)) return fail(TMLLM_UNSUPPORTED_DTYPE, "unknown dtype");
    if (num_seqs <= 0 || q_heads <= 0 || kv_heads <= 0 || head_dim <= 0)
        return fail(TMLLM_INVALID_SHAPE, "prompt attention dimensions must be positive");
    if (head_dim > 256)
        return fail(TMLLM_INVALID_SHAPE, "head_dim must be <= 256, got %d", head_dim);
    if (q_heads % kv_heads != 0)
        return fail(TMLLM_MODEL_FORMAT, "Q heads %d must be divisible by non-zero KV heads %d",
                    q_heads, kv_heads);
    if (rows < 0 || rows > INT32_MAX - 1024 || max_rows < 0)
        return fail(TMLLM_INVALID_SHAPE, "row counts must be non-negative and fit 31 bits");
    if (out_f32 != 0 && out_f32 != 1)
        return fail(TMLLM_INVALID_ARGUMENT, "out_f32 must be 0 or 1");
    if (rows == 0 || max_rows == 0) return TMLLM_OK;
    if (max_rows > rows) max_rows = static_cast<int32_t>(rows);
    const float sc = scale > 0.f ? scale : 1.0f / sqrtf(static_cast<float>(head_dim));
    if (!std::isfinite(sc * kLog2e) || std::isnan(scale))  // (scores are kept as powers of two)
        return fail(TMLLM_INVALID_SHAPE, "attention scale must be positive and finite");
    const int64_t qw = static_cast<int64_t>(q_heads) * head_dim;
    const int64_t kw = static_cast<int64_t>(kv_heads) * head_dim;
    if (!q_stride) q_stride = qw;
    if (!kv_stride) kv_stride = kw;
    int64_t span;
    if (q_stride < qw || kv_stride < kw)
        return fail(TMLLM_INVALID_SHAPE, "row strides of q / k / v must cover a row");
    for (int64_t stride : {q_stride, kv_stride})
        if (!mul_ok(rows, stride, &span) || span > INT64_MAX / 8)
            return fail(TMLLM_INVALID_SHAPE, "rows and row strides must fit 60 bits");
    if (!q || !k || !v || !q_start || !out)
        return fail(TMLLM_INVALID_ARGUMENT, "null tensor pointer");
    const size_t es = dtype_size(dtype);
    const size_t os = (out_f32 || dtype == TMLLM_F32) ? 4 : 2;
    for (const void* p : {q, k, v})
        if (reinterpret_cast<uintptr_t>(p) % es)
            return fail(TMLLM_INVALID_ARGUMENT,
                        "tensor pointers must be aligned to their element size");
    if (reinterpret_cast<uintptr_t>(out) % os || reinterpret_cast<uintptr_t>(lse) % 4)
        return fail(TMLLM_INVALID_ARGUMENT,
                    "tensor pointers must be aligned to their element size");
    // a tile's q rows are read before its out rows are written, by the same CTA; k and v are
    // read by others too
    const int64_t ow = qw * static_cast<int64_t>(os / es);  // in elements of es bytes
    const Rows ro{out, ow, ow};
    if (out == q && q_stride == qw && os == es) {
    } else if (overlaps(ro, {q, q_stride, qw}, rows, es)) {
        return fail(TMLLM_INVALID_ARGUMENT, "out may be q itself, but not overlap it");
    }
    if (overlaps(ro, {k, kv_stride, kw}, rows, es) || overlaps(ro, {v, kv_stride, kw}, rows, es))
        return fail(TMLLM_INVALID_ARGUMENT, "out overlaps k or v");
    const Span sums{lse, 4 * rows * q_heads}, starts{q_start, 4 * (int64_t{1} + num_seqs)};
    for (const Rows& r : {Rows{q, q_stride, qw}, Rows{k, kv_stride, kw}, Rows{v, kv_stride, kw}, ro})
        if (inside(sums.p, sums.bytes, r, rows, es))
            return fail(TMLLM_INVALID_ARGUMENT, "lse overlaps q, k, v or out");
    if (inside(starts.p, starts.bytes, ro, rows, es) || overlaps(starts, sums))
        return fail(TMLLM_INVALID_ARGUMENT, "out or lse overlaps q_start");
    PromptArgs a{};
    a.q = q;
    a.k = k;
    a.v = v;
    a.out = out;
    a.lse = lse;
    a.q_start = q_start;
    a.rows = rows;
    a.q_stride = q_stride;
    a.kv_stride = kv_stride;
    a.out_stride = qw;
    a.num_seqs = num_seqs;
    a.max_rows = max_rows;
    a.q_heads = q_heads;
    a.kv_heads = kv_heads;
    a.group = q_heads / kv_heads;
    a.head_dim = head_dim;
    a.out_f32 = out_f32 || dtype == TMLLM_F32;
    a.scale_log2 = sc * kLog2e;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    if (dtype == TMLLM_F32) return launch_fma_d<float>(a, s);
    const bool tc = head_dim % 8 == 0 && head_dim <= 128 && q_stride % 8 == 0 &&
                    kv_stride % 8 == 0 && aligned16(q) && aligned16(k) && aligned16(v) &&
                    aligned16(out) && q_stride < (int64_t{1} << 38) && kv_stride < (int64_t{1} << 38);
    if (!tc) return launch_fma_d<__half>(a, s);
    if (head_dim > 64) return launch_tc<128, 64>(a, s);
    // (see KS at the kernel; 32 prompts of 1024 tokens of 15/5 heads of 64: 130 us in steps of 128,
    // 133 of 64; 64 of 1 to 1500 tokens 200 and 186)
    if (rows < 1024 * static_cast<int64_t>(num_seqs)) return launch_tc<64, 64>(a, s);
    return launch_tc<64, 128>(a, s);
}

}  // extern "C"
