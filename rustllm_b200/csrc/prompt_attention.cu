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
    int32_t pairs;  // tensor-core form: two 128-row items a unit, or one
    float scale_log2;
};

__device__ int g_attention_status;

// First row and row count of sequence s, clipped to the packed rows that exist.
__device__ __forceinline__ int seq_rows(const PromptArgs& a, int s, int64_t* row0) {
    int64_t lo = a.q_start[s], hi = a.q_start[s + 1];
    if (hi > a.rows) hi = a.rows;
    if (lo < 0 || lo >= hi) return 0;
    *row0 = lo;
    const int64_t n = hi - lo;
    return static_cast<int>(n < a.max_rows ? n : a.max_rows);
}

// ---- CUDA-core form: any type and head size up to 256 -----------------------------------
// One CTA per (64 query rows, query head, sequence), 256 threads; thread (ty, tx) holds rows
// 4 ty .. 4 ty + 3 of S (columns tx + 16 c) and of O (columns tx + 16 c).  DP: head size
// rounded up to 64 / 128 / 256.
constexpr int kFmaTile = 64;

template <typename T, int DP>
__global__ void __launch_bounds__(256) prompt_fma_kernel(const PromptArgs a, int row_tiles) {
    constexpr int LD = DP + 1;  // odd pitch: column walks hit every bank
    extern __shared__ float fsm[];
    float* qs = fsm;                       // [64][LD]
    float* ks = qs + kFmaTile * LD;        // [64][LD]
    float* vs = ks + kFmaTile * LD;        // [64][DP]
    float* ps = vs + kFmaTile * DP;        // [64][65]
    const int64_t hb = static_cast<int64_t>(a.q_heads) * a.num_seqs;
    const int tile = row_tiles - 1 - static_cast<int>(blockIdx.x / hb);
    const int h = static_cast<int>(blockIdx.x % hb) % a.q_heads;
    const int s = static_cast<int>(blockIdx.x % hb) / a.q_heads;
    int64_t row0 = 0;
    const int n = seq_rows(a, s, &row0);
    const int q_lo = tile * kFmaTile;
    if (q_lo >= n) return;
    const int kvh = h / a.group, D = a.head_dim;
    const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
    const T* qg = static_cast<const T*>(a.q) + (row0 + q_lo) * a.q_stride +
                  static_cast<int64_t>(h) * D;
    const T* kg = static_cast<const T*>(a.k) + row0 * a.kv_stride + static_cast<int64_t>(kvh) * D;
    const T* vg = static_cast<const T*>(a.v) + row0 * a.kv_stride + static_cast<int64_t>(kvh) * D;
    for (int i = tid; i < kFmaTile * DP; i += 256) {
        const int r = i / DP, c = i % DP;
        qs[r * LD + c] = (q_lo + r < n && c < D) ? to_f32<T>(qg[r * a.q_stride + c]) : 0.f;
    }
    float o[4][DP / 16], m[4], l[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        m[i] = -INFINITY;
        l[i] = 0.f;
#pragma unroll
        for (int c = 0; c < DP / 16; ++c) o[i][c] = 0.f;
    }
    const int q_hi = q_lo + kFmaTile < n ? q_lo + kFmaTile : n;  // keys [0, q_hi) are visible
    for (int j0 = 0; j0 < q_hi; j0 += kFmaTile) {
        __syncthreads();
        for (int i = tid; i < kFmaTile * DP; i += 256) {
            const int r = i / DP, c = i % DP;
            const bool in = j0 + r < q_hi && c < D;
            const int64_t off = static_cast<int64_t>(j0 + r) * a.kv_stride + c;
            ks[r * LD + c] = in ? to_f32<T>(kg[off]) : 0.f;
            vs[r * DP + c] = in ? to_f32<T>(vg[off]) : 0.f;
        }
        __syncthreads();
        float sc[4][4] = {};
        for (int d = 0; d < D; ++d) {
            float qv[4], kv[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) qv[i] = qs[(4 * ty + i) * LD + d];
#pragma unroll
            for (int c = 0; c < 4; ++c) kv[c] = ks[(tx + 16 * c) * LD + d];
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int c = 0; c < 4; ++c) sc[i][c] = fmaf(qv[i], kv[c], sc[i][c]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int qi = q_lo + 4 * ty + i;
            float mt = -INFINITY;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                sc[i][c] = j0 + tx + 16 * c <= qi ? sc[i][c] * a.scale_log2 : -INFINITY;
                mt = fmaxf(mt, sc[i][c]);
            }
#pragma unroll
            for (int w = 8; w > 0; w >>= 1) mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, w));
            const float mn = fmaxf(m[i], mt);
            const float base = mn == -INFINITY ? 0.f : mn;  // nothing visible yet: exp2(-inf)
            const float corr = exp2f(m[i] - base);
            float ls = 0.f;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const float p = exp2f(sc[i][c] - base);
                ps[(4 * ty + i) * 65 + tx + 16 * c] = p;
                ls += p;
            }
#pragma unroll
            for (int w = 8; w > 0; w >>= 1) ls += __shfl_xor_sync(0xffffffffu, ls, w);
            l[i] = l[i] * corr + ls;
            m[i] = mn;
#pragma unroll
            for (int c = 0; c < DP / 16; ++c) o[i][c] *= corr;
        }
        __syncwarp();  // the rows of ps a warp reads are the ones its own lanes wrote
        const int nk = q_hi - j0 < kFmaTile ? q_hi - j0 : kFmaTile;
        const bool diag = j0 + nk - 1 > q_lo;
        for (int j = 0; j < nk; ++j) {
            float pv[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) pv[i] = ps[(4 * ty + i) * 65 + j];
#pragma unroll
            for (int c = 0; c < DP / 16; ++c) {
                const float vv = vs[j * DP + tx + 16 * c];
#pragma unroll
                for (int i = 0; i < 4; ++i)  // a masked value must not reach a sum (0 * inf)
                    if (!diag || j0 + j <= q_lo + 4 * ty + i) o[i][c] = fmaf(pv[i], vv, o[i][c]);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = q_lo + 4 * ty + i;
        if (r >= n) continue;
        const float inv = l[i] == 0.f ? 0.f : 1.f / l[i];  // every score -inf: zeros
        const int64_t off = (row0 + r) * a.out_stride + static_cast<int64_t>(h) * D;
#pragma unroll
        for (int c = 0; c < DP / 16; ++c) {
            const int d = tx + 16 * c;
            if (d >= D) continue;
            if (a.out_f32) static_cast<float*>(a.out)[off + d] = o[i][c] * inv;
            else static_cast<T*>(a.out)[off + d] = from_f32<T>(o[i][c] * inv);
        }
        if (a.lse && tx == 0)
            a.lse[(row0 + r) * a.q_heads + h] = (m[i] + log2f(l[i])) * kLn2;
    }
}

template <typename T, int DP>
int launch_fma(const PromptArgs& a, cudaStream_t s) {
    const int row_tiles = (a.max_rows + kFmaTile - 1) / kFmaTile;
    int64_t ctas;
    if (!mul_ok(static_cast<int64_t>(row_tiles) * a.q_heads, a.num_seqs, &ctas) ||
        ctas > INT32_MAX)
        return fail(TMLLM_INVALID_SHAPE, "too many prompt tiles");
    constexpr int smem = (2 * kFmaTile * (DP + 1) + kFmaTile * DP + kFmaTile * 65) * 4;
    TMLLM_CUDA_TRY(cudaFuncSetAttribute(prompt_fma_kernel<T, DP>,
                                        cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    prompt_fma_kernel<T, DP><<<static_cast<unsigned>(ctas), 256, smem, s>>>(a, row_tiles);
    TMLLM_LAUNCH_TRY();
    return TMLLM_OK;
}

template <typename T>
int launch_fma_d(const PromptArgs& a, cudaStream_t s) {
    if (a.head_dim <= 64) return launch_fma<T, 64>(a, s);
    if (a.head_dim <= 128) return launch_fma<T, 128>(a, s);
    return launch_fma<T, 256>(a, s);
}


// ---- tensor-core form: F16, head size a multiple of 8 up to 128 -------------------------
// An item is 128 query rows of one (sequence, query head).  The items of a (sequence, KV head)
// are numbered row tile by row tile, heads of the group innermost; a unit is two neighbours, so
// the K and V tiles it streams serve two items (two heads of the group over the same rows, or
// two row tiles of one head when the group is one).  Per CTA:
//   warps 0-3, 4-7  softmax of item 0 / 1, one thread per query row
//   warp 8          TMA producer: Q tiles, then K and V tiles through a ring
//   warp 9          MMA issuer
// S = Q K^T sits in tensor memory; its row is read to registers, exponentiated, and P written
// back as F16 over the same columns, from where it is the A operand of O += P V (so only V
// crosses shared memory for the second product).  While one item is exponentiated the tensor
// cores work for the other one.
//   tensor memory: S_i / P_i at [128 i, 128 i + 128), O_i at [256 + DP i, ...)
//
// Masked places never reach a result: scores behind a row are replaced by -inf before the
// maximum, and since 0 * inf is not 0, V's non-finite entries in a unit's diagonal tiles are
// zeroed in shared memory before the product and added afterwards to the rows that see them.
constexpr int kTile = 128;
constexpr int kTcThreads = 384;  // warps 10 and 11 complete a warpgroup and idle
constexpr int kMaxSeqs = 1024;    // sequences a launch schedules
constexpr int kMaxLevels = 4096;  // row tiles of a sequence: prompts of up to 524,288 rows

template <int DP>
struct AttCfg {
    static constexpr int BLK = 16384;          // 64 columns x 128 rows, swizzled
    static constexpr int TILE = DP / 64 * BLK; // Q, K or V tile
    static constexpr int QBUF = DP == 64 ? 2 : 1;
    static constexpr int STAGES = DP == 64 ? 6 : 4;
    static constexpr int OFF_KV = 2 * QBUF * TILE;
    static constexpr int OFF_BASE = OFF_KV + STAGES * TILE;    // int32 units before each level
    static constexpr int OFF_ORDER = OFF_BASE + kMaxLevels * 4;  // uint16 sequences, longest first
    static constexpr int OFF_TILES = OFF_ORDER + kMaxSeqs * 2;  // int32 their row tiles
    static constexpr int OFF_BAR = OFF_TILES + kMaxSeqs * 4;
    static constexpr int SMEM = OFF_BAR + 512 + 1024;  // + alignment
    static_assert(SMEM <= 227 * 1024, "shared memory of one CTA");
};

// Barriers: QF/QE Q tile full / empty, KF/KE ring full / empty, S scores ready, P probabilities
// written, O product done, E accumulator read, VR diagonal V tile loaded, SB scrubbed, DONE all
// products.  VR and SB exist twice, for a unit's first and second diagonal tile ("events"): every
// unit passes the first one, and both softmax groups take part in each, so no thread ever falls
// more than a phase behind a barrier that it waits on.
template <int DP>
struct AttBar {
    using Cfg = AttCfg<DP>;
    static constexpr int QF = 0, QE = QF + 2 * Cfg::QBUF, KF = QE + 2 * Cfg::QBUF,
                         KE = KF + Cfg::STAGES, S = KE + Cfg::STAGES, P = S + 2, O = P + 2,
                         E = O + 2, VR = E + 2, SB = VR + 2, DONE = SB + 2, COUNT = DONE + 1;
    static_assert(COUNT * 8 + 64 <= 512, "barrier area");
};

struct AttUnit {
    int64_t row0;
    int n;           // rows of the sequence
    int kvh;
    int head[2], q_lo[2];
    int nt[2];       // key tiles of each item; 0: no such item
};

// The work list every role of every CTA walks in the same order: longest key range first, dealt
// to the CTAs in a snake, so their sums come out alike.  A level is a row tile index; levels
// are visited from the last to the first, the sequences that reach one in order of length.
struct AttSched {
    const int32_t* base;    // units in the levels above
    const uint16_t* order;
    int level, levels, total, k;

    __device__ __forceinline__ bool next(const PromptArgs& a, AttUnit& u) {
        for (;;) {
            const int G = gridDim.x;
            const int64_t at = (k & 1) ? static_cast<int64_t>(k + 1) * G - 1 - blockIdx.x
                                       : static_cast<int64_t>(k) * G + blockIdx.x;
            if (static_cast<int64_t>(k) * G >= total) return false;
            ++k;
            if (at >= total) continue;
            const int idx = static_cast<int>(at);
            while (level > 0 && idx >= base[level - 1]) --level;
            const int g = a.group, t = level;
            const int p0 = a.pairs ? (t * g + 1) / 2 : t * g;
            const int np = a.pairs ? ((t + 1) * g + 1) / 2 - p0 : g;
            int r = idx - base[t];
            const int p = p0 + r % np;
            r /= np;
            u.kvh = r % a.kv_heads;
            const int s = order[r / a.kv_heads];
            u.n = seq_rows(a, s, &u.row0);
            const int tiles = (u.n + kTile - 1) / kTile;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int item = a.pairs ? 2 * p + i : p;
                const int tile = item / g;
                const bool in = (i == 0 || a.pairs) && tile < tiles;
                u.head[i] = u.kvh * g + item % g;
                u.q_lo[i] = tile * kTile;
                u.nt[i] = in ? tile + 1 : 0;
            }
            return true;
        }
    }
};

__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ bool odd_half(uint32_t bits) { return (bits & 0x7C00u) == 0x7C00u; }

template <int DP>
__global__ void __launch_bounds__(kTcThreads, 1)
    prompt_tc_kernel(const __grid_constant__ CUtensorMap qmap,
                     const __grid_constant__ CUtensorMap kmap,
                     const __grid_constant__ CUtensorMap vmap, const PromptArgs a) {
    using Cfg = AttCfg<DP>;
    using B = AttBar<DP>;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    const uint32_t sbase = smem_u32(smem);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t bars = sbase + Cfg::OFF_BAR;
    auto bar = [&](int i) { return bars + 8u * static_cast<uint32_t>(i); };
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + Cfg::OFF_BAR + B::COUNT * 8);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    volatile int* odd_flag = reinterpret_cast<volatile int*>(tmem_slot + 2);  // [parity][event]
    int* scan = reinterpret_cast<int*>(tmem_slot + 6);  // one total
    constexpr unsigned FULL = 0xffffffffu;

    if (tid == 0) {
        for (int i = 0; i < B::COUNT; ++i) {
            const bool softmax = i >= B::P && i < B::P + 2;
            const bool epilogue = i >= B::E && i < B::E + 2;
            mbar_init(bar(i), i >= B::SB && i < B::SB + 2 ? 256u : (softmax || epilogue) ? 128u : 1u);
        }
        *abort_flag = 0;
        for (int i = 0; i < 4; ++i) odd_flag[i] = 0;
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
    int32_t* base = reinterpret_cast<int32_t*>(smem + Cfg::OFF_BASE);
    uint16_t* order = reinterpret_cast<uint16_t*>(smem + Cfg::OFF_ORDER);
    int32_t* tiles = reinterpret_cast<int32_t*>(smem + Cfg::OFF_TILES);
    int32_t* raw = base;  // unsorted row tiles, until the levels are written
    for (int s = tid; s < a.num_seqs; s += kTcThreads) {
        int64_t r0;
        raw[s] = (seq_rows(a, s, &r0) + kTile - 1) / kTile;
    }
    __syncthreads();
    for (int s = tid; s < a.num_seqs; s += kTcThreads) {
        const int mine = raw[s];
        int rank = 0;  // longer sequences, and equally long ones in front
        for (int o = 0; o < a.num_seqs; ++o) rank += raw[o] > mine || (raw[o] == mine && o < s);
        order[rank] = static_cast<uint16_t>(s);
        tiles[rank] = mine;
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    AttSched sched{base, order, 0, tiles[0], 0, 0};
    {
        // units of level t: the sequences with more than t tiles x KV heads x pairs starting in
        // it; then the sum over the levels above, one warp scanning downwards
        for (int t = tid; t < sched.levels; t += kTcThreads) {
            int lo = 0, hi = a.num_seqs;  // first rank with at most t tiles
            while (lo < hi) {
                const int mid = (lo + hi) >> 1;
                if (tiles[mid] > t) lo = mid + 1;
                else hi = mid;
            }
            const int np = a.pairs ? ((t + 1) * a.group + 1) / 2 - (t * a.group + 1) / 2 : a.group;
            base[t] = lo * a.kv_heads * np;
        }
        __syncthreads();
        if (warp == 0) {
            int above = 0;
            for (int t0 = sched.levels - 1; t0 >= 0; t0 -= 32) {
                const int t = t0 - lane;
                const int own = t >= 0 ? base[t] : 0;
                int sum = own;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int x = __shfl_up_sync(FULL, sum, o);
                    if (lane >= o) sum += x;
                }
                if (t >= 0) base[t] = above + sum - own;
                above += __shfl_sync(FULL, sum, 31);
            }
            if (lane == 0) *scan = above;
        }
        __syncthreads();
        sched.total = *scan;
        sched.level = sched.levels > 0 ? sched.levels - 1 : 0;
    }
    const uint32_t tmem = *tmem_slot;
    auto tmem_s = [&](int i) { return tmem + 128u * i; };
    auto tmem_o = [&](int i) { return tmem + 256u + static_cast<uint32_t>(DP) * i; };
    auto wait = [&](int b, uint32_t parity) {
        return mbar_wait_bounded(bar(b), parity & 1u, abort_flag, &g_attention_status);
    };
    AttUnit u;

    // A row of S takes 128 registers: the softmax groups get 200 each out of the launch's 168,
    // the others' warpgroup 96 (2 x 200 + 96 <= 3 x 168 in each quarter of the SM).
    if (warp < 8) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 200;");
        // ---- softmax: thread r of group w owns row r of item w
        const int w = warp >> 2, r = tid & 127;
        const uint32_t lane_base = static_cast<uint32_t>((warp & 3) * 32) << 16;
        const uint32_t ts = tmem_s(w) + lane_base, to = tmem_o(w) + lane_base;
        int step = 0, ring0 = 0, unit = 0, second = 0;
        bool ok = true;
        // Non-finite entries of the V tile of key tile j become zeros (and raise the flag); all
        // 256 softmax threads share the tile.
        auto scrub = [&](int j, int event) {
            const int st = (ring0 + 2 * j + 1) % Cfg::STAGES;
            ok = wait(B::VR + event, event ? second++ : unit);
            ok = __all_sync(FULL, ok);
            if (!ok) return;
            unsigned char* v = smem + Cfg::OFF_KV + st * Cfg::TILE;
            uint4 x[DP / 16];
            __half2 probe = __floats2half2_rn(0.f, 0.f);
            const __half2 zero = probe;
            const int nb = (a.head_dim + 63) / 64;  // boxes behind it were never loaded
#pragma unroll
            for (int c = 0; c < DP / 16; ++c) {
                if (c * 4096 < nb * Cfg::BLK) {
                    x[c] = *reinterpret_cast<const uint4*>(v + (tid + 256 * c) * 16);
                    const __half2* h = reinterpret_cast<const __half2*>(&x[c]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) probe = __hfma2(h[e], zero, probe);  // 0 or NaN
                }
            }
            if (!(__low2float(probe) == 0.f && __high2float(probe) == 0.f)) {
                odd_flag[(unit & 1) * 2 + event] = unit + 1;
                for (int c = 0; c * 4096 < nb * Cfg::BLK; ++c) {
                    __half* p = reinterpret_cast<__half*>(v + (tid + 256 * c) * 16);
                    for (int e = 0; e < 8; ++e)
                        if (odd_half(__half_as_ushort(p[e]))) p[e] = __float2half_rn(0.f);
                }
            }
            fence_async_smem();
            mbar_arrive(bar(B::SB + event));
        };
        for (; ok && sched.next(a, u); ++unit) {
            const int nt = u.nt[w];
            const int jd0 = u.nt[0] - 1, jd1 = u.nt[1] - 1;
            const int rows = u.n - u.q_lo[w] < kTile ? u.n - u.q_lo[w] : kTile;
            const int qpos = u.q_lo[w] + r;  // keys 0 .. qpos are visible
            float m = -INFINITY, l = 0.f;
            for (int j = 0; j < nt; ++j, ++step) {
                if (j == jd0 || j == jd1) {
                    scrub(j, j == jd0 ? 0 : 1);
                    if (!ok) break;
                }
                ok = wait(B::S + w, step);
                ok = __all_sync(FULL, ok);
                if (!ok) break;
                tc_fence_after();
                float v[128];
                tmem_ld4x32(ts, v);
                const int lim = qpos - j * kTile;  // columns 0 .. lim are visible
                const bool diag = j == nt - 1;
                if (diag) {
#pragma unroll
                    for (int i = 0; i < 128; ++i) v[i] = i <= lim ? v[i] : -INFINITY;
                }
                float mx = -INFINITY;
#pragma unroll
                for (int i = 0; i < 128; ++i) mx = fmaxf(mx, v[i]);
                const float mt = mx * a.scale_log2;
                // O and l are rescaled only when the maximum grew by more than 2^8: P stays
                // below 2^8 and 1 / l makes up for it.  -inf (nothing visible yet) always is.
                float alpha = 1.f;
                const bool grow = j == 0 || mt > m + 8.f;
                const bool need = j > 0 && grow;
                if (grow) {
                    if (need) {
                        alpha = m == -INFINITY ? 0.f : exp2_approx(m - mt);
                        l *= alpha;
                    }
                    m = mt;
                }
                const float sub = m == -INFINITY ? 0.f : -m;
                const float2 sc2 = make_float2(a.scale_log2, a.scale_log2);
                const float2 sub2 = make_float2(sub, sub);
                float2 l2 = make_float2(0.f, 0.f);
#pragma unroll
                for (int hf = 0; hf < 2; ++hf) {
                    uint32_t pk[32];
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        // 32 columns no row of the warp can see: zeros without exponentials
                        const int c0 = hf * 64 + c * 32;
                        const bool dark = diag && c0 > (warp & 3) * 32 + 31;
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            const int i = c0 + 2 * e;
                            uint32_t bits = 0u;
                            if (!dark) {
                                const float2 x = __ffma2_rn(make_float2(v[i], v[i + 1]), sc2, sub2);
                                const float2 p = make_float2(exp2_approx(x.x), exp2_approx(x.y));
                                l2 = __fadd2_rn(l2, p);
                                bits = pack_half2(p.x, p.y);
                            }
                            pk[c * 16 + e] = bits;
                        }
                    }
                    tmem_st32_bits(ts + hf * 32, pk);
                }
                l += l2.x + l2.y;
                if (__any_sync(FULL, need)) {  // the product before is done: S of this step follows it
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
            }
            if (!ok) break;
            if (w == 0 && jd1 > jd0) scrub(jd1, 1);
            if (w == 1 && nt == 0) scrub(jd0, 0);
            if (!ok) break;
            ring0 += 2 * (u.nt[1] > u.nt[0] ? u.nt[1] : u.nt[0]);
            if (nt == 0) continue;
            // ---- epilogue
            ok = wait(B::O + w, step - 1);
            ok = __all_sync(FULL, ok);
            if (!ok) break;
            tc_fence_after();
            const bool live = r < rows;
            const bool odd0 = odd_flag[(unit & 1) * 2] == unit + 1;
            const bool odd1 = jd1 > jd0 && odd_flag[(unit & 1) * 2 + 1] == unit + 1;
            const float inv = l == 0.f ? 0.f : 1.f / l;  // every score -inf: zeros
            const int64_t row = u.row0 + u.q_lo[w] + (live ? r : 0);
            const int64_t orow = row * a.out_stride + static_cast<int64_t>(u.head[w]) * a.head_dim;
#pragma unroll 1
            for (int c = 0; c < DP / 32; ++c) {
                if (c * 32 >= a.head_dim) break;
                float o[32];
                tmem_ld32(to + c * 32, o);
#pragma unroll
                for (int i = 0; i < 32; ++i) o[i] *= inv;
                if (odd0 || odd1) {
                    // the entries scrub() took out, for the rows that see them
                    const __half* vg = static_cast<const __half*>(a.v) + u.row0 * a.kv_stride +
                                       static_cast<int64_t>(u.kvh) * a.head_dim + c * 32;
                    for (int ev = 0; ev < 2; ++ev) {
                        if (!(ev ? odd1 : odd0)) continue;
                        const int k0 = (ev ? jd1 : jd0) * kTile;
                        for (int key = k0; key < k0 + kTile && key < u.n && key <= qpos; ++key) {
#pragma unroll
                            for (int i = 0; i < 32; ++i) {
                                if (c * 32 + i >= a.head_dim) continue;
                                const __half hv = vg[key * a.kv_stride + i];
                                if (odd_half(__half_as_ushort(hv))) o[i] += __half2float(hv);
                            }
                        }
                    }
                }
                if (!live) continue;
#pragma unroll
                for (int i = 0; i < 32; i += 8) {
                    if (c * 32 + i >= a.head_dim) break;
                    if (a.out_f32) {
                        float4* dst = reinterpret_cast<float4*>(static_cast<float*>(a.out) + orow +
                                                                c * 32 + i);
                        dst[0] = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
                        dst[1] = make_float4(o[i + 4], o[i + 5], o[i + 6], o[i + 7]);
                    } else {
                        *reinterpret_cast<uint4*>(static_cast<__half*>(a.out) + orow + c * 32 + i) =
                            make_uint4(pack_half2(o[i], o[i + 1]), pack_half2(o[i + 2], o[i + 3]),
                                       pack_half2(o[i + 4], o[i + 5]),
                                       pack_half2(o[i + 6], o[i + 7]));
                    }
                }
            }
            tc_fence_before();
            mbar_arrive(bar(B::E + w));
            if (a.lse && live)
                a.lse[row * a.q_heads + u.head[w]] =
                    ((m == -INFINITY ? 0.f : m) + log2f(l)) * kLn2;
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 96;");
        if (warp == 8) {
            if (lane == 0) {
                const int nb = (a.head_dim + 63) / 64;  // 64-column boxes that hold anything
                int ring = 0, cnt[2] = {0, 0};
                bool ok = true;
                auto load_q = [&](int i) {
                    const int qb = cnt[i] % Cfg::QBUF, round = cnt[i] / Cfg::QBUF;
                    ++cnt[i];
                    const int b = qb * 2 + i;
                    if (round > 0) ok = wait(B::QE + b, round - 1);
                    if (!ok) return;
                    mbar_arrive_tx(bar(B::QF + b), static_cast<uint32_t>(nb * Cfg::BLK));
                    for (int c = 0; c < nb; ++c)
                        tma_load_3d(sbase + b * Cfg::TILE + c * Cfg::BLK, &qmap, c * 64, u.head[i],
                                    static_cast<int>(u.row0) + u.q_lo[i], bar(B::QF + b));
                };
                auto load_kv = [&](const CUtensorMap* map, int j) {
                    const int st = ring % Cfg::STAGES, round = ring / Cfg::STAGES;
                    if (round > 0) ok = wait(B::KE + st, round - 1);
                    if (!ok) return;
                    ++ring;
                    mbar_arrive_tx(bar(B::KF + st), static_cast<uint32_t>(nb * Cfg::BLK));
                    for (int c = 0; c < nb; ++c)
                        tma_load_3d(sbase + Cfg::OFF_KV + st * Cfg::TILE + c * Cfg::BLK, map, c * 64,
                                    u.kvh, static_cast<int>(u.row0) + j * kTile, bar(B::KF + st));
                };
                while (ok && sched.next(a, u)) {
                    const int nt = u.nt[1] > u.nt[0] ? u.nt[1] : u.nt[0];
                    load_q(0);
                    if (ok) load_kv(&kmap, 0);
                    if (ok && u.nt[1]) load_q(1);
                    if (ok) load_kv(&vmap, 0);
                    for (int j = 1; ok && j < nt; ++j) {
                        load_kv(&kmap, j);
                        if (ok) load_kv(&vmap, j);
                    }
                }
                if (!ok) {  // another role gave up: let the copies in flight land
                    for (int i = ring < Cfg::STAGES ? 0 : ring - Cfg::STAGES; i < ring; ++i)
                        mbar_drain(bar(B::KF + i % Cfg::STAGES), (i / Cfg::STAGES) & 1);
                }
            }
        } else if (warp == 9) {
            if (lane == 0) {
                constexpr uint32_t IDESC_QK = f16_idesc(128, 128, false);
                constexpr uint32_t IDESC_PV = f16_idesc(128, DP, true);
                const int ksteps = (a.head_dim + 15) / 16;
                int ring0 = 0, qcnt[2] = {0, 0}, steps[2] = {0, 0}, events[2] = {0, 0};
                bool ok = true;
                auto stage_of = [&](int r) { return r % Cfg::STAGES; };
                auto full = [&](int r) { return wait(B::KF + stage_of(r), r / Cfg::STAGES); };
                // S_i = Q_i K_j^T.  P_i of the step before lies in S_i's columns: its product has to
                // be done.
                auto qk = [&](int i, int j) {
                    const int r = ring0 + 2 * j, qb = qcnt[i] % Cfg::QBUF;
                    if (j == 0) ok = wait(B::QF + qb * 2 + i, qcnt[i] / Cfg::QBUF);
                    ok = ok && full(r);
                    if (ok && steps[i] > 0) ok = wait(B::O + i, steps[i] - 1);
                    if (!ok) return;
                    tc_fence_after();
                    const uint32_t qa = sbase + (qb * 2 + i) * Cfg::TILE;
                    const uint32_t ka = sbase + Cfg::OFF_KV + stage_of(r) * Cfg::TILE;
                    for (int kk = 0; kk < ksteps; ++kk) {
                        const uint32_t off = (kk >> 2) * Cfg::BLK + (kk & 3) * 32;
                        tc_mma(tmem_s(i), sw128_desc(qa + off, 16, 1024),
                               sw128_desc(ka + off, 16, 1024), IDESC_QK, kk > 0);
                    }
                    tc_commit(bar(B::S + i));
                    if (i == 1 || u.nt[1] == 0) tc_commit(bar(B::KE + stage_of(r)));
                    if (j == u.nt[i] - 1) {
                        tc_commit(bar(B::QE + qb * 2 + i));
                    }
                };
                auto pv = [&](int i, int j) {
                    const int r = ring0 + 2 * j + 1;
                    ok = wait(B::P + i, steps[i]) && full(r);
                    // the accumulator still holds this item's previous unit
                    if (ok && j == 0 && qcnt[i] > 0) ok = wait(B::E + i, qcnt[i] - 1);
                    if (!ok) return;
                    tc_fence_after();
                    const uint32_t va = sbase + Cfg::OFF_KV + stage_of(r) * Cfg::TILE;
    #pragma unroll
                    for (int kk = 0; kk < kTile / 16; ++kk)
                        tc_mma_ts(tmem_o(i), tmem_s(i) + 8u * kk,
                                  sw128_desc(va + kk * 2048, Cfg::BLK, 1024), IDESC_PV,
                                  j > 0 || kk > 0);
                    tc_commit(bar(B::O + i));
                    ++steps[i];
                    if (i == 1 || u.nt[1] == 0) tc_commit(bar(B::KE + stage_of(r)));
                };
                // the diagonal tile's V has landed: the softmax groups may scrub it
                auto v_ready = [&](int j, int event) {
                    ok = ok && full(ring0 + 2 * j + 1);
                    if (ok) mbar_arrive(bar(B::VR + event));
                };
                while (ok && sched.next(a, u)) {
                    const int nt = u.nt[1] > u.nt[0] ? u.nt[1] : u.nt[0];
                    const int jd0 = u.nt[0] - 1, jd1 = u.nt[1] - 1;
                    qk(0, 0);
                    if (ok && u.nt[1]) qk(1, 0);
                    if (jd0 == 0) v_ready(0, 0);
                    for (int j = 0; ok && j < nt; ++j) {
                        // a diagonal tile's V is scrubbed by both softmax groups first
                        if (ok && (j == jd0 || j == jd1)) {
                            const int ev = j == jd0 ? 0 : 1;
                            ok = wait(B::SB + ev, events[ev]++);
                        }
                        if (ok && j < u.nt[0]) {
                            pv(0, j);
                            if (ok && j + 1 < u.nt[0]) qk(0, j + 1);
                            if (j + 1 == jd0) v_ready(j + 1, 0);
                        }
                        if (ok && j < u.nt[1]) {
                            pv(1, j);
                            if (ok && j + 1 < u.nt[1]) qk(1, j + 1);
                            if (j + 1 == jd1 && jd1 > jd0) v_ready(j + 1, 1);
                        }
                    }
                    ring0 += 2 * nt;
                    ++qcnt[0];
                    if (u.nt[1]) ++qcnt[1];
                }
                tc_commit(bar(B::DONE));  // every product is done before the CTA frees its memory
                mbar_drain(bar(B::DONE), 0);
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

template <int DP>
int launch_tc(PromptArgs a, cudaStream_t s) {
    using Cfg = AttCfg<DP>;
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
        TMLLM_CUDA_TRY(cudaFuncSetAttribute(prompt_tc_kernel<DP>,
                                            cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::SMEM));
        opted.fetch_or(bit, std::memory_order_relaxed);
    }
    const int sms = device_sm_count();
    const int total = a.num_seqs;
    const int32_t* starts = a.q_start;
    for (int s0 = 0; s0 < total; s0 += kMaxSeqs) {  // a launch schedules up to 1024 sequences
        a.num_seqs = total - s0 < kMaxSeqs ? total - s0 : kMaxSeqs;
        a.q_start = starts + s0;
        // at most one ragged tile a sequence
        const int64_t items = ((a.rows + kTile - 1) / kTile + a.num_seqs) * a.q_heads;
        if (items > INT32_MAX) return fail(TMLLM_INVALID_SHAPE, "too many prompt tiles");
        a.pairs = items > 2 * sms;
        const int64_t ctas = items < sms ? items : sms;
        prompt_tc_kernel<DP><<<static_cast<unsigned>(ctas), kTcThreads, Cfg::SMEM, s>>>(qmap, kmap,
                                                                                       vmap, a);
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
    int linear = 0, attention = 0, zero = 0;
    if (int st = take_linear_wait_status(&linear)) return st;
    TMLLM_CUDA_TRY(cudaMemcpyFromSymbol(&attention, g_attention_status, sizeof(int)));
    TMLLM_CUDA_TRY(cudaMemcpyToSymbol(g_attention_status, &zero, sizeof(int)));
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
    if (!std::isfinite(sc) || std::isnan(scale))
        return fail(TMLLM_INVALID_SHAPE, "attention scale must be positive and finite");
    const int64_t qw = static_cast<int64_t>(q_heads) * head_dim;
    const int64_t kw = static_cast<int64_t>(kv_heads) * head_dim;
    if (!q_stride) q_stride = qw;
    if (!kv_stride) kv_stride = kw;
    int64_t span;
    if (q_stride < qw || kv_stride < kw || !mul_ok(rows, q_stride, &span) ||
        !mul_ok(rows, kv_stride, &span) || span > INT64_MAX / 8)
        return fail(TMLLM_INVALID_SHAPE, "row strides of q / k / v must cover a row");
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
                    aligned16(out) && max_rows <= kMaxLevels * kTile &&
                    q_stride < (int64_t{1} << 38) && kv_stride < (int64_t{1} << 38);
    if (!tc) return launch_fma_d<__half>(a, s);
    return head_dim <= 64 ? launch_tc<64>(a, s) : launch_tc<128>(a, s);
}

}  // extern "C"
