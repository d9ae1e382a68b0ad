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
#include <cmath>

#include "common.cuh"

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
    float scale_log2;
};

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
    int linear = 0;
    if (int st = take_linear_wait_status(&linear)) return st;
    *status = linear;
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
    return dtype == TMLLM_F16 ? launch_fma_d<__half>(a, s) : launch_fma_d<float>(a, s);
}

}  // extern "C"
