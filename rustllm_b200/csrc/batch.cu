// Packed batches of requests: block tables and row maps built on the GPU from request
// lengths (tmllm_batch_tables), and the RoPE + paged append of packed rows by those maps
// (tmllm_rope_append).
#include "common.cuh"

namespace tmllm {
bool cache_owns_table(const int32_t* table);  // cache.cu

namespace {

// ---- block tables and slot maps ---------------------------------------------------------
constexpr int kTabThreads = 256;
constexpr int kTabItems = 4;                          // requests per thread and round
constexpr int kTabTile = kTabThreads * kTabItems;     // requests scanned per round
constexpr int kTabRows = 512;                         // rows per CTA before the grid grows

struct TableArgs {
    int32_t* block_table;
    const int32_t* seq_lens;
    const int32_t* new_lens;
    const int32_t* free_blocks;  // null: nothing is assigned
    const int32_t* free_start;   // null: 0
    int32_t* q_start;
    int32_t* positions;
    int32_t* row_seq;
    int64_t* slots;
    int32_t* info;
    int64_t num_blocks, rows, rows_per_cta;
    int32_t num_seqs, max_blocks, block_size, bs_shift, num_free;
};

__device__ __forceinline__ int64_t div_bs(const TableArgs& a, int64_t x) {
    if (a.bs_shift >= 0) return x >> a.bs_shift;
    if (x >> 32) return x / a.block_size;
    return static_cast<uint32_t>(x) / static_cast<uint32_t>(a.block_size);
}

// Exclusive prefix sums over the CTA of one (rows, blocks) pair per thread; `tot` receives
// the CTA's totals.
__device__ __forceinline__ void scan_pair(int64_t& rows, int64_t& blocks, int64_t (*warp_sums)[2],
                                          int64_t* tot) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t r0 = rows, b0 = blocks;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t r = __shfl_up_sync(0xffffffffu, rows, o);
        const int64_t b = __shfl_up_sync(0xffffffffu, blocks, o);
        if (lane >= o) {
            rows += r;
            blocks += b;
        }
    }
    if (lane == 31) {
        warp_sums[warp][0] = rows;
        warp_sums[warp][1] = blocks;
    }
    __syncthreads();
    int64_t pr = 0, pb = 0, tr = 0, tb = 0;
#pragma unroll
    for (int w = 0; w < kTabThreads / 32; ++w) {
        if (w == warp) {
            pr = tr;
            pb = tb;
        }
        tr += warp_sums[w][0];
        tb += warp_sums[w][1];
    }
    rows += pr - r0;
    blocks += pb - b0;
    tot[0] = tr;
    tot[1] = tb;
}

// Every CTA scans all requests (two loads and a prefix sum per 1024 of them), then writes
// its own share of the rows and of the table entries: no CTA waits for another, so one
// launch does everything.  A row finds its request by a binary search of the tile's row
// offsets in shared memory.  A block the call assigns is read from the free list, not from
// the table entry that another CTA writes.
// Bound by its chain of dependent steps (launch, lengths, prefix sum, search, table entry, store):
// 5.0 us a call in a graph for 64 requests of one token, 6.0 us for 512 requests of 83,929 rows
// (1.4 MB, 0.2 us of memory traffic).
__global__ void __launch_bounds__(kTabThreads) batch_tables_kernel(const TableArgs a) {
    __shared__ int64_t row0[kTabTile + 1];  // first row of each request of the tile
    __shared__ int64_t from[kTabTile];      // free-list index of its first new block
    __shared__ int32_t cached[kTabTile];    // cached length, or -1: refused
    __shared__ int64_t warp_sums[kTabThreads / 32][2];
    const int tid = threadIdx.x;
    const bool assign = a.free_blocks != nullptr;
    const int64_t start = (assign && a.free_start) ? *a.free_start : 0;
    const int64_t lo = static_cast<int64_t>(blockIdx.x) * a.rows_per_cta;
    const int64_t hi = lo + a.rows_per_cta < a.rows ? lo + a.rows_per_cta : a.rows;
    const int64_t cap = static_cast<int64_t>(a.max_blocks) * a.block_size;
    const int gwarp = blockIdx.x * (kTabThreads / 32) + (tid >> 5);
    const int nwarps = gridDim.x * (kTabThreads / 32);
    const int lane = tid & 31;
    int64_t rows_before = 0, blocks_before = 0, taken = 0;
    int32_t refused = 0;

    for (int base = 0; base < a.num_seqs; base += kTabTile) {
        int64_t n[kTabItems], need[kTabItems], sum_n = 0, sum_b = 0;
        int32_t len[kTabItems];
        bool fits[kTabItems];
#pragma unroll
        for (int i = 0; i < kTabItems; ++i) {
            const int s = base + tid * kTabItems + i;
            const bool in = s < a.num_seqs;
            len[i] = in ? __ldg(a.seq_lens + s) : 0;
            const int32_t nn = in ? __ldg(a.new_lens + s) : 0;
            n[i] = nn > 0 ? nn : 0;
            const int64_t end = len[i] + n[i];
            fits[i] = len[i] >= 0 && end <= cap;
            need[i] = 0;
            if (assign && fits[i])
                need[i] = div_bs(a, end + a.block_size - 1) -
                          div_bs(a, static_cast<int64_t>(len[i]) + a.block_size - 1);
            sum_n += n[i];
            sum_b += need[i];
        }
        int64_t pr = sum_n, pb = sum_b, tot[2];
        __syncthreads();  // the previous tile's rows are done with the shared arrays
        scan_pair(pr, pb, warp_sums, tot);
        pr += rows_before;
        pb += blocks_before;
#pragma unroll
        for (int i = 0; i < kTabItems; ++i) {
            const int t = tid * kTabItems + i, s = base + t;
            const bool placed =
                fits[i] &&
                (need[i] == 0 || (start >= 0 && start + pb + need[i] <= a.num_free));
            row0[t] = pr;
            from[t] = start + pb;
            cached[t] = placed ? len[i] : -1;
            if (s < a.num_seqs) {
                if (placed) taken += need[i];
                else ++refused;
                if (blockIdx.x == 0)
                    a.q_start[s] = static_cast<int32_t>(pr < INT32_MAX ? pr : INT32_MAX);
            }
            pr += n[i];
            pb += need[i];
        }
        rows_before += tot[0];
        blocks_before += tot[1];
        if (tid == 0) row0[kTabTile] = rows_before;
        __syncthreads();
        const int count = a.num_seqs - base < kTabTile ? a.num_seqs - base : kTabTile;

        // new table entries: one warp per request
        if (assign) {
            for (int t = gwarp; t < count; t += nwarps) {
                if (cached[t] < 0) continue;
                const int64_t len_t = cached[t], nt = row0[t + 1] - row0[t];
                const int64_t held = div_bs(a, len_t + a.block_size - 1);
                const int64_t after = div_bs(a, len_t + nt + a.block_size - 1);
                int32_t* row = a.block_table + static_cast<int64_t>(base + t) * a.max_blocks;
                for (int64_t b = held + lane; b < after; b += 32)
                    row[b] = __ldg(a.free_blocks + from[t] + (b - held));
            }
        }
        // this CTA's rows that belong to the tile's requests
        const int64_t r_lo = lo > row0[0] ? lo : row0[0];
        const int64_t r_hi = hi < rows_before ? hi : rows_before;
        for (int64_t r = r_lo + tid; r < r_hi; r += kTabThreads) {
            int x = 0, y = count - 1;  // the last request whose first row is <= r
            while (x < y) {
                const int mid = (x + y + 1) >> 1;
                if (row0[mid] <= r) x = mid;
                else y = mid - 1;
            }
            int32_t pos = -1;
            int64_t slot = -1;
            if (cached[x] >= 0) {
                const int64_t p = cached[x] + (r - row0[x]);  // < cap <= INT32_MAX
                const int64_t idx = div_bs(a, p);
                const int64_t held = div_bs(a, static_cast<int64_t>(cached[x]) + a.block_size - 1);
                pos = static_cast<int32_t>(p);
                const int32_t blk =
                    (assign && idx >= held)
                        ? __ldg(a.free_blocks + from[x] + (idx - held))
                        : a.block_table[static_cast<int64_t>(base + x) * a.max_blocks + idx];
                if (blk >= 0 && blk < a.num_blocks)
                    slot = static_cast<int64_t>(blk) * a.block_size + (p - idx * a.block_size);
            }
            a.positions[r] = pos;
            a.row_seq[r] = base + x;
            a.slots[r] = slot;
        }
    }
    // rows behind the last request belong to nobody
    const int64_t tail = lo > rows_before ? lo : rows_before;
    for (int64_t r = tail + tid; r < hi; r += kTabThreads) {
        a.positions[r] = -1;
        a.row_seq[r] = -1;
        a.slots[r] = -1;
    }
    if (blockIdx.x == 0) {
        int64_t c = refused, tot[2];
        __syncthreads();
        scan_pair(taken, c, warp_sums, tot);
        if (tid == 0) {
            const int64_t over = rows_before - a.rows;
            auto sat = [](int64_t v) {
                return static_cast<int32_t>(v < INT32_MAX ? v : INT32_MAX);
            };
            a.q_start[a.num_seqs] = sat(rows_before);
            a.info[0] = sat(start + tot[0]);
            a.info[1] = sat(rows_before);
            a.info[2] = sat(tot[1]);
            a.info[3] = sat(over > 0 ? over : 0);
        }
    }
}

// ---- RoPE + paged append of packed rows -------------------------------------------------
struct AppendArgs {
    const void* q;
    const void* k;
    const void* v;
    void* q_out;
    void* k_out;  // null: the rotated keys go to the cache only
    void* k_cache;
    void* v_cache;
    const int32_t* positions;
    const int64_t* slots;
    const float* cos_table;
    const float* sin_table;
    int64_t rows, arena_slots;
    int64_t q_stride, kv_stride, qo_stride, ko_stride;
    int32_t q_heads, kv_heads, head_dim, block_size, rope_len;
};

// TMLLM_POSITION_OUT_OF_RANGE once a row's position was past the rotation tables: it is cached
// unrotated, which no output shows.
__device__ int g_append_status;

__device__ __forceinline__ bool turned(const AppendArgs& a, int pos, bool report) {
    if (a.cos_table == nullptr) return false;
    if (pos < a.rope_len) return true;
    if (report) g_append_status = TMLLM_POSITION_OUT_OF_RANGE;
    return false;
}

// kernels/rope.metal:57-63 without contraction, F32.
__device__ __forceinline__ void rotate(float& x1, float& x2, float c, float s) {
    const float y1 = __fsub_rn(__fmul_rn(x1, c), __fmul_rn(x2, s));
    const float y2 = __fadd_rn(__fmul_rn(x2, c), __fmul_rn(x1, s));
    x1 = y1;
    x2 = y2;
}

// Any head size and alignment: one thread per (row, head of q | k | v, pair).
template <typename T>
__global__ void __launch_bounds__(256) rope_append_scalar_kernel(const AppendArgs a) {
    const int half = a.head_dim / 2;
    const int heads = a.q_heads + 2 * a.kv_heads;
    const int64_t total = a.rows * heads * half;
    for (int64_t idx = blockIdx.x * static_cast<int64_t>(blockDim.x) + threadIdx.x; idx < total;
         idx += static_cast<int64_t>(gridDim.x) * blockDim.x) {
        const int i = static_cast<int>(idx % half);
        const int64_t t = idx / half;
        const int hh = static_cast<int>(t % heads);
        const int64_t row = t / heads;
        const int pos = a.positions[row];
        if (pos < 0) continue;
        const bool is_q = hh < a.q_heads, is_v = hh >= a.q_heads + a.kv_heads;
        const int h = is_q ? hh : is_v ? hh - a.q_heads - a.kv_heads : hh - a.q_heads;
        const T* src = (is_q ? static_cast<const T*>(a.q) + row * a.q_stride
                             : static_cast<const T*>(is_v ? a.v : a.k) + row * a.kv_stride) +
                       static_cast<int64_t>(h) * a.head_dim;
        T y1 = src[i], y2 = src[i + half];
        if (!is_v && turned(a, pos, hh == 0 && i == 0)) {
            float x1 = to_f32<T>(y1), x2 = to_f32<T>(y2);
            const int64_t e = static_cast<int64_t>(pos) * half + i;
            rotate(x1, x2, __ldg(a.cos_table + e), __ldg(a.sin_table + e));
            y1 = from_f32<T>(x1);
            y2 = from_f32<T>(x2);
        }
        if (is_q) {
            T* o = static_cast<T*>(a.q_out) + row * a.qo_stride +
                   static_cast<int64_t>(h) * a.head_dim;
            o[i] = y1;
            o[i + half] = y2;
            continue;
        }
        if (!is_v && a.k_out) {
            T* o = static_cast<T*>(a.k_out) + row * a.ko_stride +
                   static_cast<int64_t>(h) * a.head_dim;
            o[i] = y1;
            o[i + half] = y2;
        }
        const int64_t slot = a.slots[row];
        if (slot < 0 || slot >= a.arena_slots) continue;
        const int64_t blk = slot / a.block_size;
        T* o = static_cast<T*>(is_v ? a.v_cache : a.k_cache) +
               ((blk * a.kv_heads + h) * a.block_size + (slot - blk * a.block_size)) * a.head_dim;
        o[i] = y1;
        o[i + half] = y2;
    }
}

// 16-byte form (D / 2 a multiple of a 16-byte chunk, aligned rows).  A warp takes one row (or a
// share of its heads): lane = (head of the pass, chunk c of the first half), so a lane's chunk -
// and with it its cos / sin entries - stays the same while it walks the heads, and the tables are
// read once a row.  kUnroll heads are loaded before the first is used.
// Bound by memory: every element is read once and written once or twice (cache and dense):
// 22,054 rows of 32/8 heads of 128 take 98 us, 6.1 TB/s or 93 % of the measured copy rate; 24 rows
// of 9/3 heads of 64 2.8 us in a graph.
template <typename T>
__global__ void __launch_bounds__(256) rope_append_vec_kernel(const AppendArgs a, int parts) {
    constexpr int EPC = 16 / sizeof(T), kUnroll = 4;
    const int lane = threadIdx.x & 31;
    const int64_t unit = blockIdx.x * static_cast<int64_t>(blockDim.x >> 5) + (threadIdx.x >> 5);
    const int64_t row = unit / parts;
    const int part = static_cast<int>(unit - row * parts);
    if (row >= a.rows) return;
    const int half = a.head_dim / 2, cph = half / EPC, hpp = 32 / cph;  // heads a pass
    const int hl = lane / cph, c = lane - hl * cph;
    const int pos = __ldg(a.positions + row);
    if (pos < 0 || hl >= hpp) return;
    const int64_t slot = __ldg(a.slots + row);
    const bool cached = slot >= 0 && slot < a.arena_slots;
    int64_t cell = 0;  // element of (block, head 0, offset) in the arenas
    if (cached) {
        const int64_t blk = (slot >> 32) ? slot / a.block_size
                                         : static_cast<uint32_t>(slot) / a.block_size;
        cell = (blk * a.kv_heads * a.block_size + (slot - blk * a.block_size)) * a.head_dim;
    }
    const int64_t head_step = static_cast<int64_t>(a.block_size) * a.head_dim;
    float cs[EPC], sn[EPC];
    const bool turn = turned(a, pos, part == 0 && lane == 0);
    if (turn) {
        const int64_t e = static_cast<int64_t>(pos) * half + c * EPC;
#pragma unroll
        for (int i = 0; i < EPC; i += 4) {
            const float4 x = __ldg(reinterpret_cast<const float4*>(a.cos_table + e + i));
            const float4 y = __ldg(reinterpret_cast<const float4*>(a.sin_table + e + i));
            cs[i] = x.x, cs[i + 1] = x.y, cs[i + 2] = x.z, cs[i + 3] = x.w;
            sn[i] = y.x, sn[i + 1] = y.y, sn[i + 2] = y.z, sn[i + 3] = y.w;
        }
    }
    const int heads = a.q_heads + 2 * a.kv_heads;
    const T* qr = static_cast<const T*>(a.q) + row * a.q_stride + c * EPC;
    const T* kr = static_cast<const T*>(a.k) + row * a.kv_stride + c * EPC;
    const T* vr = static_cast<const T*>(a.v) + row * a.kv_stride + c * EPC;
    for (int h0 = part * hpp + hl; h0 < heads; h0 += kUnroll * parts * hpp) {
        uint4 x1[kUnroll], x2[kUnroll];
#pragma unroll
        for (int k = 0; k < kUnroll; ++k) {
            const int h = h0 + k * parts * hpp;
            if (h >= heads) break;
            const T* src = h < a.q_heads ? qr + static_cast<int64_t>(h) * a.head_dim
                           : h < a.q_heads + a.kv_heads
                               ? kr + static_cast<int64_t>(h - a.q_heads) * a.head_dim
                               : vr + static_cast<int64_t>(h - a.q_heads - a.kv_heads) * a.head_dim;
            x1[k] = *reinterpret_cast<const uint4*>(src);
            x2[k] = *reinterpret_cast<const uint4*>(src + half);
        }
#pragma unroll
        for (int k = 0; k < kUnroll; ++k) {
            const int h = h0 + k * parts * hpp;
            if (h >= heads) break;
            const bool is_q = h < a.q_heads, is_v = h >= a.q_heads + a.kv_heads;
            if (turn && !is_v) {
                float f1[EPC], f2[EPC];
                Chunk<T>::unpack(x1[k], f1);
                Chunk<T>::unpack(x2[k], f2);
                T* p1 = reinterpret_cast<T*>(&x1[k]);
                T* p2 = reinterpret_cast<T*>(&x2[k]);
#pragma unroll
                for (int e = 0; e < EPC; ++e) {
                    rotate(f1[e], f2[e], cs[e], sn[e]);
                    p1[e] = from_f32<T>(f1[e]);
                    p2[e] = from_f32<T>(f2[e]);
                }
            }
            const int kvh = is_v ? h - a.q_heads - a.kv_heads : h - a.q_heads;
            if (is_q || (!is_v && a.k_out)) {
                T* o = is_q ? static_cast<T*>(a.q_out) + row * a.qo_stride +
                                  static_cast<int64_t>(h) * a.head_dim + c * EPC
                            : static_cast<T*>(a.k_out) + row * a.ko_stride +
                                  static_cast<int64_t>(kvh) * a.head_dim + c * EPC;
                *reinterpret_cast<uint4*>(o) = x1[k];
                *reinterpret_cast<uint4*>(o + half) = x2[k];
            }
            if (!is_q && cached) {
                T* o = static_cast<T*>(is_v ? a.v_cache : a.k_cache) + cell + kvh * head_step + c * EPC;
                *reinterpret_cast<uint4*>(o) = x1[k];
                *reinterpret_cast<uint4*>(o + half) = x2[k];
            }
        }
    }
}

int grid_of(int64_t items) {
    int64_t blocks = (items + 255) / 256;
    const int64_t cap = static_cast<int64_t>(device_sm_count()) * 32;
    if (blocks > cap) blocks = cap;
    return static_cast<int>(blocks < 1 ? 1 : blocks);
}

}  // namespace
}  // namespace tmllm

using namespace tmllm;

extern "C" {

int tmllm_append_status(int32_t* status) {
    clear_error();
    if (!status) return fail(TMLLM_INVALID_ARGUMENT, "null status pointer");
    return take_status(g_append_status, status);
}

int tmllm_batch_tables(const tmllm_paged_kv* kv, const int32_t* new_lens,
                       const int32_t* free_blocks, int32_t num_free, const int32_t* free_start,
                       int64_t rows, int32_t* q_start, int32_t* positions, int32_t* row_seq,
                       int64_t* slots, int32_t* info, tmllm_stream stream) {
    clear_error();
    if (!kv) return fail(TMLLM_INVALID_ARGUMENT, "null paged KV descriptor");
    if (kv->num_seqs <= 0 || kv->block_size <= 0 || kv->max_blocks_per_seq <= 0 ||
        kv->num_blocks <= 0)
        return fail(TMLLM_INVALID_SHAPE, "paged KV dimensions must be positive");
    if (rows < 0 || rows > INT32_MAX)
        return fail(TMLLM_INVALID_SHAPE, "rows must be in [0, 2^31), got %lld",
                    static_cast<long long>(rows));
    if (num_free < 0) return fail(TMLLM_INVALID_SHAPE, "num_free must be non-negative");
    int64_t cap;
    if (!mul_ok(kv->max_blocks_per_seq, kv->block_size, &cap) || cap > INT32_MAX)
        return fail(TMLLM_INVALID_SHAPE, "a sequence's capacity must fit 31 bits");
    if (!kv->block_table || !kv->seq_lens || !new_lens || !q_start || !info ||
        (rows > 0 && (!positions || !row_seq || !slots)))
        return fail(TMLLM_INVALID_ARGUMENT, "null tensor pointer");
    if (free_start && free_start >= info && free_start < info + 4)
        return fail(TMLLM_INVALID_ARGUMENT, "free_start must not lie in info, which is written");
    if (free_blocks && cache_owns_table(kv->block_table))
        return fail(TMLLM_INVALID_ARGUMENT,
                    "the table is a cache's, which hands out its own blocks (tmllm_cache_reserve): "
                    "no free list");
    // every CTA reads the lengths and lists while others write: nothing written may be read, or
    // written as something else
    const Span table{kv->block_table, int64_t{4} * kv->num_seqs * kv->max_blocks_per_seq};
    const Span out[6] = {{q_start, int64_t{4} * (kv->num_seqs + int64_t{1})},
                         {positions, 4 * rows},
                         {row_seq, 4 * rows},
                         {slots, 8 * rows},
                         {info, 16},
                         free_blocks ? table : Span{nullptr, 0}};
    const Span in[5] = {{kv->seq_lens, int64_t{4} * kv->num_seqs},
                        {new_lens, int64_t{4} * kv->num_seqs},
                        {free_blocks, int64_t{4} * num_free},
                        {free_start, 4},
                        free_blocks ? Span{nullptr, 0} : table};
    for (int o = 0; o < 6; ++o) {
        for (const Span& i : in)
            if (overlaps(out[o], i))
                return fail(TMLLM_INVALID_ARGUMENT, "an output overlaps an input");
        for (int p = 0; p < o; ++p)
            if (overlaps(out[o], out[p]))
                return fail(TMLLM_INVALID_ARGUMENT, "two outputs overlap");
    }
    TableArgs a{};
    a.block_table = const_cast<int32_t*>(kv->block_table);  // written only with free_blocks
    a.seq_lens = kv->seq_lens;
    a.new_lens = new_lens;
    a.free_blocks = free_blocks;
    a.free_start = free_start;
    a.q_start = q_start;
    a.positions = positions;
    a.row_seq = row_seq;
    a.slots = slots;
    a.info = info;
    a.num_blocks = kv->num_blocks;
    a.rows = rows;
    a.num_seqs = kv->num_seqs;
    a.max_blocks = kv->max_blocks_per_seq;
    a.block_size = kv->block_size;
    a.num_free = num_free;
    a.bs_shift = -1;
    if ((kv->block_size & (kv->block_size - 1)) == 0)
        for (a.bs_shift = 0; (1 << a.bs_shift) < kv->block_size;) ++a.bs_shift;
    int64_t ctas = (rows + kTabRows - 1) / kTabRows;
    if (ctas < 1) ctas = 1;
    if (ctas > device_sm_count()) ctas = device_sm_count();
    a.rows_per_cta = (rows + ctas - 1) / ctas;
    batch_tables_kernel<<<static_cast<unsigned>(ctas), kTabThreads, 0,
                          reinterpret_cast<cudaStream_t>(stream)>>>(a);
    TMLLM_LAUNCH_TRY();
    return TMLLM_OK;
}

int tmllm_rope_append(const tmllm_paged_kv* kv, const void* q, const void* k, const void* v,
                      int64_t rows, int32_t q_heads, int64_t q_stride, int64_t kv_stride,
                      const int32_t* positions, const int64_t* slots, const float* rope_cos,
                      const float* rope_sin, int32_t rope_len, void* q_out, int64_t q_out_stride,
                      void* k_out, int64_t k_out_stride, tmllm_stream stream) {
    clear_error();
    if (!kv) return fail(TMLLM_INVALID_ARGUMENT, "null paged KV descriptor");
    if (!valid_dtype(kv->dtype)) return fail(TMLLM_UNSUPPORTED_DTYPE, "unknown cache dtype");
    const int64_t D = kv->head_dim, Hkv = kv->num_kv_heads;
    if (Hkv <= 0 || D <= 0 || kv->block_size <= 0 || kv->num_blocks <= 0)
        return fail(TMLLM_INVALID_SHAPE, "paged KV dimensions must be positive");
    if (D % 2 != 0) return fail(TMLLM_INVALID_SHAPE, "RoPE requires an even head dimension");
    if (q_heads <= 0 || q_heads % Hkv != 0)
        return fail(TMLLM_MODEL_FORMAT, "Q heads %d must be divisible by non-zero KV heads %d",
                    q_heads, static_cast<int>(Hkv));
    if (rows < 0 || rows > INT32_MAX)
        return fail(TMLLM_INVALID_SHAPE, "rows must be in [0, 2^31)");
    if (rows == 0) return TMLLM_OK;
    const int64_t qw = q_heads * D, kw = Hkv * D;
    if (!q_stride) q_stride = qw;
    if (!kv_stride) kv_stride = kw;
    if (!q_out_stride) q_out_stride = qw;
    if (!k_out_stride) k_out_stride = kw;
    int64_t span, arena_slots, arena;
    if (q_stride < qw || q_out_stride < qw || kv_stride < kw || k_out_stride < kw)
        return fail(TMLLM_INVALID_SHAPE, "row strides must cover a row");
    for (int64_t stride : {q_stride, kv_stride, q_out_stride, k_out_stride})
        if (!mul_ok(rows, stride, &span) || span > INT64_MAX / 8)
            return fail(TMLLM_INVALID_SHAPE, "rows and row strides must fit 60 bits");
    if (!mul_ok(kv->num_blocks, kv->block_size, &arena_slots) || !mul_ok(arena_slots, kw, &arena) ||
        arena > INT64_MAX / 8)
        return fail(TMLLM_INVALID_SHAPE, "the arenas must fit 60 bits");
    if (!q || !k || !v || !q_out || !kv->k_cache || !kv->v_cache || !positions || !slots)
        return fail(TMLLM_INVALID_ARGUMENT, "null tensor pointer");
    if ((rope_cos == nullptr) != (rope_sin == nullptr) || (rope_cos && rope_len <= 0))
        return fail(TMLLM_INVALID_ARGUMENT, "RoPE needs both tables and a positive length");
    const size_t es = dtype_size(kv->dtype);
    for (const void* p : {q, k, v, static_cast<const void*>(q_out),
                          static_cast<const void*>(k_out), static_cast<const void*>(kv->k_cache),
                          static_cast<const void*>(kv->v_cache)})
        if (reinterpret_cast<uintptr_t>(p) % es)
            return fail(TMLLM_INVALID_ARGUMENT,
                        "tensor pointers must be aligned to their element size");
    // an output may be its own input, row for row; any other overlap would be read after it
    // was written
    const Rows in[3] = {{q, q_stride, qw}, {k, kv_stride, kw}, {v, kv_stride, kw}};
    const Rows out[2] = {{q_out, q_out_stride, qw}, {k_out, k_out_stride, kw}};
    for (int o = 0; o < (k_out ? 2 : 1); ++o)
        for (int i = 0; i < 3; ++i) {
            if (o == i && out[o].p == in[i].p && out[o].stride == in[i].stride) continue;
            if (overlaps(out[o], in[i], rows, es))
                return fail(TMLLM_INVALID_ARGUMENT,
                            "q_out / k_out may be q / k themselves, but not overlap an input");
        }
    if (k_out && overlaps(out[0], out[1], rows, es))
        return fail(TMLLM_INVALID_ARGUMENT, "q_out and k_out overlap");
    // nor may anything written be cache for the one and row, index or table for the other
    const int64_t table = rope_cos ? int64_t{2} * rope_len * D : 0;
    const Span arenas[2] = {{kv->k_cache, arena * static_cast<int64_t>(es)},
                            {kv->v_cache, arena * static_cast<int64_t>(es)}};
    const Span read[4] = {{positions, 4 * rows}, {slots, 8 * rows}, {rope_cos, table},
                          {rope_sin, table}};
    for (const Rows& o : out) {
        for (const Span& c : arenas)
            if (inside(c.p, c.bytes, o, rows, es))
                return fail(TMLLM_INVALID_ARGUMENT, "q_out / k_out overlap the cache");
        for (const Span& r : read)
            if (inside(r.p, r.bytes, o, rows, es))
                return fail(TMLLM_INVALID_ARGUMENT,
                            "q_out / k_out overlap the positions, slots or RoPE tables");
    }
    for (const Span& c : arenas)
        for (const Span& r : read)
            if (overlaps(c, r))
                return fail(TMLLM_INVALID_ARGUMENT,
                            "the cache overlaps the positions, slots or RoPE tables");
    AppendArgs a{};
    a.q = q;
    a.k = k;
    a.v = v;
    a.q_out = q_out;
    a.k_out = k_out;
    a.k_cache = kv->k_cache;
    a.v_cache = kv->v_cache;
    a.positions = positions;
    a.slots = slots;
    a.cos_table = rope_cos;
    a.sin_table = rope_sin;
    a.rows = rows;
    a.arena_slots = arena_slots;
    a.q_stride = q_stride;
    a.kv_stride = kv_stride;
    a.qo_stride = q_out_stride;
    a.ko_stride = k_out_stride;
    a.q_heads = q_heads;
    a.kv_heads = kv->num_kv_heads;
    a.head_dim = kv->head_dim;
    a.block_size = kv->block_size;
    a.rope_len = rope_len;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    const int64_t epc = 16 / static_cast<int64_t>(es);
    bool vec = (D / 2) % epc == 0 && D / 2 / epc <= 32 && q_stride % epc == 0 &&
               kv_stride % epc == 0 && q_out_stride % epc == 0 && k_out_stride % epc == 0 &&
               (!rope_cos || (aligned16(rope_cos) && aligned16(rope_sin)));
    for (const void* p : {q, k, v, static_cast<const void*>(q_out),
                          static_cast<const void*>(k_out), static_cast<const void*>(kv->k_cache),
                          static_cast<const void*>(kv->v_cache)})
        vec = vec && aligned16(p);
    if (vec) {
        // a warp a row; few rows: as many warps a row as its heads give, up to 8 warps an SM
        const int64_t passes = (q_heads + 2 * Hkv) * (D / 2 / epc) / 32 + 1;
        int64_t parts = static_cast<int64_t>(device_sm_count()) * 8 / rows;
        if (parts > passes) parts = passes;
        if (parts < 1) parts = 1;
        const int64_t ctas = (rows * parts + 7) / 8;
        if (ctas > INT32_MAX) return fail(TMLLM_INVALID_SHAPE, "too many rows");
        if (kv->dtype == TMLLM_F16)
            rope_append_vec_kernel<__half>
                <<<static_cast<unsigned>(ctas), 256, 0, s>>>(a, static_cast<int>(parts));
        else
            rope_append_vec_kernel<float>
                <<<static_cast<unsigned>(ctas), 256, 0, s>>>(a, static_cast<int>(parts));
    } else {
        const int nb = grid_of(rows * (q_heads + 2 * Hkv) * (D / 2));
        if (kv->dtype == TMLLM_F16) rope_append_scalar_kernel<__half><<<nb, 256, 0, s>>>(a);
        else rope_append_scalar_kernel<float><<<nb, 256, 0, s>>>(a);
    }
    TMLLM_LAUNCH_TRY();
    return TMLLM_OK;
}

}  // extern "C"
