// The weights that many queries (a prompt, or its last tokens) give the slots that they see, summed over queries and over the query heads of a key/value head, added to the slots' weights:
//
//     y_vj = q_v . k_j scale log2(e),   m_v = max_j y_vj,   l_v = sum_j 2^(y_vj - m_v),   weights[j] += sum_v 2^(y_vj - m_v) / l_v
//
// v counts a request's (token, head) rows of a key/value head, token by token; token i of n sees the first length - n + i + 1 slots.  There is no result beside the weights, so values are not read.
//
// A weight is known only when its row's sum is, and a sum over rows has another owner than a row's, so the scores are made twice: the first walk goes along the slots and leaves m and 1 / l of every row,
// the second goes along the rows and adds up every slot's weights.  (Keeping them would move 8 bytes a score, against 2 d operations for making them again.)  Both walks have one shape: a tile of 64 rows
// (of Q; then of K) stays in registers as the products' operand of 16 rows a warp, tiles of the others pass through shared memory, two at a time.  Sums over what passes end up in one lane's hands, and
// nothing is added by atomics, so results do not depend on which block came first.
//
// Where few rows would leave the device empty, the first walk's slots are cut, and its blocks leave (m, l) of every row and cut, which a small kernel puts together.
//
// Slots beyond a request's length may hold anything: they are read as zeros and their scores are not looked at.
#include "common.cuh"

#ifndef HB_HEAD_DIM
#define HB_HEAD_DIM 128
#endif

namespace {
typedef __nv_bfloat16 bf16;
constexpr int D = HB_HEAD_DIM;
static_assert(D == 64 || D == 128, "head sizes 64 and 128");
constexpr int ROWS = 64, WARPS = 4, THREADS = 32 * WARPS, TILE = ROWS * D * 2, CHUNKS = D / 8;

__device__ __forceinline__ unsigned smem_u32(const void* p) { return (unsigned)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void ldmatrix_x4(unsigned (&r)[4], unsigned at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];\n" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at));
}
__device__ __forceinline__ void mma(float (&c)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float fast_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// 16-byte chunk c of row r of a tile: rows of 128 bytes in panels, their chunks permuted so that eight rows of one column meet eight banks.
__device__ __forceinline__ unsigned tile_at(int r, int c) { return (unsigned)((c >> 3) * (ROWS * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4)); }

struct Args {
    const bf16* q; int q_stride;
    const bf16* cache;
    const int* block_table; int table_width;
    const int* starts;    // [requests + 1]
    const int* lengths;   // [requests]
    int tokens, most, longest;
    float* weights;       // [requests, kv_heads, capacity]
    int capacity;
    float2* rows;         // [tokens * heads]: (m, 1 / l)
    float2* cuts;         // [n_cuts, tokens * heads]: (m, l), where the slots are cut
    int n_cuts;
    int heads, kv_heads, page_shift, pages;
    float scale_log2;
    int* status;
};
struct Request {
    int first, tokens, length;  // its queries, its slots
};
__device__ __forceinline__ Request request_of(const Args& a, int r, bool reports) {
    int first = a.starts[r], tokens = a.starts[r + 1] - first, length = a.lengths[r];
    if (reports && (first < 0 || tokens < 0 || tokens > a.most || first > a.tokens - tokens || length > a.longest)) atomicOr(a.status, HB_STATUS_BAD_POSITION);
    first = min(max(first, 0), a.tokens), tokens = min(min(max(tokens, 0), a.most), a.tokens - first), length = min(max(length, 0), a.longest);
    return {first, tokens, length};
}

// Rows row0 .. row0 + 63 of a request's queries, or slots slot0 .. of its keys, on their way into a tile; zeros beyond their end.
__device__ __forceinline__ void copy_chunk(unsigned dst, const void* src, bool valid) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}
__device__ __forceinline__ void fetch_queries(const Args& a, const Request& q, int kvh, int group, int row0, unsigned tile) {
    for (int i = threadIdx.x; i < ROWS * CHUNKS; i += THREADS) {
        const int r = i / CHUNKS, c = i % CHUNKS, v = row0 + r, token = v / group;
        const bool valid = token < q.tokens;
        copy_chunk(tile + tile_at(r, c), valid ? a.q + (size_t)(q.first + token) * a.q_stride + (size_t)(kvh * group + v - token * group) * D + c * 8 : a.q, valid);
    }
}
__device__ __forceinline__ void fetch_keys(const Args& a, int request, int length, int kvh, int slot0, unsigned tile) {
    for (int i = threadIdx.x; i < ROWS * CHUNKS; i += THREADS) {
        const int r = i / CHUNKS, c = i % CHUNKS, slot = slot0 + r;
        int page = -1;
        if (slot < length) {
            page = __ldg(a.block_table + (size_t)request * a.table_width + (slot >> a.page_shift));
            if (page < 0 || page >= a.pages) {
                atomicOr(a.status, HB_STATUS_BAD_PAGE);
                page = -1;
            }
        }
        const size_t row = (((size_t)(page < 0 ? 0 : page) * 2 * a.kv_heads + kvh) << a.page_shift) + (slot & ((1 << a.page_shift) - 1));
        copy_chunk(tile + tile_at(r, c), page < 0 ? a.cache : a.cache + row * D + c * 8, page >= 0);
    }
}
__device__ __forceinline__ void committed() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void arrived() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// This warp's 16 rows of the tile that stays.
__device__ __forceinline__ void load_staying(unsigned (&x)[D / 16][4], unsigned tile) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int k = 0; k < D / 16; ++k) ldmatrix_x4(x[k], tile + tile_at(warp * 16 + (lane & 15), 2 * k + (lane >> 4)));
}
// The scores of this warp's 16 rows and the 64 of the passing tile: [8 of them][(row g or g + 8, row 2 t or 2 t + 1 of the 8)].
__device__ __forceinline__ void products(float (&s)[8][4], const unsigned (&x)[D / 16][4], unsigned tile) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int n = 0; n < 8; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
    for (int k = 0; k < D / 32; ++k)
#pragma unroll
        for (int n = 0; n < 8; ++n) {
            unsigned b[4];
            ldmatrix_x4(b, tile + tile_at(n * 8 + (lane & 7), 4 * k + (lane >> 3)));
            mma(s[n], x[2 * k], b[0], b[1]);
            mma(s[n], x[2 * k + 1], b[2], b[3]);
        }
}

// The first walk: block (cut, row tile and key/value head, request).
__global__ void __launch_bounds__(THREADS) rows_kernel(const Args a) {
    extern __shared__ __align__(128) unsigned char smem[];
    const unsigned tiles = smem_u32(smem);
    let_next_kernel_start();
    wait_for_previous_kernels();
    const int kvh = blockIdx.y % a.kv_heads, row0 = blockIdx.y / a.kv_heads * ROWS, group = a.heads / a.kv_heads;
    const Request r = request_of(a, blockIdx.z, blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0);
    const int n_rows = r.tokens * group;
    if (row0 >= n_rows) return;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3, before = r.length - r.tokens;  // row v sees before + v / group + 1 slots
    const int reach = min(r.length, max(0, before + min(row0 + ROWS - 1, n_rows - 1) / group + 1));  // slots that any of the rows sees
    const int n_tiles = (reach + ROWS - 1) / ROWS, from = (int)((long long)n_tiles * blockIdx.x / a.n_cuts), to = (int)((long long)n_tiles * (blockIdx.x + 1) / a.n_cuts);
    unsigned x[D / 16][4];
    fetch_queries(a, r, kvh, group, row0, tiles);
    committed();
    arrived<0>();
    __syncthreads();
    load_staying(x, tiles);
    __syncthreads();
    int sees[2];
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
    for (int h = 0; h < 2; ++h) sees[h] = min(r.length, before + (row0 + warp * 16 + h * 8 + g) / group + 1);
    if (from < to) fetch_keys(a, blockIdx.z, r.length, kvh, from * ROWS, tiles);
    committed();
    for (int i = from; i < to; ++i) {
        const unsigned tile = tiles + ((i - from) & 1) * TILE;
        if (i + 1 < to) fetch_keys(a, blockIdx.z, r.length, kvh, (i + 1) * ROWS, tiles + ((i - from + 1) & 1) * TILE);
        committed();
        arrived<1>();
        __syncthreads();
        float s[8][4];
        products(s, x, tile);
        __syncthreads();  // the tile is free
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float top = m[h];
#pragma unroll
            for (int n = 0; n < 8; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float& y = s[n][2 * h + e];
                    y = i * ROWS + n * 8 + 2 * t + e < sees[h] ? y * a.scale_log2 : -INFINITY;
                    top = fmaxf(top, y);
                }
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const float base = top == -INFINITY ? 0.f : top;
            l[h] *= m[h] == -INFINITY ? 1.f : fast_exp2(m[h] - base);  // nothing but zeros and NaN has been added up below -infinity
            m[h] = top;
#pragma unroll
            for (int n = 0; n < 8; ++n) l[h] += fast_exp2(s[n][2 * h] - base) + fast_exp2(s[n][2 * h + 1] - base);
        }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
        const int v = row0 + warp * 16 + h * 8 + g;
        if (t == 0 && v < n_rows) {
            const size_t at = (size_t)(r.first + v / group) * a.heads + kvh * group + v % group;
            if (a.n_cuts == 1) a.rows[at] = make_float2(m[h] == -INFINITY ? 0.f : m[h], l[h] > 0.f ? 1.f / l[h] : (l[h] == 0.f ? 0.f : l[h]));
            else a.cuts[(size_t)blockIdx.x * a.tokens * a.heads + at] = make_float2(m[h], l[h]);
        }
    }
}

__global__ void __launch_bounds__(256) cuts_kernel(const Args a) {
    let_next_kernel_start();
    wait_for_previous_kernels();
    const int n = a.tokens * a.heads, at = blockIdx.x * 256 + threadIdx.x;
    if (at >= n) return;
    float top = -INFINITY, all = 0.f;
    for (int c = 0; c < a.n_cuts; ++c) top = fmaxf(top, a.cuts[(size_t)c * n + at].x);
    for (int c = 0; c < a.n_cuts; ++c) {
        const float2 ml = a.cuts[(size_t)c * n + at];
        all = fmaf(ml.x == -INFINITY ? 0.f : fast_exp2(ml.x - top), ml.y, all);
    }
    a.rows[at] = make_float2(top == -INFINITY ? 0.f : top, all > 0.f ? 1.f / all : (all == 0.f ? 0.f : all));
}

// The second walk: block (tile of slots, key/value head, request).
__global__ void __launch_bounds__(THREADS) slots_kernel(const Args a) {
    extern __shared__ __align__(128) unsigned char smem[];
    float2* sums = reinterpret_cast<float2*>(smem + 2 * TILE);  // [2][ROWS]
    const unsigned tiles = smem_u32(smem);
    let_next_kernel_start();
    wait_for_previous_kernels();
    const int kvh = blockIdx.y, slot0 = blockIdx.x * ROWS, group = a.heads / a.kv_heads;
    const Request r = request_of(a, blockIdx.z, false);
    const int n_rows = r.tokens * group;
    if (slot0 >= r.length || n_rows == 0) return;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3, before = r.length - r.tokens;
    const int from = max(0, slot0 - before) * group / ROWS, to = (n_rows + ROWS - 1) / ROWS;  // token slot0 - before is the first that sees slot slot0
    auto fetch = [&](int i) {
        const int buffer = (i - from) & 1;
        fetch_queries(a, r, kvh, group, i * ROWS, tiles + buffer * TILE);
        if (threadIdx.x < ROWS) {
            const int v = min(i * ROWS + (int)threadIdx.x, n_rows - 1);
            const float2* src = a.rows + (size_t)(r.first + v / group) * a.heads + kvh * group + v % group;
            asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(smem_u32(sums + buffer * ROWS + threadIdx.x)), "l"(src) : "memory");
        }
        committed();
    };
    unsigned x[D / 16][4];
    fetch_keys(a, blockIdx.z, r.length, kvh, slot0, tiles);
    committed();
    arrived<0>();
    __syncthreads();
    load_staying(x, tiles);
    __syncthreads();
    float sum[2] = {0.f, 0.f};
    fetch(from);
    for (int i = from; i < to; ++i) {
        const int buffer = (i - from) & 1;
        if (i + 1 < to) fetch(i + 1);
        else committed();
        arrived<1>();
        __syncthreads();
        float s[8][4];
        products(s, x, tiles + buffer * TILE);
#pragma unroll
        for (int n = 0; n < 8; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int v = i * ROWS + n * 8 + 2 * t + e, token = v / group;
                const float2 ml = sums[buffer * ROWS + n * 8 + 2 * t + e];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const bool sees = token < r.tokens && slot0 + warp * 16 + h * 8 + g <= before + token;
                    const float p = fast_exp2(s[n][2 * h + e] * a.scale_log2 - ml.x) * ml.y;
                    if (sees) sum[h] += p;
                }
            }
        __syncthreads();
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], 1);
        sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], 2);
        const int slot = slot0 + warp * 16 + h * 8 + g;
        if (t == 0 && slot < r.length) a.weights[((size_t)blockIdx.z * a.kv_heads + kvh) * a.capacity + slot] += sum[h];
    }
}
}  // namespace

// Into how many cuts the first walk's slots go: as many as fill the device four times over, of four tiles at least.
static int cuts_for(int requests, int most, int longest, int heads, int kv_heads, int sms) {
    const long long rows = (long long)most * (heads / kv_heads), blocks = (rows + ROWS - 1) / ROWS * kv_heads * requests;
    const long long wanted = 4LL * sms / (blocks ? blocks : 1), most_cuts = (longest + 4 * ROWS - 1) / (4 * ROWS);
    return (int)(wanted < 1 ? 1 : wanted < most_cuts ? wanted : most_cuts);
}
// Bytes of scratch that hb_tally_queries takes.
HB_EXPORT long long hb_tally_queries_scratch(int tokens, int requests, int most, int longest, int heads, int kv_heads, int sms) {
    if (tokens <= 0 || requests <= 0 || most <= 0 || longest <= 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads || sms <= 0) return 0;
    const int cuts = cuts_for(requests, most, longest, heads, kv_heads, sms);
    return 8LL * tokens * heads * (cuts > 1 ? cuts + 1 : 1);
}
// q [tokens, heads * D] with rows q_stride apart, request r's from starts[r] to starts[r + 1] - 1, at most `most`, the last of which stands in its last slot; cache [pages, 2, kv_heads, page_size, D];
// lengths [requests], at most `longest`, which table and capacity hold; weights [requests, kv_heads, capacity].  scratch: hb_tally_queries_scratch bytes on an 8-byte boundary.
HB_EXPORT int hb_tally_queries(const void* q, long long q_stride, int tokens, const void* cache, const int* block_table, int table_width, const int* starts, const int* lengths, int requests, int most,
                               int longest, float* weights, int capacity, int heads, int kv_heads, int page_size, int pages, float scale, int sms, void* scratch, int* status, cudaStream_t stream) {
    if (requests <= 0 || tokens <= 0) return 0;
    if (!q || !cache || !block_table || !starts || !lengths || !weights || !scratch || !status) return HB_BAD_ARGUMENT;
    if (kv_heads <= 0 || heads <= 0 || heads % kv_heads || pages <= 0 || table_width <= 0 || longest <= 0 || most <= 0 || capacity < longest || sms <= 0 || q_stride % 8 || !(scale > 0.f)) return HB_BAD_ARGUMENT;
    if (page_size < 8 || page_size > 64 || (page_size & (page_size - 1))) return HB_UNSUPPORTED_SIZE;
    if ((((uintptr_t)q | (uintptr_t)cache) & 15) || ((uintptr_t)scratch & 7) || (long long)table_width * page_size < longest) return HB_BAD_ARGUMENT;
    const int group = heads / kv_heads;
    if (q_stride > 0x7fffffffLL || (long long)tokens * heads > 0x7fffffffLL - 256 || longest > 0x7fffffff - ROWS || requests > 65535 || kv_heads > 65535) return HB_UNSUPPORTED_SIZE;
    const long long row_blocks = ((long long)most * group + ROWS - 1) / ROWS * kv_heads;
    if (row_blocks > 65535) return HB_UNSUPPORTED_SIZE;
    const int cuts = cuts_for(requests, most, longest, heads, kv_heads, sms), page_shift = __builtin_ctz(page_size);
    float2* rows = (float2*)scratch;
    const Args a{(const bf16*)q, (int)q_stride, (const bf16*)cache, block_table, table_width, starts, lengths, tokens, most, longest, weights, capacity, rows, rows + (size_t)tokens * heads, cuts,
                 heads, kv_heads, page_shift, pages, scale * 1.4426950408889634f, status};
    if (int code = launch_after_previous(rows_kernel, dim3(cuts, (unsigned)row_blocks, requests), dim3(THREADS), 2 * TILE, stream, a)) return code;
    if (cuts > 1)
        if (int code = launch_after_previous(cuts_kernel, dim3((tokens * heads + 255) / 256), dim3(256), 0, stream, a)) return code;
    return launch_after_previous(slots_kernel, dim3((longest + ROWS - 1) / ROWS, kv_heads, requests), dim3(THREADS), 2 * TILE + 2 * ROWS * 8, stream, a);
}
