// Attention of one new token per request over its pages, whose weights are kept: what the token gives each slot, summed over the query heads of a key/value head, is added to
// the slot's weight, by which a cache of a fixed budget is cut back later (evict.cu).  bfloat16 pages, head sizes 64 and 128 (HB_HEAD_DIM), pages of 8 to 64 slots.
//
//     y_hj = q_h . k_j scale log2(e),   m_h = max_j y_hj,   l_h = sum_j 2^(y_hj - m_h),   out_h = sum_j 2^(y_hj - m_h) v_j / l_h
//     weights[j] += sum_h 2^(y_hj - m_h) / l_h                  the token's own slot, the last: = instead of +=, and its position is written beside
//
// A weight is known only when its head's whole row has been seen, so the scores themselves are kept until then: 4 bytes a head and slot beside the 4 d bytes of a key and a value.  (Reading the
// keys a second time would cost 2 d bytes a slot against 8 a head and slot for writing the scores and reading them back.)
//
// Where there is much to do there are two kernels.  The first walks keys and values.  The lengths stay on the device: the requests' slots stand in a line, in tiles of 64, and each of the blocks works out where its
// equal share of the line begins and ends.  A share's part of one request is a piece (m, l and o of its heads); block b's piece of request r has the number b + r, which grows along the line and so is no other one's.
// The second kernel puts the pieces of a request together, in the order of the line, and adds the weights; the scores between the two stay in L2, which keys and values only pass through.
//
// Where there is little, a request and key/value head is a cluster's of one to eight blocks: each walks its share and keeps its scores in shared memory, then they read one another's results there (mapa,
// ld.shared::cluster) and add the weights of their own slots.
//
// In a block one lane of a producer warp per page fetches keys and values by TMA into a ring of stages, and each of four warps takes 16 of a stage's 64 slots for all rows (or for a set's rows: a block has one set of four
// warps, or three).  The products are
// S^T = K Q^T and O^T = V^T P^T (mma.sync m16n8k16): slots and entries stand where the instruction has 16 rows, the few heads of a key/value head where it has 8 columns.  The weights are taken into the second
// product in two parts, rounded to bfloat16 and what that left over: rounded once they would cost the result as much as its own rounding does.
//
// Measured (28 heads over 4 of 128): 64 requests of up to 8,192 slots 150 us for the 823 MB of keys, values and weights (5.5 TB/s), 16 of up to 4,099 26.1 us for 105 MB (4.0 TB/s).  The first kernel alone
// takes 133 us (6.2 TB/s) and 24 (4.4); writing scores is a tenth of it, the second kernel's exposed part the rest.  For heads of 128 a few of the line's registers do not fit (32 bytes spilled for groups of up to 8 heads, 72 of up to 16,
// 20 by three sets); what that costs has not been measured apart.  One token of 14 heads over 2 of 64 at 512 slots: 5.8 us, a start, three dependent trips to memory and the cluster's meeting.
//
// Slots beyond a request's length may hold anything: their scores are replaced and their values read as zeros.  Every wait is bounded; one that runs out sets HB_STATUS_WAIT_EXPIRED and the
// block leaves, once the copies that it has on their way have arrived.
#include <cuda.h>

#include "common.cuh"

#ifndef HB_HEAD_DIM
#define HB_HEAD_DIM 128
#endif
#ifndef HB_WAIT_LIMIT
#define HB_WAIT_LIMIT (1u << 24)
#endif

namespace {
typedef __nv_bfloat16 bf16;
constexpr int D = HB_HEAD_DIM;
static_assert(D == 64 || D == 128, "head sizes 64 and 128");
constexpr int WARPS = 4;  // that compute for the same rows
constexpr int BN = 64;    // slots of a tile
constexpr int TILE = BN * D * 2, PANELS = D / 64;
constexpr unsigned WAIT_LIMIT = HB_WAIT_LIMIT, LAST_WAIT_LIMIT = 1u << 24;
static_assert(BN / WARPS == 16, "a warp takes the 16 rows of a product");

__device__ __forceinline__ unsigned smem_u32(const void* p) { return (unsigned)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void mbar_init(unsigned long long* bar, unsigned count) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(count)); }
__device__ __forceinline__ void mbar_expect_tx(unsigned long long* bar, unsigned bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ void mbar_arrive(unsigned long long* bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory"); }
__device__ __forceinline__ bool mbar_over(unsigned long long* bar, unsigned parity) {
    unsigned done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.b32 %0, 1, 0, p;\n\t}"
        : "=r"(done) : "r"(smem_u32(bar)), "r"(parity) : "memory");
    return done != 0;
}
__device__ __forceinline__ bool mbar_wait(unsigned long long* bar, unsigned parity, volatile int* failed) {
    for (unsigned spin = 0; spin < WAIT_LIMIT; ++spin) {
        if (mbar_over(bar, parity)) return true;
        if ((spin & 1023) == 1023 && *failed) return false;
    }
    return false;
}
// Before a block leaves: what it has set going is done, whatever has become of its other waits.
__device__ __forceinline__ void mbar_last_wait(unsigned long long* bar, unsigned parity) {
    for (unsigned spin = 0; spin < LAST_WAIT_LIMIT; ++spin)
        if (mbar_over(bar, parity)) return;
}
__device__ __forceinline__ void tma_load_2d(void* dst, const CUtensorMap* map, unsigned long long* bar, int x, int y, unsigned long long policy) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1, {%3, %4}], [%2], %5;"
                 ::"r"(smem_u32(dst)), "l"(map), "r"(smem_u32(bar)), "r"(x), "r"(y), "l"(policy) : "memory");
}
__device__ __forceinline__ unsigned turned(unsigned w) {  // an 8 x 8 matrix of 16-bit entries, two of a row a lane, transposed
    unsigned r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(w));
    return r;
}
__device__ __forceinline__ void ldmatrix_x4_trans(unsigned (&r)[4], const void* p) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];\n"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(smem_u32(p)));
}
__device__ __forceinline__ void mma(float (&c)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ unsigned pack(float lo, float hi) {
    unsigned w;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(hi), "f"(lo));
    return w;
}
__device__ __forceinline__ float fast_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// 16-byte chunk cc of slot `key` of a tile as TMA's swizzle has placed it.
__device__ __forceinline__ int tile_at(int key, int cc) { return (cc >> 3) * (BN * 128) + key * 128 + (((cc & 7) ^ (key & 7)) << 4); }

template <int NQ, int SETS>  // eights of rows that four warps have; sets of four warps, each with rows of its own; one more warp fetches
struct Shape {
    static constexpr int ROWS = 8 * NQ, THREADS = 32 * (WARPS * SETS + 1);
    static_assert(SETS == 1 || (NQ == 1 && SETS == 3 && D == 128), "what registers hold");
    static constexpr int BLOCKS = SETS > 1 ? 1 : NQ == 1 ? 3 : 2;  // an SM, by registers
    static constexpr int STAGES = SETS > 1 ? 6 : (D == 128 ? 2 : 4) + (NQ == 1 ? 0 : 1);  // BLOCKS blocks share an SM's memory
    // Where the warps' results meet: COLS entries of every row at a time, a row's LINE floats apart (lanes that store side by side then take different banks).
    static constexpr int COLS = 64 / NQ, LINE = COLS + 4;
    static constexpr int JOIN = WARPS * ROWS * LINE * 4;  // a set
    static constexpr size_t SMEM = 1024 + (size_t)STAGES * 2 * TILE + SETS * (JOIN + 2 * WARPS * ROWS * 4) + 2 * STAGES * 8 + 32 + 4 * SETS;
    static_assert(BLOCKS * (SMEM + 1024) <= 228 * 1024, "an SM's shared memory");
};

struct Args {
    const bf16* q; int q_stride;
    bf16* out; int out_stride;
    const int* block_table; int table_width;
    const int* lengths; int requests;
    int longest, slots;      // the longest that a request may be; the same in whole tiles: a row of scores
    float* scores;           // [requests, heads, slots]
    float* pieces;           // [blocks + requests, heads, D]
    float2* sums;            // [blocks + requests, heads]: (m, l)
    float* weights;          // [requests, kv_heads, capacity]
    int* positions;          // [requests, kv_heads, capacity]
    const int* newest;       // [requests]
    int capacity;
    int heads, kv_heads, page_size, pages;
    int gc, chunks;          // heads of a set, blocks' chunks of a key/value head's group
    int blocks;              // of the first kernel, side by side
    int join_blocks, by_head;  // of the second, a request and key/value head, that put results together: one a head, or one for all of them, a warp each
    int together, kept;      // or 0, or the blocks of a cluster, which has one request and key/value head; slots whose scores each of them keeps
    float scale_log2;
    int* status;
};

// The line of all requests' tiles, as one warp sees it.
__device__ __forceinline__ int length_of(const Args& a, int request) { return min(max(a.lengths[request], 0), a.longest); }
__device__ __forceinline__ int tiles_of(const Args& a, int request) { return (length_of(a, request) + BN - 1) / BN; }
__device__ __forceinline__ long long line_length(const Args& a, int lane) {
    long long total = 0;
    for (int r = lane; r < a.requests; r += 32) total += tiles_of(a, r);
#pragma unroll
    for (int offset = 16; offset > 0; offset >>= 1) total += __shfl_xor_sync(0xffffffffu, total, offset);
    return total;
}
// The last request that begins at or before tile `at` of the line and has tiles, and where it begins.  `at` is below the line's length.
__device__ __forceinline__ int request_at(const Args& a, long long at, long long& begins, int lane) {
    long long before = 0;
    for (int r0 = 0; r0 < a.requests; r0 += 32) {
        const int n = r0 + lane < a.requests ? tiles_of(a, r0 + lane) : 0;
        long long end = n;  // inclusive sum
#pragma unroll
        for (int offset = 1; offset < 32; offset <<= 1) {
            const long long other = __shfl_up_sync(0xffffffffu, end, offset);
            if (lane >= offset) end += other;
        }
        end += before;
        const unsigned beyond = __ballot_sync(0xffffffffu, end > at);
        if (beyond) {
            const int who = __ffs(beyond) - 1;
            begins = __shfl_sync(0xffffffffu, end - n, who);
            return r0 + who;
        }
        before = __shfl_sync(0xffffffffu, end, 31);
    }
    begins = before;
    return a.requests;
}
constexpr int FEW = 4;  // requests of a lane whose tiles stay in registers
// Block b of n takes the tiles from b total / n on; the block that has tile `at`.  n <= total: every block has one.
__device__ __forceinline__ long long share_from(long long b, long long n, long long total) { return b * total / n; }
__device__ __forceinline__ int block_at(long long at, long long n, long long total) { return (int)(((at + 1) * n - 1) / total); }

// A kept row of scores is 4 floats longer than its slots: lanes that store side by side then take different banks.
__host__ __device__ constexpr size_t kept_bytes(int rows, int kept) { return 32 + (size_t)rows * ((kept + 4) * 4 + 8); }
constexpr int MOST_TOGETHER = 8, KEPT_LOADS = 8, MOST_KEPT = KEPT_LOADS * 32 * WARPS;  // slots that a block keeps, KEPT_LOADS of a thread
// The blocks of a cluster.
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }
__device__ __forceinline__ unsigned their(const void* p, int rank) {  // what another block of the cluster has at this place of its shared memory
    unsigned at;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(p)), "r"(rank));
    return at;
}
__device__ __forceinline__ float2 theirs2(const float2* p, int rank) {
    float2 v;
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(their(p, rank)) : "memory");
    return v;
}
__device__ __forceinline__ float4 theirs4(const float* p, int rank) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(their(p, rank)) : "memory");
    return v;
}

// TOGETHER: the blocks of a cluster share one request's slots of one key/value head (all of whose query heads a strip has), keep their scores in shared memory, and end with the result and the weights.
template <int NQ, int SETS, bool TOGETHER>
__global__ void __launch_bounds__(Shape<NQ, SETS>::THREADS, (TOGETHER ? (NQ == 1 ? 2 : 1) : Shape<NQ, SETS>::BLOCKS)) attention_tallied_kernel(const __grid_constant__ CUtensorMap kv_map, const Args a) {
    typedef Shape<NQ, SETS> S;
    constexpr int ROWS = S::ROWS, PRODUCER = WARPS * SETS;
    static_assert(SETS == 1 || !TOGETHER, "a cluster's blocks have one set");
    extern __shared__ unsigned char smem_raw[];
    unsigned char* ring = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    const int tid = threadIdx.x, lane = tid & 31, set = threadIdx.x / (32 * WARPS), warp = (threadIdx.x >> 5) - (SETS > 1 ? set * WARPS : 0);  // of its set; the producer's is PRODUCER or, behind other sets, 0
    const bool producer = (tid >> 5) == PRODUCER;
    float* of_sets = reinterpret_cast<float*>(ring + (size_t)S::STAGES * 2 * TILE);
    float* join = of_sets + (producer ? 0 : set) * (S::JOIN / 4 + 2 * WARPS * ROWS);  // [WARPS][ROWS][LINE]
    float* tops = join + S::JOIN / 4;                                                   // [WARPS][ROWS]: maxima
    float* parts = tops + WARPS * ROWS;                                                 // [WARPS][ROWS]: sums
    unsigned long long* full = reinterpret_cast<unsigned long long*>(of_sets + SETS * (S::JOIN / 4 + 2 * WARPS * ROWS));
    unsigned long long* empty = full + S::STAGES;
    volatile int* failed = reinterpret_cast<volatile int*>(empty + S::STAGES);
    int* share = const_cast<int*>(failed) + 1;  // first request, its first tile here, tiles in all
    volatile int* lost = failed + 4 + (producer ? 0 : set);  // a computing warp of the set has given up
    [[maybe_unused]] float2* factors = reinterpret_cast<float2*>((reinterpret_cast<uintptr_t>(share + 3 + SETS) + 15) & ~(uintptr_t)15);  // TOGETHER: [ROWS]: (m, 1 / l) of the request's rows
    [[maybe_unused]] float* kept = reinterpret_cast<float*>(factors + ROWS);                                                   // [ROWS][a.kept + 4]

    if (tid == 0) {
        for (int s = 0; s < S::STAGES; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], WARPS * SETS); }
        *failed = 0;
        for (int k = 0; k < SETS; ++k) lost[k] = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (producer && lane == 0) asm volatile("prefetch.tensormap [%0];" ::"l"(&kv_map) : "memory");
    wait_for_previous_kernels();
    let_next_kernel_start();  // behind the wait: the second kernel reads what came before this one without waiting for this one
    if (!TOGETHER && producer) {
        int request = 0, tile = 0, tiles = 0;
        if (a.requests <= 32 * FEW && (long long)a.requests * a.slots / BN < 0x7fffffffLL) {
            // the requests' tiles stay in registers, and everything fits 32 bits
            int n[FEW], sum = 0;
#pragma unroll
            for (int k = 0; k < FEW; ++k) n[k] = 32 * k + lane < a.requests ? tiles_of(a, 32 * k + lane) : 0;
#pragma unroll
            for (int k = 0; k < FEW; ++k) sum += n[k];
            const unsigned total = __reduce_add_sync(0xffffffffu, (unsigned)sum), blocks = min((unsigned)a.blocks, total), b = blockIdx.x;
            if (b < blocks) {
                const unsigned each = total / blocks, rest = total - each * blocks;  // floor(b total / blocks) = b each + floor(b rest / blocks); blocks are a few an SM, below 2^16
                const int from = (int)(b * each + b * rest / blocks), to = (int)((b + 1) * each + (b + 1) * rest / blocks);
                int before = 0;
#pragma unroll
                for (int k = 0; k < FEW; ++k) {
                    int end = n[k];  // inclusive sum
#pragma unroll
                    for (int offset = 1; offset < 32; offset <<= 1) {
                        const int other = __shfl_up_sync(0xffffffffu, end, offset);
                        if (lane >= offset) end += other;
                    }
                    const unsigned beyond = __ballot_sync(0xffffffffu, before + end > from && before <= from);
                    if (beyond) {
                        const int who = __ffs(beyond) - 1;
                        request = 32 * k + who, tile = from - before - __shfl_sync(0xffffffffu, end - n[k], who), tiles = to - from;
                        break;
                    }
                    before += __shfl_sync(0xffffffffu, end, 31);
                }
            }
        } else {
            const long long total = line_length(a, lane), n = min((long long)a.blocks, total);
            if ((long long)blockIdx.x < n) {
                const long long from = share_from(blockIdx.x, n, total), to = share_from(blockIdx.x + 1, n, total);
                long long begins;
                request = request_at(a, from, begins, lane);
                tile = (int)(from - begins), tiles = (int)(to - from);
            }
        }
        if (lane == 0) share[0] = request, share[1] = tile, share[2] = tiles;
    }
    __syncthreads();
    const int kvh = blockIdx.y / a.chunks, chunk = blockIdx.y - kvh * a.chunks;
    const int group = a.heads / a.kv_heads, head0 = (SETS > 1 ? chunk * SETS + set : chunk) * a.gc, first_head = kvh * group + head0, heads_here = max(0, min(a.gc, group - head0));  // (those of the producer are no one's)
    int request, tile, left, stage = 0;  // the ring runs on across the block's requests
    [[maybe_unused]] int rank = 0;
    if constexpr (TOGETHER) {
        request = blockIdx.x / a.together, rank = blockIdx.x % a.together;
        const long long n = tiles_of(a, request);
        tile = (int)(n * rank / a.together), left = (int)(n * (rank + 1) / a.together) - tile;
        if (tid == 0 && rank == 0 && kvh == 0 && (a.lengths[request] > a.longest || a.lengths[request] < 0)) atomicOr(a.status, HB_STATUS_BAD_POSITION);
    } else {
        request = share[0], tile = share[1], left = share[2];
    }

    if (producer) {
        // ------------------------------------------------------------------ producer (the whole warp)
        const int shift = 31 - __clz(a.page_size), pages_per_tile = BN >> shift, tiles_per_look = 32 / pages_per_tile;
        constexpr int OPS_PER_PAGE = 2 * PANELS;
        const int ops = pages_per_tile * OPS_PER_PAGE;
        const unsigned page_bytes = 2u * a.page_size * D * 2;
        unsigned long long once;  // keys and values pass through L2, where the scores are to stay until the second kernel reads them
        asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(once));
        int ok = 1;
        for (; left > 0 && ok; ++request, tile = 0) {
            const int length = length_of(a, request), here = min(left, (length + BN - 1) / BN - tile);
            const int* table = a.block_table + (size_t)request * a.table_width;
            int looked = -1;
            for (int it = 0; it < here; ++it, ++stage) {
                const int s = stage % S::STAGES, round = stage / S::STAGES, base = (tile + it) * BN;
                if (it % tiles_per_look == 0) {  // a page number per lane, for the next tiles
                    const int block = (base >> shift) + lane;
                    looked = block < a.table_width ? table[block] : -1;
                }
                if (lane == 0) ok = mbar_wait(&empty[s], (round & 1) ^ 1, failed) ? 1 : 0;
                ok = __shfl_sync(0xffffffffu, ok, 0);
                if (!ok) {
                    if (lane == 0) { *failed = 1; atomicOr(a.status, HB_STATUS_WAIT_EXPIRED | HB_STATUS_IN_ATTENTION_TALLIED); }
                    break;
                }
                int page = __shfl_sync(0xffffffffu, looked, (it % tiles_per_look) * pages_per_tile + (lane & (pages_per_tile - 1)));
                const bool wanted = lane < pages_per_tile && base + lane * a.page_size < length;
                if (wanted && (page < 0 || page >= a.pages)) atomicOr(a.status, HB_STATUS_BAD_PAGE);
                if (!wanted || page >= a.pages) page = -1;
                const unsigned valid = __popc(__ballot_sync(0xffffffffu, page >= 0));
                if (lane == 0) {
                    if (valid) mbar_expect_tx(&full[s], valid * page_bytes); else mbar_arrive(&full[s]);
                }
                __syncwarp();
                unsigned char* tiles = ring + (size_t)s * 2 * TILE;
                for (int op0 = 0; op0 < ops; op0 += 32) {
                    const int op = op0 + lane;
                    const int p = min(op, ops - 1) / OPS_PER_PAGE, rest = op % OPS_PER_PAGE, which = rest / PANELS, panel = rest - which * PANELS;
                    const int from = __shfl_sync(0xffffffffu, page, p);
                    if (op < ops && from >= 0)
                        tma_load_2d(tiles + which * TILE + panel * (BN * 128) + p * a.page_size * 128, &kv_map, &full[s], panel * 64, ((from * 2 + which) * a.kv_heads + kvh) * a.page_size, once);
                }
            }
            left -= here;
        }
        if (lane == 0)
            for (int k = max(0, stage - S::STAGES); k < stage; ++k) mbar_last_wait(&full[k % S::STAGES], (k / S::STAGES) & 1);
        __syncwarp();
        if constexpr (TOGETHER) cluster_arrive(), cluster_wait(), cluster_arrive(), cluster_wait();
        return;
    }
    // ---------------------------------------------------------------------- consumers
    const int t = lane & 3, g = lane >> 2;
    auto meet = [&] { asm volatile("bar.sync %0, %1;" ::"r"(SETS > 1 ? 1 + set : 1), "n"(32 * WARPS) : "memory"); };  // the set's warps
    constexpr int LANES_PER_ROW = S::COLS / 16;
    const int store_row = lane / LANES_PER_ROW, store_col = warp * (S::COLS / 4) + lane % LANES_PER_ROW * 4;  // what this lane stores of every COLS entries
    const bool stores = store_row < heads_here;
    [[maybe_unused]] float* rows_here = reinterpret_cast<float*>(ring);                    // TOGETHER: [ROWS][D], what the block brings; the ring has been read to its end by then
    [[maybe_unused]] float2* sums_here = reinterpret_cast<float2*>(rows_here + ROWS * D);  // [ROWS]
    static_assert(ROWS * (D * 4 + 8) <= S::STAGES * 2 * TILE, "a cluster's results lie where the ring was");
    bool once = TOGETHER;  // a block of a cluster has its part in it without slots, too
    for (; left > 0 || once; ++request, tile = 0) {
        once = false;
        const int length = length_of(a, request), here = min(left, (length + BN - 1) / BN - tile), start = tile * BN;
        left -= here;
        // Q's fragments: a lane's 16-byte chunk t + 4 j of a key feeds products 2 j and 2 j + 1, four of its entries each, so a query's entries stand in the fragments likewise.
        unsigned qf[NQ][D / 16][2];
#pragma unroll
        for (int q = 0; q < NQ; ++q) {
            const int head = q * 8 + g;
            const bf16* src = a.q + (size_t)request * a.q_stride + (size_t)(first_head + (head < heads_here ? head : 0)) * D;
#pragma unroll
            for (int j = 0; j < D / 32; ++j) {
                const uint4 raw = head < heads_here ? *reinterpret_cast<const uint4*>(src + (t + 4 * j) * 8) : make_uint4(0, 0, 0, 0);
                qf[q][2 * j][0] = raw.x, qf[q][2 * j][1] = raw.y, qf[q][2 * j + 1][0] = raw.z, qf[q][2 * j + 1][1] = raw.w;
            }
        }
        float* scores[NQ][2];  // of columns 2 t and 2 t + 1
#pragma unroll
        for (int q = 0; q < NQ; ++q)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int head = q * 8 + 2 * t + e;
                if constexpr (TOGETHER) scores[q][e] = kept + (size_t)head * (a.kept + 4) - start;  // all rows: those that are no one's are not added up
                else scores[q][e] = head < heads_here ? a.scores + ((size_t)request * a.heads + first_head + head) * a.slots : nullptr;
            }
        float m[NQ][2], l[NQ][2], o[NQ][D / 16][4];
#pragma unroll
        for (int q = 0; q < NQ; ++q) {
            m[q][0] = m[q][1] = -INFINITY, l[q][0] = l[q][1] = 0.f;
#pragma unroll
            for (int i = 0; i < D / 16; ++i) o[q][i][0] = o[q][i][1] = o[q][i][2] = o[q][i][3] = 0.f;
        }
        for (int it = 0; it < here; ++it, ++stage) {
            const int s = stage % S::STAGES, round = stage / S::STAGES;
            if (!mbar_wait(&full[s], round & 1, failed)) {
                *failed = 1, *lost = 1;
                atomicOr(a.status, HB_STATUS_WAIT_EXPIRED | HB_STATUS_IN_ATTENTION_TALLIED);
                break;
            }
            const unsigned char* ks = ring + (size_t)s * 2 * TILE;
            const unsigned char* vs = ks + TILE;
            const int key0 = warp * 16, pos0 = start + it * BN + key0;  // this warp's slots
            if (pos0 < length) {
                const bool whole = pos0 + 16 <= length;
                float sc[NQ][4];  // of slots g and g + 8 and columns 2 t and 2 t + 1: [(slot, column)]
#pragma unroll
                for (int q = 0; q < NQ; ++q) sc[q][0] = sc[q][1] = sc[q][2] = sc[q][3] = 0.f;
#pragma unroll
                for (int j = 0; j < D / 32; ++j) {
                    const uint4 k0 = *reinterpret_cast<const uint4*>(ks + tile_at(key0 + g, t + 4 * j)), k1 = *reinterpret_cast<const uint4*>(ks + tile_at(key0 + 8 + g, t + 4 * j));
#pragma unroll
                    for (int q = 0; q < NQ; ++q) {
                        mma(sc[q], k0.x, k1.x, k0.y, k1.y, qf[q][2 * j][0], qf[q][2 * j][1]);
                        mma(sc[q], k0.z, k1.z, k0.w, k1.w, qf[q][2 * j + 1][0], qf[q][2 * j + 1][1]);
                    }
                }
                bool rescale = false;
                float alpha[NQ][2];
#pragma unroll
                for (int q = 0; q < NQ; ++q) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        sc[q][e] *= a.scale_log2;
                        const int pos = pos0 + (e >> 1) * 8 + g;
                        if (!whole && pos >= length) sc[q][e] = -INFINITY;
                        else if (TOGETHER || scores[q][e & 1]) scores[q][e & 1][pos] = sc[q][e];
                    }
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float mx = fmaxf(sc[q][e], sc[q][2 + e]);
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
                        const float m_new = fmaxf(m[q][e], mx);
                        alpha[q][e] = m_new == -INFINITY ? 1.f : fast_exp2(m[q][e] - m_new);
                        m[q][e] = m_new;
                        rescale |= alpha[q][e] != 1.f;
                        const float base = m_new == -INFINITY ? 0.f : m_new;
                        l[q][e] *= alpha[q][e];
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            sc[q][2 * h + e] = fast_exp2(sc[q][2 * h + e] - base);
                            l[q][e] += sc[q][2 * h + e];  // of this lane's slots; the lanes are added up at the end
                        }
                    }
                }
                if (__any_sync(0xffffffffu, rescale)) {
#pragma unroll
                    for (int q = 0; q < NQ; ++q)
#pragma unroll
                        for (int i = 0; i < D / 16; ++i) o[q][i][0] *= alpha[q][0], o[q][i][1] *= alpha[q][1], o[q][i][2] *= alpha[q][0], o[q][i][3] *= alpha[q][1];
                }
                // Values beyond the length read as zeros, whatever their slots hold.  A fragment register holds slots 2 t and 2 t + 1 in its halves.
                unsigned keep[2] = {0xffffffffu, 0xffffffffu};
                if (!whole) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int pos = pos0 + h * 8 + t * 2;
                        keep[h] = (pos < length ? 0xffffu : 0u) | (pos + 1 < length ? 0xffff0000u : 0u);
                    }
                }
                unsigned pf[NQ][2], pr[NQ][2];  // the weights, and what they lose by rounding, as weights of their own
#pragma unroll
                for (int q = 0; q < NQ; ++q)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const float p0 = sc[q][2 * h], p1 = sc[q][2 * h + 1];
                        const unsigned w = pack(p0, p1);
                        pf[q][h] = turned(w);
                        pr[q][h] = turned(pack(p0 - __uint_as_float(w << 16), p1 - __uint_as_float(w & 0xffff0000u)));
                    }
#pragma unroll
                for (int c = 0; c < D / 8; c += 2) {
                    unsigned b[4];
                    ldmatrix_x4_trans(b, vs + tile_at(key0 + (lane & 15), c + (lane >> 4)));
                    if (!whole) b[0] &= keep[0], b[1] &= keep[1], b[2] &= keep[0], b[3] &= keep[1];
#pragma unroll
                    for (int q = 0; q < NQ; ++q) {
                        mma(o[q][c / 2], b[0], b[2], b[1], b[3], pf[q][0], pf[q][1]);
                        mma(o[q][c / 2], b[0], b[2], b[1], b[3], pr[q][0], pr[q][1]);
                    }
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&empty[s]);
        }
        // The warps' results meet: every warp brings its sums to the largest maximum and lays COLS entries of its rows down, then takes a quarter of them, adds up the four
        // warps' in their order, and stores.
#pragma unroll
        for (int q = 0; q < NQ; ++q)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                l[q][e] += __shfl_xor_sync(0xffffffffu, l[q][e], 4);
                l[q][e] += __shfl_xor_sync(0xffffffffu, l[q][e], 8);
                l[q][e] += __shfl_xor_sync(0xffffffffu, l[q][e], 16);
                if (g == 0) tops[warp * ROWS + q * 8 + 2 * t + e] = m[q][e], parts[warp * ROWS + q * 8 + 2 * t + e] = l[q][e];
            }
        meet();
        if (*lost && !TOGETHER) break;  // all four warps see the same: they set it before they come here only.  (A cluster's blocks leave together, whatever it is that they join.)
        float f[NQ][2];
#pragma unroll
        for (int q = 0; q < NQ; ++q)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int row = q * 8 + 2 * t + e;
                const float top = fmaxf(fmaxf(tops[row], tops[ROWS + row]), fmaxf(tops[2 * ROWS + row], tops[3 * ROWS + row]));
                f[q][e] = m[q][e] == -INFINITY ? 0.f : fast_exp2(m[q][e] - top);
            }
        float top = -INFINITY, all = 0.f;  // of the row that this lane stores
#pragma unroll
        for (int w = 0; w < WARPS; ++w) top = fmaxf(top, tops[w * ROWS + store_row]);
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            const float mw = tops[w * ROWS + store_row];
            all = fmaf(mw == -INFINITY ? 0.f : fast_exp2(mw - top), parts[w * ROWS + store_row], all);
        }
        const size_t slot = ((size_t)blockIdx.x + request) * a.heads + first_head + store_row;
        if (!TOGETHER && stores && store_col == 0) a.sums[slot] = make_float2(top, all);
        if (TOGETHER && store_col == 0) sums_here[store_row] = make_float2(top, all);
#pragma unroll
        for (int col = 0; col < D; col += S::COLS) {
#pragma unroll
            for (int q = 0; q < NQ; ++q)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float* dst = join + (warp * ROWS + q * 8 + 2 * t + e) * S::LINE;
#pragma unroll
                    for (int i = 0; i < S::COLS / 16; ++i) dst[16 * i + g] = o[q][col / 16 + i][e] * f[q][e], dst[16 * i + 8 + g] = o[q][col / 16 + i][2 + e] * f[q][e];
                }
            meet();
            if (stores) {
                float sum[4];
                load4(join + store_row * S::LINE + store_col, sum);
#pragma unroll
                for (int w = 1; w < WARPS; ++w) {
                    float more[4];
                    load4(join + (w * ROWS + store_row) * S::LINE + store_col, more);
#pragma unroll
                    for (int i = 0; i < 4; ++i) sum[i] += more[i];
                }
                if (TOGETHER) store4(rows_here + store_row * D + col + store_col, sum);
                else store4(a.pieces + slot * D + col + store_col, sum);
            }
            meet();
        }
        if constexpr (TOGETHER) {
            // the old weights are on their way while the blocks meet
            float* weights = a.weights + ((size_t)request * a.kv_heads + kvh) * a.capacity + start;
            const int mine = max(0, min(here * BN, length - start));  // slots of this block
            float old[KEPT_LOADS];
#pragma unroll
            for (int k = 0; k < KEPT_LOADS; ++k) {
                const int at = k * 32 * WARPS + tid;
                old[k] = at < mine && start + at != length - 1 ? weights[at] : 0.f;  // the token's own slot enters the tally
            }
            cluster_arrive(), cluster_wait();
            float2 ml[MOST_TOGETHER];
            auto joined = [&](int row) {  // (m, 1 / l) over the blocks
                float above = -INFINITY, sum = 0.f;
#pragma unroll
                for (int r = 0; r < MOST_TOGETHER; ++r) ml[r] = theirs2(sums_here + row, min(r, a.together - 1)), above = fmaxf(above, ml[r].x);
#pragma unroll
                for (int r = 0; r < MOST_TOGETHER; ++r) {
                    ml[r].x = ml[r].x == -INFINITY ? 0.f : fast_exp2(ml[r].x - above);  // the block's share of it
                    if (r < a.together) sum = fmaf(ml[r].x, ml[r].y, sum);
                }
                return make_float2(above == -INFINITY ? 0.f : above, sum > 0.f ? 1.f / sum : (sum == 0.f ? 0.f : sum));  // a row that sees nothing is zeros; a NaN stays one
            };
            if (tid < ROWS) factors[tid] = joined(tid);
            for (int at = rank * 32 * WARPS + tid; at < heads_here * (D / 4); at += a.together * 32 * WARPS) {
                const int row = at / (D / 4), col = at % (D / 4) * 4;
                const float2 f = joined(row);
                float sum[4] = {0.f, 0.f, 0.f, 0.f};
                float4 part[MOST_TOGETHER];
#pragma unroll
                for (int r = 0; r < MOST_TOGETHER; ++r) part[r] = theirs4(rows_here + row * D + col, min(r, a.together - 1));
#pragma unroll
                for (int r = 0; r < MOST_TOGETHER; ++r) {
                    if (r >= a.together) break;
                    sum[0] = fmaf(ml[r].x, part[r].x, sum[0]), sum[1] = fmaf(ml[r].x, part[r].y, sum[1]), sum[2] = fmaf(ml[r].x, part[r].z, sum[2]), sum[3] = fmaf(ml[r].x, part[r].w, sum[3]);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) sum[i] *= f.y;
                store4(a.out + (size_t)request * a.out_stride + (size_t)(first_head + row) * D + col, sum);
            }
            cluster_arrive();  // nothing of the others is read any more
            meet();
#pragma unroll
            for (int k = 0; k < KEPT_LOADS; ++k) {
                const int at = k * 32 * WARPS + tid;
                if (at >= mine) break;
                float given = 0.f;
                for (int row = 0; row < heads_here; ++row) {
                    const float2 f = factors[row];
                    given = fmaf(fast_exp2(kept[(size_t)row * (a.kept + 4) + at] - f.x), f.y, given);
                }
                weights[at] = old[k] + given;
                if (start + at == length - 1) a.positions[((size_t)request * a.kv_heads + kvh) * a.capacity + length - 1] = a.newest[request];
            }
            cluster_wait();
        }
    }
}

// The second kernel: block x of a (key/value head, request) adds the weights of SPAN slots, four of them a thread; behind those one block puts the request's results together, a warp a head, or, where pieces are many, a block a head.  What the first kernel has not written is
// read while that one still runs; behind it the scores are on their way while each block brings the pieces' sums together.
constexpr int ADD_THREADS = 256, SPAN = 4 * ADD_THREADS, HEADS = 8;  // heads at a time
__global__ void __launch_bounds__(ADD_THREADS, 3) tally_kernel(const Args a) {
    __shared__ float2 heads_sum[HEADS];  // (m, 1 / l) of the heads
    __shared__ int range[2];             // the request's first block of the first kernel, and its pieces
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, kvh = blockIdx.y, request = blockIdx.z, group = a.heads / a.kv_heads;
    const int head = (int)blockIdx.x - (int)(gridDim.x - a.join_blocks);  // that this block puts together (or all of them), or below 0
    const bool puts_together = head >= 0;
    const int length = length_of(a, request), slot0 = blockIdx.x * SPAN + 4 * tid;
    let_next_kernel_start();
    if (!puts_together && (int)blockIdx.x * SPAN >= length) return;
    if (length && warp == 0) {
        const long long total = line_length(a, lane), n = min((long long)a.blocks, total);
        long long begins = 0;
        for (int r = lane; r < request; r += 32) begins += tiles_of(a, r);
#pragma unroll
        for (int offset = 16; offset > 0; offset >>= 1) begins += __shfl_xor_sync(0xffffffffu, begins, offset);
        const int b0 = block_at(begins, n, total), b1 = block_at(begins + (length + BN - 1) / BN - 1, n, total);
        if (lane == 0) range[0] = b0, range[1] = b1 - b0 + 1;
    }
    float* weights = a.weights + ((size_t)request * a.kv_heads + kvh) * a.capacity + slot0;
    const bool whole = slot0 + 4 <= length && ((uintptr_t)weights & 15) == 0;
    float added[4] = {0.f, 0.f, 0.f, 0.f}, given[4] = {0.f, 0.f, 0.f, 0.f};
    if (!puts_together) {
        if (whole) {
            load4(weights, added);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (slot0 + e < length) added[e] = weights[e];
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (slot0 + e == length - 1) added[e] = 0.f;  // the token's own slot enters the tally
    }
    if (tid == 0 && head == 0 && kvh == 0 && (a.lengths[request] > a.longest || a.lengths[request] < 0)) atomicOr(a.status, HB_STATUS_BAD_POSITION);
    __syncthreads();
    const int count = length ? range[1] : 0;
    const size_t piece0 = ((size_t)(length ? range[0] : 0) + request) * a.heads + (size_t)kvh * group;  // of the group's first head
    const float* scores = a.scores + ((size_t)request * a.heads + (size_t)kvh * group) * a.slots + slot0;
    const bool mine = !puts_together && slot0 < length;  // a row of scores has whole tiles
    wait_for_previous_kernels();
    auto joined = [&](const float2* sums) {  // (m, 1 / l) of a head, by one warp
        float top = -INFINITY, all = 0.f;
        for (int p = lane; p < count; p += 32) {
            const float2 ml = sums[(size_t)p * a.heads];
            const float above = fmaxf(top, ml.x);
            all = above == -INFINITY ? all + ml.y : fmaf(ml.x == -INFINITY ? 0.f : fast_exp2(ml.x - above), ml.y, all * (top == -INFINITY ? 0.f : fast_exp2(top - above)));
            top = above;
        }
        const float above = warp_max(top);
        all = warp_sum(top == -INFINITY ? all : all * fast_exp2(top - above));
        return make_float2(above == -INFINITY ? 0.f : above, all > 0.f ? 1.f / all : (all == 0.f ? 0.f : all));
    };
    if (puts_together && !a.by_head) {
        constexpr int TOGETHER = 4;  // pieces that are on their way together
        for (int h = warp; h < group; h += ADD_THREADS / 32) {
            const size_t slot0 = piece0 + h;
            const float2 ml = joined(a.sums + slot0);
            if (lane >= D / 4) continue;
            float sum[4] = {0.f, 0.f, 0.f, 0.f};
            for (int p0 = 0; p0 < count; p0 += TOGETHER) {
                float m[TOGETHER], part[TOGETHER][4];
#pragma unroll
                for (int k = 0; k < TOGETHER; ++k) {
                    const size_t slot = slot0 + (size_t)min(p0 + k, count - 1) * a.heads;
                    m[k] = a.sums[slot].x;
                    load4(a.pieces + slot * D + 4 * lane, part[k]);
                }
#pragma unroll
                for (int k = 0; k < TOGETHER; ++k) {
                    if (p0 + k >= count) break;
                    const float f = m[k] == -INFINITY ? 0.f : fast_exp2(m[k] - ml.x);
#pragma unroll
                    for (int e = 0; e < 4; ++e) sum[e] = fmaf(f, part[k][e], sum[e]);
                }
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) sum[e] *= ml.y;
            store4(a.out + (size_t)request * a.out_stride + ((size_t)kvh * group + h) * D + 4 * lane, sum);
        }
        return;
    }
    if (puts_together) {
        // a team of threads has the head's entries, four each, and every TEAMS-th piece; the teams' sums are added up in their order
        constexpr int TEAM = D / 4, TEAMS = ADD_THREADS / TEAM, TOGETHER = 4;  // pieces of a team that are on their way together
        __shared__ __align__(16) float parts[TEAMS][D];
        const int team = tid / TEAM, col = tid % TEAM * 4;
        const size_t slot0 = piece0 + head;
        const float2 ml = joined(a.sums + slot0);  // every warp for itself
        float sum[4] = {0.f, 0.f, 0.f, 0.f};
        for (int p0 = team; p0 < count; p0 += TEAMS * TOGETHER) {
            float m[TOGETHER], part[TOGETHER][4];
#pragma unroll
            for (int k = 0; k < TOGETHER; ++k) {
                const size_t slot = slot0 + (size_t)min(p0 + k * TEAMS, count - 1) * a.heads;
                m[k] = a.sums[slot].x;
                load4(a.pieces + slot * D + col, part[k]);
            }
#pragma unroll
            for (int k = 0; k < TOGETHER; ++k) {
                if (p0 + k * TEAMS >= count) break;
                const float f = m[k] == -INFINITY ? 0.f : fast_exp2(m[k] - ml.x);
#pragma unroll
                for (int e = 0; e < 4; ++e) sum[e] = fmaf(f, part[k][e], sum[e]);
            }
        }
        store4(&parts[team][col], sum);
        __syncthreads();
        if (team == 0) {
#pragma unroll
            for (int t = 1; t < TEAMS; ++t) {
                float more[4];
                load4(&parts[t][col], more);
#pragma unroll
                for (int e = 0; e < 4; ++e) sum[e] += more[e];
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) sum[e] *= ml.y;
            store4(a.out + (size_t)request * a.out_stride + ((size_t)kvh * group + head) * D + col, sum);
        }
        return;
    }
    for (int g0 = 0; g0 < group; g0 += HEADS) {
        const int here = min(HEADS, group - g0);
        float y[HEADS][4];
        if (mine) {
#pragma unroll
            for (int h = 0; h < HEADS; ++h)
                if (h < here) load4(scores + (size_t)(g0 + h) * a.slots, y[h]);
        }
        if (warp < here) {
            const float2 ml = joined(a.sums + piece0 + g0 + warp);
            if (lane == 0) heads_sum[warp] = ml;
        }
        __syncthreads();
        if (mine) {
#pragma unroll
            for (int h = 0; h < HEADS; ++h) {
                if (h >= here) break;
                const float2 ml = heads_sum[h];
#pragma unroll
                for (int e = 0; e < 4; ++e) given[e] = fmaf(fast_exp2(y[h][e] - ml.x), ml.y, given[e]);
            }
        }
        __syncthreads();
    }
    if (!mine) return;
#pragma unroll
    for (int e = 0; e < 4; ++e) added[e] += given[e];
    if (whole) {
        store4(weights, added);
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (slot0 + e < length) weights[e] = added[e];
    }
    if (slot0 <= length - 1 && length - 1 < slot0 + 4) a.positions[((size_t)request * a.kv_heads + kvh) * a.capacity + length - 1] = a.newest[request];
}

typedef CUresult (*EncodeTiled)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiled encode_tiled() {
    static EncodeTiled fn = [] {
        void* found = nullptr;
        cudaDriverEntryPointQueryResult result;
        const bool ok = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &found, cudaEnableDefault, &result) == cudaSuccess && result == cudaDriverEntryPointSuccess;
        return ok ? reinterpret_cast<EncodeTiled>(found) : nullptr;
    }();
    return fn;
}
// The cache as a matrix [pages * 2 * kv_heads * page_size, D], fetched in boxes of a page's rows and 64 entries.
int cache_map(CUtensorMap* map, const void* cache, const Args& a) {
    EncodeTiled encode = encode_tiled();
    if (!encode) return HB_BAD_ARGUMENT;
    const cuuint64_t dims[2] = {(cuuint64_t)D, (cuuint64_t)a.pages * 2 * a.kv_heads * a.page_size};
    const cuuint64_t strides[1] = {(cuuint64_t)D * 2};
    const cuuint32_t box[2] = {64, (cuuint32_t)a.page_size};
    const cuuint32_t elem[2] = {1, 1};
    return encode(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(cache), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS ? 0 : HB_BAD_ARGUMENT;
}
// launch_after_previous with clusters of `together` blocks along x.
template <typename... Params, typename... Values>
int launch_clusters(void (*kernel)(Params...), int together, dim3 grid, dim3 block, size_t shared_bytes, cudaStream_t stream, Values&&... values) {
    cudaLaunchConfig_t config = {};
    config.gridDim = grid, config.blockDim = block, config.dynamicSmemBytes = shared_bytes, config.stream = stream;
    cudaLaunchAttribute attributes[2];
    attributes[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attributes[0].val.programmaticStreamSerializationAllowed = overlap_launches() ? 1 : 0;
    attributes[1].id = cudaLaunchAttributeClusterDimension;
    attributes[1].val.clusterDim = {(unsigned)together, 1, 1};
    config.attrs = attributes, config.numAttrs = 2;
    return (int)cudaLaunchKernelEx(&config, kernel, static_cast<Params>(values)...);
}
template <int NQ, int SETS>
int launch_strips(const Args& a, const CUtensorMap& map, cudaStream_t stream) {
    typedef Shape<NQ, SETS> S;
    if constexpr (SETS == 1) if (a.together) {
        const auto kernel = attention_tallied_kernel<NQ, 1, true>;
        constexpr size_t most = S::SMEM + kept_bytes(S::ROWS, MOST_KEPT);
        static_assert(most <= 227 * 1024, "a block's shared memory");
        static std::atomic<unsigned long long> allowed{0};
        if (const cudaError_t error = allow_shared((const void*)kernel, most, allowed)) return (int)error;
        return launch_clusters(kernel, a.together, dim3(a.requests * a.together, a.kv_heads), dim3(S::THREADS), S::SMEM + kept_bytes(S::ROWS, a.kept), stream, map, a);
    }
    const auto kernel = attention_tallied_kernel<NQ, SETS, false>;
    static std::atomic<unsigned long long> allowed{0};
    if (const cudaError_t error = allow_shared((const void*)kernel, S::SMEM, allowed)) return (int)error;
    return launch_after_previous(kernel, dim3(a.blocks, a.kv_heads * a.chunks), dim3(S::THREADS), S::SMEM, stream, map, a);
}
template <int DIM>
int launch_first(int heads, int sets, const Args& a, const CUtensorMap& map, cudaStream_t stream) {
    if constexpr (DIM == 128) {
        if (sets == 3) return launch_strips<1, 3>(a, map, stream);
    }
    return heads <= 8 ? launch_strips<1, 1>(a, map, stream) : launch_strips<2, 1>(a, map, stream);
}
}  // namespace

// Whether the second kernel has a block for each head.
static bool few_heads(int requests, int heads, int sms) { return (long long)requests * heads <= 2LL * sms; }
// The blocks of a cluster that keeps its scores, and how many slots each keeps; or 0, where there are two kernels.  A cluster has one request and key/value head, so its work is as long as the longest request; the line's is
// equal for all blocks but costs a second kernel.  Clusters are the faster ones for few tiles of 64 slots, in all or a block, and for more of them where the second kernel has no
// block for each head, as long as all of them are on the device at once (us, clusters / line, 28 heads over 4 of 128: one request at 512 slots 6.5 / 6.2 and a launch less for the host, at 2,048 10.1 / 7.4, at 8,192 24.3 / 14.9; 16 at 256 7.3 / 8.5, at 512 9.1 / 10.8, at 2,048
// 18.9 / 18.4; 64 at 256 11.7 / 15.0; 16 heads over 1: eight at 1,024 8.8 / 10.4, one at 4,099 16.4 / 9.7).  As many blocks a cluster as leave room, with some to spare: two are on an SM, one of more than eight heads, and
// few clusters of eight fit a group of SMs (eight requests at 512: of eight blocks 10.0, of four 8.0).
static int together_for(int requests, int longest, int heads, int kv_heads, int sms, int* kept) {
    const bool narrow = heads / kv_heads <= 8;
    const long long pairs = (long long)requests * kv_heads, tiles = (longest + BN - 1) / BN, room = narrow ? 2LL * sms : sms;
    if (heads / kv_heads > 16 || pairs > room) return 0;
    int blocks = 1;
    while (blocks < MOST_TOGETHER && blocks < tiles && pairs * blocks * 2 * 100 <= room * (blocks == 4 ? 65 : 87)) blocks *= 2;
    const long long each = (tiles + blocks - 1) / blocks;
    if (tiles > (narrow ? 8 : 16) && each > (few_heads(requests, heads, sms) ? (narrow ? 2 : 3) : (narrow ? 4 : 8))) return 0;
    *kept = (int)each * BN;
    return blocks;
}
// How a key/value head's group of heads is cut: into chunks, each a block's, and those into sets.
struct Strips { int heads, sets, chunks, blocks; };  // of a set; of a chunk; of a group; that an SM holds
static Strips strips_for(int group) {
    if (group <= 8) return {group, 1, 1, Shape<1, 1>::BLOCKS};
    if (group <= 16) return {group, 1, 1, Shape<2, 1>::BLOCKS};
    // Three sets read keys and values once where two strips of 16 read them twice (us, 24 heads over 1: of 128, 11 requests at 23,692 slots 40.2 / 47.0, 64 of them 184 / 224, one at 512 9.9 / 9.3; of 64, where they are half as
    // many bytes for as many instructions, 11 30.6 / 30.6 and 64 141 / 136).  Two sets of 16 rows for 32 heads gain nothing: 51.2 / 51.4.  Rows of 24 or 32 in a warp's registers do not fit: 56 and 70.
    if (group <= 24 && D == 128) return {(group + 2) / 3, 3, 1, 1};
    return {16, 1, (group + 15) / 16, Shape<2, 1>::BLOCKS};
}
// Blocks of the first kernel that stand side by side for a key/value head's strip: what the device holds, but no more than there can be tiles.
static int blocks_for(int requests, int longest, int heads, int kv_heads, int sms) {
    const Strips strips = strips_for(heads / kv_heads);
    const long long room = (long long)sms * strips.blocks / ((long long)kv_heads * strips.chunks), tiles = (long long)requests * ((longest + BN - 1) / BN);
    return (int)(room < 1 ? 1 : room < tiles ? room : tiles);
}
// Bytes of scratch that hb_attention_tallied takes.
HB_EXPORT long long hb_attention_tallied_scratch(int requests, int longest, int heads, int kv_heads, int sms) {
    if (requests <= 0 || longest <= 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads || sms <= 0) return 0;
    int kept;
    if (together_for(requests, longest, heads, kv_heads, sms, &kept)) return 0;
    const long long slots = (longest + BN - 1) / BN * BN, pieces = (long long)blocks_for(requests, longest, heads, kv_heads, sms) + requests;
    return 4 * heads * (requests * slots + pieces * (D + 2));
}
// q [requests, heads * D] with rows q_stride apart; cache [pages, 2, kv_heads, page_size, D]; weights, positions [requests, kv_heads, capacity]; lengths, newest [requests], lengths at most
// `longest`, which table and capacity hold.  scratch: hb_attention_tallied_scratch bytes on a 16-byte boundary, null where it takes none.
HB_EXPORT int hb_attention_tallied(const void* q, long long q_stride, void* out, long long out_stride, const void* cache, const int* block_table, int table_width, const int* lengths, int requests,
                                   int longest, float* weights, int* positions, const int* newest, int capacity, int heads, int kv_heads, int page_size, int pages, float scale, int sms, void* scratch,
                                   int* status, cudaStream_t stream) {
    if (requests <= 0) return 0;
    if (!q || !out || !cache || !block_table || !lengths || !weights || !positions || !newest || !status) return HB_BAD_ARGUMENT;
    if (kv_heads <= 0 || heads <= 0 || heads % kv_heads || pages <= 0 || table_width <= 0 || longest <= 0 || capacity < longest || sms <= 0 || sms > 16384 || q_stride % 8 || out_stride % 4 || !(scale > 0.f && scale <= 0x1p127f)) return HB_BAD_ARGUMENT;
    if (page_size < 8 || page_size > 64 || (page_size & (page_size - 1))) return HB_UNSUPPORTED_SIZE;
    if ((((uintptr_t)q | (uintptr_t)cache | (uintptr_t)scratch) & 15) || ((uintptr_t)out & 7)) return HB_BAD_ARGUMENT;
    if ((long long)table_width * page_size < longest) return HB_BAD_ARGUMENT;
    if ((long long)pages * 2 * kv_heads * page_size > 0x7fffffffLL) return HB_UNSUPPORTED_SIZE;  // a row's number in the cache's tensor map
    if (q_stride > 0x7fffffffLL || out_stride > 0x7fffffffLL || longest > 0x7fffffff - SPAN - heads || requests > 65535) return HB_UNSUPPORTED_SIZE;
    const int group = heads / kv_heads, slots = (longest + BN - 1) / BN * BN;
    const Strips strips = strips_for(group);
    if ((long long)kv_heads * strips.chunks > 65535) return HB_UNSUPPORTED_SIZE;
    int kept = 0;
    const int together = together_for(requests, longest, heads, kv_heads, sms, &kept), blocks = together ? 0 : blocks_for(requests, longest, heads, kv_heads, sms);
    if (!together && !scratch) return HB_BAD_ARGUMENT;
    // One block a head where they are few or have many pieces (us, one block for all heads / one a head: 28 heads over 4, one request at 1,024 slots 9.6 / 6.5, four 11.2 / 8.0, but 16 at 1,024 14.1 / 14.9, at 4,099
    // 26.1 / 27.4; 14 over 2 of 64, 16 at 2,048 12.1 / 8.7, three at 23,080, 74 pieces each, 34 / 14).
    const int by_head = few_heads(requests, heads, sms) || (blocks / requests) * ((group + 7) / 8) > 16, join_blocks = by_head ? group : 1;
    const size_t n_pieces = (size_t)blocks + requests;
    float* pieces = (float*)scratch;
    float* scores = pieces + n_pieces * heads * D;  // before the sums, so that its rows begin on 16 bytes
    float2* sums = (float2*)(scores + (size_t)requests * heads * slots);
    const Args a{(const bf16*)q, (int)q_stride, (bf16*)out, (int)out_stride, block_table, table_width, lengths, requests, longest, slots, scores, pieces, sums, weights, positions, newest, capacity,
                 heads, kv_heads, page_size, pages, strips.heads, strips.chunks, blocks, join_blocks, by_head, together, kept, scale * 1.4426950408889634f, status};
    CUtensorMap map;
    if (int code = cache_map(&map, cache, a)) return code;
    if (int code = launch_first<D>(strips.heads, strips.sets, a, map, stream)) return code;
    if (together) return 0;
    return launch_after_previous(tally_kernel, dim3((longest + SPAN - 1) / SPAN + join_blocks, kv_heads, requests), dim3(ADD_THREADS), 0, stream, a);
}
HB_EXPORT int hb_attention_tallied_packed(const void* arguments) { return call_packed(&hb_attention_tallied, arguments); }
