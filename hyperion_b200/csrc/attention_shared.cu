// Attention of a step's queries over paged caches in which groups of requests share their first positions, for caches of bfloat16 and of
// 8-bit records (cache8.cu), head sizes 64 and 128 (HB_HEAD_DIM) and pages of 8 to 64 tokens.
//
// The host (host/shared_plan.cpp) cuts the step into items: (tokens that stand together, a table row, a range of keys).  A group's shared positions are one range
// for all of its tokens, so they are fetched once for all of them; what a request holds beyond them is a range for its own tokens; either may
// be cut further so that the device is filled.  An item leaves for each of its (token, head) rows a piece
//     m,  l = sum_j 2^(y_j - m),  o = sum_j 2^(y_j - m) v_j          y_j = score_j * scale * log2(e)
// and the pieces of a row are put together afterwards, in the order of the ranges: with M = max m, out = sum 2^(m - M) o / sum 2^(m - M) l.
// A step whose rows have one piece each is stored at once.  Where every row has one range and the device has room for two to eight blocks a range, those are a cluster: each walks its
// share, and at the end they read one another's results out of shared memory (mapa, ld.shared::cluster), so that no piece goes through memory and no kernel follows.  (Both ways, over
// 8-bit records, 28 heads over 4: one request at 512 positions 6.3 us against 7.6, eight at 2,048 10.4 against 10.8, 32 at 2,048 21 against 26, 32 at 9,000 59 against 86; a call
// that the host bounds 12 against 15.5.)
//
// This file has the strip kernel, for items of few rows: it is bound by the bytes of the keys and values.  One lane of a producer warp per
// page fetches K and V by TMA (one box a page and 128-byte panel, no multicast) into a ring of stages; each of four warps takes a quarter of a
// stage's keys for all rows, and at the end the warps' results are put together in shared memory.  The products are S^T = K Q^T and O^T = V^T P^T
// (mma.sync m16n8k16): keys and entries stand where the instruction has 16 rows, the few (token, head) rows where it has 8 columns, so that a decoded token of 7 heads a
// key/value head wastes one column of 8 and not 9 rows of 16, and O takes half the registers.  P^T is turned from the one's result into the other's operand by movmatrix.
//
// 8-bit records become float16, which holds every e4m3 code: one conversion instruction for two codes and nothing else per entry.  (mma.sync takes
// e4m3 as it is, too, but on this architecture each such product costs the conversions and four additions besides: 46 us against 42 where both were built.)  The
// exponents are kept out of the entries: a key's multiplies its score, and a value's goes into the softmax's exponent,
//     z_j = y_j + e_j,  P_j = 2^(z_j - m),  o = sum P_j code_j,  l = sum P_j 2^-e_j,
// with m 2^8 below the maximum of z.  A P below 2^-14 is rounded to 2^-25, 2^-33 of the largest: with the value's exponent in it that is a share of what the heaviest record brings.  Which entry of a head a lane's fragment holds does not matter to Q K^T as long as it is the same one in Q and K, so a
// lane takes 16 bytes of a key at once, and Q's fragments are loaded to match; the columns of P V come out in another order than they are stored in, and are
// stored where they belong.
//
// Where the values' exponents lie far apart (a value 2^12 times smaller than another one of its range), a weight that counts can be too small for float16
// beside the other's: such a stage's weights are multiplied in lots by their size.
//
// Over a bfloat16 cache the weights are taken in two parts, rounded to bfloat16 and what that left over: rounded once they would cost the result as much as
// its own rounding does (1.4 times the error in all), and float16, whose rounding does not show, does not hold every bfloat16 value.
//
// Measured: 64 requests at 2,048 positions each, 28 heads over 4 of 128, 31 us over 8-bit records (3.3 TB/s) and 43 us over bfloat16 (4.7 TB/s), the joining by a kernel included; 32 at
// 9,000, in clusters, 59 us (5.0 TB/s) and 94 us (6.3 TB/s).  Over
// bfloat16 the bytes and the starts and ends of the blocks bound it, over 8-bit records the instructions around the products (conversion, exponents, softmax of rows that stand
// across lanes).  One token of 14 heads at 512 positions: 5.5 us, a start and three dependent trips to memory.
//
// Slots beyond a range's end may hold anything: their scores are replaced and their values are read as zeros.  Every mbarrier wait is
// bounded (HB_WAIT_LIMIT looks); one that runs out sets HB_STATUS_WAIT_EXPIRED and the block leaves, once the copies that it has on their way have arrived.
#include <cuda.h>
#include <cuda_fp16.h>

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
constexpr int MOST_ROWS = 16;   // (token, head) rows of a strip: 8 or 16
constexpr int WARPS = 4;        // that compute; one more fetches
constexpr int THREADS = 32 * (WARPS + 1);
constexpr int ITEM_WORDS = 7;   // first token, tokens, table row, first key, last key + 1, number of the piece (with OWN_PIECE: among those of a request's own positions), -
constexpr int OWN_PIECE = 1 << 30;
constexpr unsigned WAIT_LIMIT = HB_WAIT_LIMIT, LAST_WAIT_LIMIT = 1u << 24;
constexpr float HEADROOM = 8.f;  // m stands so far below the maximum: P up to 2^8 keeps float16's small weights further from its smallest number

constexpr int FAR_APART = 12;    // exponents of values that differ by more: a weight P that counts may lie below what float16 holds well

__device__ __forceinline__ unsigned smem_u32(const void* p) { return (unsigned)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void mbar_init(unsigned long long* bar, unsigned count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(count));
}
__device__ __forceinline__ void mbar_expect_tx(unsigned long long* bar, unsigned bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ void mbar_arrive(unsigned long long* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
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
__device__ __forceinline__ void tma_load_2d(void* dst, const CUtensorMap* map, unsigned long long* bar, int x, int y) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
                 ::"r"(smem_u32(dst)), "l"(map), "r"(smem_u32(bar)), "r"(x), "r"(y) : "memory");
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
template <bool E8>
__device__ __forceinline__ void mma(float (&c)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) {
    if constexpr (E8)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <bool E8>
__device__ __forceinline__ unsigned pack(float lo, float hi) {
    unsigned w;
    if constexpr (E8) asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(hi), "f"(lo));
    else asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(hi), "f"(lo));
    return w;
}
__device__ __forceinline__ unsigned halves_of(unsigned codes) {  // the two codes in the lower half word
    unsigned w;
    asm("{.reg .b16 l, h;\n\tmov.b32 {l, h}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\t}" : "=r"(w) : "r"(codes));
    return w;
}
__device__ __forceinline__ unsigned upper_halves_of(unsigned codes) {
    unsigned w;
    asm("{.reg .b16 l, h;\n\tmov.b32 {l, h}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, h;\n\t}" : "=r"(w) : "r"(codes));
    return w;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ float fast_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float((unsigned)(127 + e) << 23); }  // -126 <= e <= 127

template <bool E8, int NQ>  // NQ: eights of rows
struct Shape {
    static constexpr int ROWS = 8 * NQ;
    static constexpr int BLOCKS = NQ == 1 ? 3 : 2;            // an SM, by registers
    static constexpr int BYTES = E8 ? 1 : 2;                  // of an entry
    static constexpr int BN = E8 ? 128 : 64;                  // keys of a stage
    static constexpr int KEYS = BN / WARPS;                   // of which a warp takes so many
    static constexpr int TILE = BN * D * BYTES;               // one K or V tile
    static constexpr int PANEL_BYTES = D * BYTES < 128 ? D * BYTES : 128;  // of a row, in one box
    static constexpr int PANELS = D * BYTES / PANEL_BYTES;
    static constexpr int EXPS = E8 ? 2 * BN : 0;              // the exponents of K and V
    static constexpr int STAGES = (D == 128 ? 2 : 4) + (NQ == 1 ? 0 : 1);  // BLOCKS blocks share an SM's memory
    static constexpr int CHUNKS = D * BYTES / 16;             // 16-byte chunks of a row
    static constexpr int STEPS = 4 / BYTES;                   // products of 16 entries that a chunk a lane feeds
    // Where the warps' results meet: COLS entries of every row at a time, a row's LINE floats apart (lanes that store side by side then take different banks), over the
    // keys' factors, which nobody wants any more by then.
    static constexpr int COLS = 64 / NQ, LINE = COLS + 4;
    static constexpr int JOIN = WARPS * ROWS * LINE * 4, FACTORS = E8 ? WARPS * 3 * KEYS * 4 : 0;
    static_assert(FACTORS <= JOIN, "the factors lie where the results meet");
    static constexpr size_t SMEM = 1024 + (size_t)STAGES * (2 * TILE + EXPS) + JOIN + 2 * WARPS * ROWS * 4 + 2 * STAGES * 8 + 16;
    static_assert(BLOCKS * (SMEM + 1024) <= 228 * 1024, "an SM's shared memory");
    // 16-byte chunk cc of row `key` as TMA's swizzle has placed it: the panel's row of 128 bytes (of 64, in pairs) with its chunks permuted.
    static __device__ __forceinline__ int at(int key, int cc) {
        if constexpr (PANEL_BYTES == 64) return key * 64 + ((cc ^ ((key >> 1) & 3)) << 4);
        return (cc >> 3) * (BN * 128) + key * 128 + (((cc & 7) ^ (key & 7)) << 4);
    }
};

struct Args {
    const bf16* q; int q_stride;
    bf16* out; int out_stride;
    const signed char* exponents;  // of an 8-bit cache
    const int* block_table; int table_width;
    const int* items;
    const int* first_item;   // [blocks + 1]: block b takes items first_item[b] .. first_item[b + 1] - 1
    const int* last;         // [tokens]: the last position a token sees, -1 for none
    const int* piece_start;  // [tokens + 1]
    const int* own_start;    // [tokens]
    float* pieces;           // [pieces, heads, D], or null: rows have one piece each and are stored at once
    float2* sums;            // [pieces, heads]: (m, l)
    int heads, kv_heads, page_size, pages;
    int beside_tiles;        // the tile kernel of the same step was launched right before
    int together;            // 0, or the blocks of a cluster, which has one run: an item each, joined among them
    int gc, chunks;          // heads of a strip, strips of a key/value head's group
    float scale_log2;
    int* status;
};

constexpr int MOST_TOGETHER = 8;
// The blocks of a cluster: those of their threads that have not left.
__device__ __forceinline__ void cluster_meet() {
    asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
// What another block of the cluster has at this place of its shared memory.
__device__ __forceinline__ unsigned their(const void* p, int rank) {
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
// TOGETHER: an instance of its own, so that the others keep the registers that the joining takes (drafts behind prefixes beside tiles 23.6 us, against 22.5).
template <bool E8, int NQ, bool TOGETHER>
__global__ void __launch_bounds__(THREADS, (Shape<E8, NQ>::BLOCKS)) attention_strip_kernel(const __grid_constant__ CUtensorMap kv_map, const Args a) {
    typedef Shape<E8, NQ> S;
    constexpr int BN = S::BN, KEYS = S::KEYS, NK = KEYS / 16, ROWS = S::ROWS;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* ring = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    // the tiles of all stages, the exponents of all stages, and each warp's keys' factors
    unsigned char* exps = ring + (size_t)S::STAGES * 2 * S::TILE;
    float* factors = reinterpret_cast<float*>(exps + (size_t)S::STAGES * S::EXPS);
    float* join = factors;  // [WARPS][ROWS][LINE]
    float* tops = join + S::JOIN / 4;  // [WARPS][ROWS]: maxima
    float* parts = tops + WARPS * ROWS;  // [WARPS][ROWS]: sums
    unsigned long long* full = reinterpret_cast<unsigned long long*>(parts + WARPS * ROWS);
    unsigned long long* empty = full + S::STAGES;
    volatile int* failed = reinterpret_cast<volatile int*>(empty + S::STAGES);
    volatile int* lost = failed + 1;  // a computing warp has given up

    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (tid == 0) {
        for (int s = 0; s < S::STAGES; ++s) { mbar_init(&full[s], E8 ? 33 : 1); mbar_init(&empty[s], WARPS); }
        *failed = 0, *lost = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    let_next_kernel_start();
    // Behind the tile kernel of the same step, whose blocks let this one start only when all kernels before it had finished, there is nothing to wait for here: its pieces
    // are others, and the two share the device.  (Whoever comes next waits for this kernel, and this one for that at its end.)
    if (!a.beside_tiles) wait_for_previous_kernels();
    const int kvh = blockIdx.y / a.chunks, chunk = blockIdx.y - kvh * a.chunks;
    const int group = a.heads / a.kv_heads, first_head = kvh * group + chunk * a.gc, heads_here = min(a.gc, group - chunk * a.gc);
    const int first_item = a.first_item[blockIdx.x], end_item = a.first_item[blockIdx.x + 1];
    int stage = 0;  // so far: the ring runs on across the block's items

    if (warp == WARPS) {
        // ------------------------------------------------------------------ producer (the whole warp)
        const int shift = 31 - __clz(a.page_size), pages_per_tile = BN >> shift, tiles_per_look = 32 / pages_per_tile;
        constexpr int OPS_PER_PAGE = 2 * S::PANELS;
        const int ops = pages_per_tile * OPS_PER_PAGE;
        const unsigned page_bytes = 2u * a.page_size * D * S::BYTES;
        if (lane == 0) asm volatile("prefetch.tensormap [%0];" ::"l"(&kv_map) : "memory");
        int ok = 1;
        for (int index = first_item; index < end_item && ok; ++index) {
            const int* item = a.items + (size_t)index * ITEM_WORDS;
            const int key_lo = item[3], key_hi = item[4], start = key_lo / BN * BN, n_tiles = (key_hi - start + BN - 1) / BN;
            const int* table = a.block_table + (size_t)item[2] * a.table_width;
            int looked = -1;
            for (int it = 0; it < n_tiles; ++it, ++stage) {
                const int s = stage % S::STAGES, round = stage / S::STAGES;
                if (it % tiles_per_look == 0) {  // a page number per lane, for the next tiles
                    const int block = ((start + it * BN) >> shift) + lane;
                    looked = block < a.table_width ? __ldg(table + block) : -1;
                }
                if (lane == 0) ok = mbar_wait(&empty[s], (round & 1) ^ 1, failed) ? 1 : 0;
                ok = __shfl_sync(0xffffffffu, ok, 0);
                if (!ok) {
                    if (lane == 0) { *failed = 1; atomicOr(a.status, HB_STATUS_WAIT_EXPIRED | HB_STATUS_IN_ATTENTION_STRIPS); }
                    break;
                }
                const int base = start + it * BN, k0 = base + lane * a.page_size;
                int page = __shfl_sync(0xffffffffu, looked, (it % tiles_per_look) * pages_per_tile + lane);
                const bool wanted = lane < pages_per_tile && k0 < key_hi && k0 + a.page_size > key_lo;
                if (wanted && (page < 0 || page >= a.pages)) atomicOr(a.status, HB_STATUS_BAD_PAGE);
                if (!wanted || page >= a.pages) page = -1;
                const unsigned valid = __popc(__ballot_sync(0xffffffffu, page >= 0));
                if (lane == 0) {
                    if (valid) mbar_expect_tx(&full[s], valid * page_bytes); else mbar_arrive(&full[s]);
                }
                __syncwarp();
                unsigned char* tiles = ring + (size_t)s * 2 * S::TILE;
                if constexpr (E8) {  // the exponents of four keys and of four values a lane
                    const int key = lane * 4, from = __shfl_sync(0xffffffffu, page, key >> shift);
                    if (from >= 0) {
                        const signed char* src = a.exponents + ((size_t)from * 2 * a.kv_heads + kvh) * a.page_size + (key & (a.page_size - 1));
                        asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(exps + s * S::EXPS + key)), "l"(src) : "memory");
                        asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(exps + s * S::EXPS + BN + key)), "l"(src + (size_t)a.kv_heads * a.page_size) : "memory");
                    }
                    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(&full[s])) : "memory");
                }
                for (int op0 = 0; op0 < ops; op0 += 32) {
                    const int op = op0 + lane;
                    const int p = min(op, ops - 1) / OPS_PER_PAGE, rest = op % OPS_PER_PAGE, which = rest / S::PANELS, panel = rest - which * S::PANELS;
                    const int from = __shfl_sync(0xffffffffu, page, p);
                    if (op < ops && from >= 0)
                        tma_load_2d(tiles + which * S::TILE + panel * (BN * S::PANEL_BYTES) + p * a.page_size * S::PANEL_BYTES, &kv_map, &full[s],
                                    panel * (S::PANEL_BYTES / S::BYTES), ((from * 2 + which) * a.kv_heads + kvh) * a.page_size);
                }
            }
        }
        if (lane == 0)
            for (int k = max(0, stage - S::STAGES); k < stage; ++k) mbar_last_wait(&full[k % S::STAGES], (k / S::STAGES) & 1);
        __syncwarp();
        if constexpr (TOGETHER) cluster_meet(), cluster_meet();
        return;
    }
    // ---------------------------------------------------------------------- consumers
    [[maybe_unused]] float* rows_here = reinterpret_cast<float*>(ring);  // [ROWS][D]: what a block of a cluster brings; the ring has been read to its end by then
    [[maybe_unused]] float2* sums_here = reinterpret_cast<float2*>(rows_here + ROWS * D);  // [ROWS]
    static_assert(ROWS * (D * 4 + 8) <= S::STAGES * 2 * S::TILE, "a cluster's results lie where the ring was");
    const int t = lane & 3, g = lane >> 2;
    [[maybe_unused]] float* mine = factors + warp * 3 * KEYS;  // of this warp's keys: 2^e of the key, e of the value, 2^-e of the value
    auto meet = [] { asm volatile("bar.sync 1, %0;" ::"n"(32 * WARPS) : "memory"); };
    constexpr int LANES_PER_ROW = S::COLS / 16;
    const int store_row = lane / LANES_PER_ROW, store_col = warp * (S::COLS / 4) + lane % LANES_PER_ROW * 4;  // what this lane stores of every COLS entries
    struct Words { int tok0, ntok, key_lo, key_hi, piece; };
    auto words_of = [&](int index) {
        const int* item = a.items + (size_t)index * ITEM_WORDS;
        return Words{item[0], item[1], item[3], item[4], item[5]};
    };
    // An item's queries are on their way while the item before it is put together (of eight rows; sixteen have no registers for it).
    uint4 raw[NQ][D / 32];  // of rows q * 8 + g: this lane's quarter, chunks t, t + 4, ...
    int sees[NQ];
    auto fetch_queries = [&](const Words& w) {
#pragma unroll
        for (int q = 0; q < NQ; ++q) {
            const int v = q * 8 + g, tok = v / a.gc, hh = v - tok * a.gc;
            const bool valid = tok < w.ntok && hh < heads_here;
            const bf16* src = a.q + (size_t)(w.tok0 + (valid ? tok : 0)) * a.q_stride + (size_t)(first_head + (valid ? hh : 0)) * D;
            constexpr int PER_CHUNK = 16 / S::BYTES, PIECES = PER_CHUNK / 8;  // entries of a chunk; 16-byte pieces of them in bfloat16
#pragma unroll
            for (int i = 0; i < D / 32; ++i) raw[q][i] = valid ? *reinterpret_cast<const uint4*>(src + (t + 4 * (i / PIECES)) * PER_CHUNK + (i % PIECES) * 8) : make_uint4(0, 0, 0, 0);
            sees[q] = valid ? a.last[w.tok0 + tok] : 0x7fffffff;
        }
    };
    Words next = words_of(first_item);
    if (NQ == 1) fetch_queries(next);
    for (int index = first_item; index < end_item; ++index) {
        const int tok0 = next.tok0, ntok = next.ntok, key_lo = next.key_lo, key_hi = next.key_hi, piece = next.piece;
        const int start = key_lo / BN * BN, n_tiles = (key_hi - start + BN - 1) / BN;
        if (NQ != 1) fetch_queries(next);
        if (index + 1 < end_item) next = words_of(index + 1);
        // where this lane stores
        const int store_tok = store_row / a.gc, store_head = store_row - store_tok * a.gc;
        const bool stores = store_tok < ntok && store_head < heads_here;
        int piece_at = 0;
        if (stores && a.pieces) piece_at = (piece & OWN_PIECE ? a.own_start : a.piece_start)[tok0 + store_tok] + (piece & (OWN_PIECE - 1));
        // Q's fragments: a lane's 16-byte chunk t + 4 j of a key feeds products STEPS j to STEPS j + STEPS - 1, four of its entries each, so a query's entries stand
        // in the fragments likewise.
        unsigned qf[NQ][D / 16][2];
        float row_scale[NQ][2];
        int hi[NQ][2];  // of columns 2 t and 2 t + 1: the last key a row sees; a row that is no one's sees what the others see, and is never stored
        int sees_all_to = key_hi - 1;
#pragma unroll
        for (int q = 0; q < NQ; ++q) {
            const int mine_sees = min(key_hi - 1, sees[q]);
            const unsigned words[D / 8] = {
#define HB_WORDS(i) raw[q][i].x, raw[q][i].y, raw[q][i].z, raw[q][i].w
                HB_WORDS(0), HB_WORDS(1),
#if HB_HEAD_DIM == 128
                HB_WORDS(2), HB_WORDS(3),
#endif
#undef HB_WORDS
            };
            float factor = 1.f, scale = a.scale_log2;
            if constexpr (E8) {
                // As float16 with the row's largest entry between 2^13 and 2^14: an entry of eight bits keeps them all down to 2^-27 of the largest.
                float largest = 0.f;
#pragma unroll
                for (int i = 0; i < D / 8; ++i) largest = max3(largest, fabsf(__uint_as_float(words[i] << 16)), fabsf(__uint_as_float(words[i] & 0xffff0000u)));
                largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, 1));
                largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, 2));
                const int e = min(max((int)(__float_as_uint(largest) >> 23) - 127 - 13, -126), 126);
                factor = power_of_two(-e);
                scale *= power_of_two(e);
            }
#pragma unroll
            for (int i = 0; i < D / 8; ++i)
                qf[q][i >> 1][i & 1] = E8 ? pack<true>(__uint_as_float(words[i] << 16) * factor, __uint_as_float(words[i] & 0xffff0000u) * factor) : words[i];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                row_scale[q][e] = __shfl_sync(0xffffffffu, scale, (2 * t + e) * 4);
                hi[q][e] = __shfl_sync(0xffffffffu, mine_sees, (2 * t + e) * 4);
            }
            sees_all_to = min(sees_all_to, __reduce_min_sync(0xffffffffu, mine_sees));  // positions that every row sees
        }
        float m[NQ][2], l[NQ][2];
        int top_e = -128;  // the largest exponent among the values so far
        float o[NQ][D / 16][4];
#pragma unroll
        for (int q = 0; q < NQ; ++q) {
            m[q][0] = m[q][1] = -INFINITY, l[q][0] = l[q][1] = 0.f;
#pragma unroll
            for (int i = 0; i < D / 16; ++i) o[q][i][0] = o[q][i][1] = o[q][i][2] = o[q][i][3] = 0.f;
        }

        for (int it = 0; it < n_tiles; ++it, ++stage) {
            const int s = stage % S::STAGES, round = stage / S::STAGES;
            if (!mbar_wait(&full[s], round & 1, failed)) {
                *failed = 1, *lost = 1;
                atomicOr(a.status, HB_STATUS_WAIT_EXPIRED | HB_STATUS_IN_ATTENTION_STRIPS);
                break;
            }
            const unsigned char* ks = ring + (size_t)s * 2 * S::TILE;
            const unsigned char* vs = ks + S::TILE;
            const int key0 = warp * KEYS, pos0 = start + it * BN + key0;  // this warp's keys
            if (pos0 < key_hi && pos0 + KEYS > key_lo) {
                const bool whole = pos0 >= key_lo && pos0 + KEYS <= key_hi;  // all of them are in the item's range
                bool far_apart = false;
                if constexpr (E8) {  // a lane has one key; what was never stored is no exponent: kept in range, it meets only scores that are replaced
                    const signed char* ex = reinterpret_cast<const signed char*>(exps + s * S::EXPS + key0 + lane);
                    const int ke = min(max((int)ex[0], -40), 40), ve = min(max((int)ex[BN], -40), 40), pos = pos0 + lane;
                    mine[lane] = power_of_two(ke), mine[KEYS + lane] = (float)ve, mine[2 * KEYS + lane] = power_of_two(-ve);
                    const bool inside = pos >= key_lo && pos < key_hi;
                    top_e = __reduce_max_sync(0xffffffffu, inside ? max(top_e, ve) : top_e);
                    far_apart = top_e - __reduce_min_sync(0xffffffffu, inside ? ve : 127) > FAR_APART;
                    __syncwarp();
                }
                float sc[NQ][NK][4];  // of keys g and g + 8 of 16 and columns 2 t and 2 t + 1: [(key, column)]
#pragma unroll
                for (int q = 0; q < NQ; ++q)
#pragma unroll
                    for (int k = 0; k < NK; ++k) sc[q][k][0] = sc[q][k][1] = sc[q][k][2] = sc[q][k][3] = 0.f;
#pragma unroll
                for (int j = 0; j < S::CHUNKS / 4; ++j)
#pragma unroll
                    for (int k = 0; k < NK; ++k) {
                        const uint4 raw0 = *reinterpret_cast<const uint4*>(ks + S::at(key0 + k * 16 + g, t + 4 * j)), raw1 = *reinterpret_cast<const uint4*>(ks + S::at(key0 + k * 16 + 8 + g, t + 4 * j));
                        const unsigned* w0 = reinterpret_cast<const unsigned*>(&raw0);
                        const unsigned* w1 = reinterpret_cast<const unsigned*>(&raw1);
#pragma unroll
                        for (int w = 0; w < S::STEPS; ++w) {
                            unsigned x[4];
                            if constexpr (E8) x[0] = halves_of(w0[w]), x[1] = halves_of(w1[w]), x[2] = upper_halves_of(w0[w]), x[3] = upper_halves_of(w1[w]);
                            else x[0] = w0[2 * w], x[1] = w1[2 * w], x[2] = w0[2 * w + 1], x[3] = w1[2 * w + 1];
#pragma unroll
                            for (int q = 0; q < NQ; ++q) mma<E8>(sc[q][k], x, qf[q][j * S::STEPS + w][0], qf[q][j * S::STEPS + w][1]);
                        }
                    }
                float back[NK][2];
#pragma unroll
                for (int k = 0; k < NK; ++k)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {  // key g + 8 h of 16
                        float key_scale = 1.f, value_e = 0.f;
                        if constexpr (E8) key_scale = mine[k * 16 + h * 8 + g], value_e = mine[KEYS + k * 16 + h * 8 + g], back[k][h] = mine[2 * KEYS + k * 16 + h * 8 + g];
#pragma unroll
                        for (int q = 0; q < NQ; ++q)
#pragma unroll
                            for (int e = 0; e < 2; ++e) sc[q][k][2 * h + e] = E8 ? fmaf(sc[q][k][2 * h + e] * key_scale, row_scale[q][e], value_e) : sc[q][k][2 * h + e] * row_scale[q][e];
                    }
                if (pos0 < key_lo || pos0 + KEYS - 1 > sees_all_to) {
#pragma unroll
                    for (int q = 0; q < NQ; ++q)
#pragma unroll
                        for (int k = 0; k < NK; ++k)
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const int pos = pos0 + k * 16 + (e >> 1) * 8 + g;
                                if (pos > hi[q][e & 1] || pos < key_lo) sc[q][k][e] = -INFINITY;
                            }
                }
                bool rescale = false;
                float alpha[NQ][2];
#pragma unroll
                for (int q = 0; q < NQ; ++q)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float mx = fmaxf(sc[q][0][e], sc[q][0][2 + e]);
#pragma unroll
                        for (int k = 1; k < NK; ++k) mx = max3(mx, sc[q][k][e], sc[q][k][2 + e]);
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
                        const float m_new = fmaxf(m[q][e], mx - (E8 ? HEADROOM : 0.f));
                        alpha[q][e] = m_new == -INFINITY ? 1.f : fast_exp2(m[q][e] - m_new);
                        m[q][e] = m_new;
                        rescale |= alpha[q][e] != 1.f;
                        const float base = m_new == -INFINITY ? 0.f : m_new;
                        l[q][e] *= alpha[q][e];
#pragma unroll
                        for (int k = 0; k < NK; ++k)
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                const float p = fast_exp2(sc[q][k][2 * h + e] - base);
                                sc[q][k][2 * h + e] = p;
                                l[q][e] = E8 ? fmaf(p, back[k][h], l[q][e]) : l[q][e] + p;  // of this lane's keys; the lanes are added up at the end
                            }
                    }
                if (__any_sync(0xffffffffu, rescale)) {
#pragma unroll
                    for (int q = 0; q < NQ; ++q)
#pragma unroll
                        for (int i = 0; i < D / 16; ++i) o[q][i][0] *= alpha[q][0], o[q][i][1] *= alpha[q][1], o[q][i][2] *= alpha[q][0], o[q][i][3] *= alpha[q][1];
                }
#pragma unroll
                for (int k = 0; k < NK; ++k) {  // 16 keys
                    const int key = key0 + k * 16;
                    // Values beyond the range read as zeros, whatever their slots hold.  A fragment register holds keys 2 t and 2 t + 1 in its halves.
                    unsigned keep[2] = {0xffffffffu, 0xffffffffu};
                    if (!whole) {
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const int pos = pos0 + k * 16 + h * 8 + t * 2;
                            keep[h] = (pos >= key_lo && pos < key_hi ? 0xffffu : 0u) | (pos + 1 >= key_lo && pos + 1 < key_hi ? 0xffff0000u : 0u);
                        }
                    }
                    auto values = [&](int c, unsigned (&x)[2][4]) {  // 16 keys of two 16-byte chunks: 16 entries each in 8 bits; together in bfloat16, in x[0]
                        unsigned b[4];
                        ldmatrix_x4_trans(b, vs + S::at(key + (lane & 15), c + (lane >> 4)));
                        if (!whole) b[0] &= keep[0], b[1] &= keep[1], b[2] &= keep[0], b[3] &= keep[1];
                        if constexpr (E8) {
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                // bytes (key 2t: entries 2g, 2g + 1; key 2t + 1: the same) -> the two keys' even entries, rows g, and their odd ones, rows g + 8
                                const unsigned b0 = __byte_perm(b[2 * h], 0, 0x3120), b1 = __byte_perm(b[2 * h + 1], 0, 0x3120);
                                x[h][0] = halves_of(b0), x[h][1] = upper_halves_of(b0), x[h][2] = halves_of(b1), x[h][3] = upper_halves_of(b1);
                            }
                        } else {
                            x[0][0] = b[0], x[0][1] = b[2], x[0][2] = b[1], x[0][3] = b[3];
                        }
                    };
                    constexpr int TILES = E8 ? 2 : 1;  // of 16 entries, of two chunks
                    if (E8 && far_apart) {
                        // Weights by size, 2^18 at a time, each lot scaled up to where float16 holds it and the products scaled back.
#pragma unroll 1
                        for (int lot = 0; lot < 7; ++lot) {
                            const float up = power_of_two(18 * lot), down = power_of_two(-18 * lot), from = lot < 6 ? down * 0x1p-10f : 0.f, to = lot ? down * 256.f : INFINITY;
                            auto scaled = [&](float p) { return p <= from || p > to ? 0.f : p * up; };
                            unsigned part[NQ][2], any = 0;
#pragma unroll
                            for (int q = 0; q < NQ; ++q)
#pragma unroll
                                for (int h = 0; h < 2; ++h) {
                                    part[q][h] = turned(pack<true>(scaled(sc[q][k][2 * h]), scaled(sc[q][k][2 * h + 1])));
                                    any |= part[q][h];
                                }
                            if (!__any_sync(0xffffffffu, any != 0)) continue;
#pragma unroll
                            for (int c = 0; c < S::CHUNKS; c += 2) {
                                unsigned x[2][4];
                                values(c, x);
#pragma unroll
                                for (int h = 0; h < TILES; ++h)
#pragma unroll
                                    for (int q = 0; q < NQ; ++q) {
                                        float more[4] = {0.f, 0.f, 0.f, 0.f};
                                        mma<E8>(more, x[h], part[q][0], part[q][1]);
#pragma unroll
                                        for (int e = 0; e < 4; ++e) o[q][(c / 2) * TILES + h][e] = fmaf(more[e], down, o[q][(c / 2) * TILES + h][e]);
                                    }
                            }
                        }
                        continue;
                    }
                    unsigned pf[NQ][2];
                    [[maybe_unused]] unsigned pr[NQ][2];  // bfloat16: what the weights lose by rounding, as weights of their own
#pragma unroll
                    for (int q = 0; q < NQ; ++q)
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const float p0 = sc[q][k][2 * h], p1 = sc[q][k][2 * h + 1];
                            const unsigned w = pack<E8>(p0, p1);
                            pf[q][h] = turned(w);
                            if constexpr (!E8) pr[q][h] = turned(pack<false>(p0 - __uint_as_float(w << 16), p1 - __uint_as_float(w & 0xffff0000u)));
                        }
#pragma unroll
                    for (int c = 0; c < S::CHUNKS; c += 2) {
                        unsigned x[2][4];
                        values(c, x);
#pragma unroll
                        for (int h = 0; h < TILES; ++h)
#pragma unroll
                            for (int q = 0; q < NQ; ++q) {
                                mma<E8>(o[q][(c / 2) * TILES + h], x[h], pf[q][0], pf[q][1]);
                                if constexpr (!E8) mma<E8>(o[q][(c / 2) * TILES + h], x[h], pr[q][0], pr[q][1]);
                            }
                    }
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&empty[s]);
        }
        if (NQ == 1 && index + 1 < end_item) fetch_queries(next);
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
        float top = -INFINITY, total = 0.f;  // of the row that this lane stores
#pragma unroll
        for (int w = 0; w < WARPS; ++w) top = fmaxf(top, tops[w * ROWS + store_row]);
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            const float mw = tops[w * ROWS + store_row];
            total = fmaf(mw == -INFINITY ? 0.f : fast_exp2(mw - top), parts[w * ROWS + store_row], total);
        }
        const float inv = total > 0.f ? 1.f / total : (total == 0.f ? 0.f : total);  // a row that sees nothing is zeros; a NaN stays one
        const size_t slot = (size_t)piece_at * a.heads + first_head + store_head;
        if (!TOGETHER && stores && a.pieces && store_col == 0) a.sums[slot] = make_float2(top, total);
        if (TOGETHER && stores && store_col == 0) sums_here[store_row] = make_float2(top, total);
#pragma unroll
        for (int col = 0; col < D; col += S::COLS) {
#pragma unroll
            for (int q = 0; q < NQ; ++q)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float* dst = join + (warp * ROWS + q * 8 + 2 * t + e) * S::LINE;
#pragma unroll
                    for (int i = 0; i < S::COLS / 16; ++i) {
                        const float x = o[q][col / 16 + i][e] * f[q][e], y = o[q][col / 16 + i][2 + e] * f[q][e];
                        if constexpr (E8) *reinterpret_cast<float2*>(dst + 16 * i + 2 * g) = make_float2(x, y);
                        else dst[16 * i + g] = x, dst[16 * i + 8 + g] = y;
                    }
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
                if (TOGETHER) {
                    store4(rows_here + store_row * D + col + store_col, sum);
                } else if (a.pieces) {
                    store4(a.pieces + slot * D + col + store_col, sum);
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i) sum[i] *= inv;
                    store4(a.out + (size_t)(tok0 + store_tok) * a.out_stride + (size_t)(first_head + store_head) * D + col + store_col, sum);
                }
            }
            meet();
        }
        if constexpr (TOGETHER) {
            // Every block of the cluster takes a part of the rows' entries, brings the blocks' sums to the largest maximum, in the order of the blocks, and stores.
            cluster_meet();
            unsigned rank;
            asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
            for (int at = (int)rank * 32 * WARPS + tid; at < ROWS * (D / 4); at += a.together * 32 * WARPS) {
                const int row = at / (D / 4), col = at % (D / 4) * 4, tok = row / a.gc, head = row - tok * a.gc;
                if (tok >= ntok || head >= heads_here) continue;
                float above = -INFINITY, all = 0.f, sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int r = 0; r < MOST_TOGETHER; ++r) above = fmaxf(above, theirs2(sums_here + row, min(r, a.together - 1)).x);
#pragma unroll 1
                for (int r0 = 0; r0 < a.together; r0 += 4) {  // four on their way together
                    float2 ml[4];
                    float4 part[4];
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int from = min(r0 + r, a.together - 1);
                        ml[r] = theirs2(sums_here + row, from), part[r] = theirs4(rows_here + row * D + col, from);
                    }
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        if (r0 + r >= a.together) break;
                        const float f = ml[r].x == -INFINITY ? 0.f : fast_exp2(ml[r].x - above);
                        all = fmaf(f, ml[r].y, all);
                        sum[0] = fmaf(f, part[r].x, sum[0]), sum[1] = fmaf(f, part[r].y, sum[1]), sum[2] = fmaf(f, part[r].z, sum[2]), sum[3] = fmaf(f, part[r].w, sum[3]);
                    }
                }
                const float share = all > 0.f ? 1.f / all : (all == 0.f ? 0.f : all);
#pragma unroll
                for (int i = 0; i < 4; ++i) sum[i] *= share;
                store4(a.out + (size_t)(tok0 + tok) * a.out_stride + (size_t)(first_head + head) * D + col, sum);
            }
            cluster_meet();  // nobody leaves while another still reads here
        }
    }
    if (a.beside_tiles) wait_for_previous_kernels();
}

template <int N>
__device__ __forceinline__ void load_floats(const float* p, float (&v)[N]) {
    if constexpr (N == 4) {
        load4(p, v);
    } else {
        const float2 x = *reinterpret_cast<const float2*>(p);
        v[0] = x.x, v[1] = x.y;
    }
}

// Puts the pieces of a (token, head) together: TEAM warps take every TEAM-th AHEAD of them, which are on their way together, and meet in shared memory.  One warp where a
// token has few; a long context cut over the whole device leaves a hundred, which one warp would walk a latency at a time (one token at 32,768 positions: 111 pieces of 28
// heads).  Bound by its start and three dependent trips to memory: 4 to 5 us beyond the kernel before, up to some 10 MB of pieces.
constexpr int MERGE_WARPS = 4;
template <int TEAM>
__global__ void __launch_bounds__(32 * MERGE_WARPS) attention_pieces_kernel(const float* __restrict__ pieces, const float2* __restrict__ sums, const int* __restrict__ piece_start,
                                                                            bf16* __restrict__ out, int out_stride, int heads) {
    constexpr int PER = D / 32, AHEAD = 8, HEADS = MERGE_WARPS / TEAM;
    __shared__ float2 tops[MERGE_WARPS];
    __shared__ __align__(16) float values[MERGE_WARPS][D];
    let_next_kernel_start();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, member = warp % TEAM;
    const int token = blockIdx.x, head = blockIdx.y * HEADS + warp / TEAM;
    const int first = piece_start[token], n = head < heads ? piece_start[token + 1] - first : 0;  // written with the plan, long before
    wait_for_previous_kernels();
    float top = -INFINITY, total = 0.f, value[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) value[i] = 0.f;
    for (int p0 = member * AHEAD; p0 < n; p0 += AHEAD * TEAM) {
        float part[AHEAD][PER];
        float2 ml[AHEAD];
        float above = top;
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
            const size_t slot = (size_t)(first + min(p0 + k, n - 1)) * heads + head;
            ml[k] = sums[slot];
            load_floats(pieces + slot * D + lane * PER, part[k]);
        }
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) above = p0 + k < n ? fmaxf(above, ml[k].x) : above;
        const float down = top == -INFINITY ? 0.f : fast_exp2(top - above);
        total *= down;
#pragma unroll
        for (int i = 0; i < PER; ++i) value[i] *= down;
        top = above;
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
            if (p0 + k >= n) break;
            const float f = ml[k].x == -INFINITY ? 0.f : fast_exp2(ml[k].x - top);
            total = fmaf(f, ml[k].y, total);
#pragma unroll
            for (int i = 0; i < PER; ++i) value[i] = fmaf(f, part[k][i], value[i]);
        }
    }
    if constexpr (TEAM > 1) {
        if (lane == 0) tops[warp] = make_float2(top, total);
#pragma unroll
        for (int i = 0; i < PER; ++i) values[warp][lane * PER + i] = value[i];
        __syncthreads();
        if (member != 0) return;
        float above = top;
#pragma unroll
        for (int w = 1; w < TEAM; ++w) above = fmaxf(above, tops[warp + w].x);
        total = 0.f;
#pragma unroll
        for (int i = 0; i < PER; ++i) value[i] = 0.f;
#pragma unroll
        for (int w = 0; w < TEAM; ++w) {
            const float2 theirs = tops[warp + w];
            const float f = theirs.x == -INFINITY ? 0.f : fast_exp2(theirs.x - above);
            total = fmaf(f, theirs.y, total);
#pragma unroll
            for (int i = 0; i < PER; ++i) value[i] = fmaf(f, values[warp + w][lane * PER + i], value[i]);
        }
    }
    if (head >= heads) return;
    const float inv = total > 0.f ? 1.f / total : (total == 0.f ? 0.f : total);
    bf16* dst = out + (size_t)token * out_stride + (size_t)head * D + lane * PER;
#pragma unroll
    for (int i = 0; i < PER; i += 2) *reinterpret_cast<__nv_bfloat162*>(dst + i) = __floats2bfloat162_rn(value[i] * inv, value[i + 1] * inv);
}

typedef CUresult (*EncodeTiled)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiled encode_tiled() {
    static EncodeTiled fn = nullptr;
    if (!fn) {
        void* found = nullptr;
        cudaDriverEntryPointQueryResult result;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &found, cudaEnableDefault, &result) == cudaSuccess && result == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<EncodeTiled>(found);
    }
    return fn;
}

// The cache as a matrix [pages * 2 * kv_heads * page_size, D], fetched in boxes of a page's rows and up to 128 bytes.
template <bool E8, int NQ>
int cache_map(CUtensorMap* map, const void* cache, int pages, int kv_heads, int page_size) {
    EncodeTiled encode = encode_tiled();
    if (!encode) return HB_BAD_ARGUMENT;
    const cuuint64_t dims[2] = {(cuuint64_t)D, (cuuint64_t)pages * 2 * kv_heads * page_size};
    const cuuint64_t strides[1] = {(cuuint64_t)D * Shape<E8, NQ>::BYTES};
    const cuuint32_t box[2] = {(cuuint32_t)(Shape<E8, NQ>::PANEL_BYTES / Shape<E8, NQ>::BYTES), (cuuint32_t)page_size};
    const cuuint32_t elem[2] = {1, 1};
    const CUresult r = encode(map, E8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(cache), dims, strides, box, elem,
                              CU_TENSOR_MAP_INTERLEAVE_NONE, Shape<E8, NQ>::PANEL_BYTES == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B,
                              CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? 0 : HB_BAD_ARGUMENT;
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

template <bool E8, int NQ, bool TOGETHER>
int launch_strips_as(const Args& a, const CUtensorMap& map, int blocks, cudaStream_t stream) {
    const auto kernel = attention_strip_kernel<E8, NQ, TOGETHER>;
    static const cudaError_t configured = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Shape<E8, NQ>::SMEM);
    if (configured != cudaSuccess) return (int)configured;
    const dim3 grid(blocks, a.kv_heads * a.chunks);
    if constexpr (TOGETHER) return launch_clusters(kernel, a.together, grid, dim3(THREADS), Shape<E8, NQ>::SMEM, stream, map, a);
    return launch_after_previous(kernel, grid, dim3(THREADS), Shape<E8, NQ>::SMEM, stream, map, a);
}
template <bool E8, int NQ>
int launch_strips(const Args& a, const void* cache, int blocks, cudaStream_t stream) {
    CUtensorMap map;
    if (int code = cache_map<E8, NQ>(&map, cache, a.pages, a.kv_heads, a.page_size)) return code;
    return a.together ? launch_strips_as<E8, NQ, true>(a, map, blocks, stream) : launch_strips_as<E8, NQ, false>(a, map, blocks, stream);
}
}  // namespace

// Puts the n_pieces = piece_start[tokens] pieces [n_pieces, heads, D] of the tokens together.  A token without a piece is zeros.
HB_EXPORT int hb_attention_pieces(const float* pieces, const float* sums, const int* piece_start, void* out, long long out_stride, int tokens, int n_pieces, int heads, cudaStream_t stream) {
    if (tokens <= 0) return 0;
    if (!pieces || !sums || !piece_start || !out || heads <= 0 || out_stride % 2 || ((uintptr_t)pieces & 15) || ((uintptr_t)out & 3)) return HB_BAD_ARGUMENT;
    if (out_stride > 0x7fffffffLL) return HB_UNSUPPORTED_SIZE;
    const bool many = n_pieces / tokens > 12;
    const int per_block = many ? 1 : MERGE_WARPS, rows = (heads + per_block - 1) / per_block;
    if (rows > 65535) return HB_UNSUPPORTED_SIZE;
    return launch_after_previous(many ? attention_pieces_kernel<MERGE_WARPS> : attention_pieces_kernel<1>, dim3(tokens, rows), dim3(32 * MERGE_WARPS), 0, stream, pieces, (const float2*)sums,
                                 piece_start, (bf16*)out, (int)out_stride, heads);
}

// cache: [pages, 2, kv_heads, page_size, D] in bfloat16 (exponents null) or e4m3 codes with exponents [pages, 2, kv_heads, page_size].
// beside_tiles: hb_attention_shared_tiles for the same step was the launch right before on this stream.  together: 0, or 2 to 8: so many blocks in a row have one item each, of the same
// tokens, and join them; no pieces then.
// items: see ITEM_WORDS; first_item [blocks + 1]; an item has at most rows / min(heads / kv_heads, rows) tokens, rows being 8 or 16.  pieces, sums null: one piece a row;
// else tokens and n_pieces as hb_attention_pieces takes them, which follows.
HB_EXPORT int hb_attention_strips(const void* q, long long q_stride, void* out, long long out_stride, const void* cache, const void* exponents, const int* block_table, int table_width,
                                  const int* items, const int* first_item, int blocks, int rows, int beside_tiles, int together, const int* last, const int* piece_start, const int* own_start, float* pieces, float* sums, int heads, int kv_heads,
                                  int page_size, int pages, float scale, int* status, cudaStream_t stream, int tokens, int n_pieces) {
    if (blocks <= 0) return 0;
    if (!q || !out || !cache || !block_table || !items || !first_item || !last || !piece_start || !own_start || !status || (!pieces != !sums)) return HB_BAD_ARGUMENT;
    if (kv_heads <= 0 || heads <= 0 || heads % kv_heads || pages <= 0 || table_width <= 0 || q_stride % 8 || out_stride % 4) return HB_BAD_ARGUMENT;
    if (!(scale > 0.f)) return HB_BAD_ARGUMENT;  // as in the tile kernel: a step is refused or not whatever kernels it takes
    if (page_size < 8 || page_size > 64 || (page_size & (page_size - 1))) return HB_UNSUPPORTED_SIZE;
    if ((((uintptr_t)q | (uintptr_t)cache | (uintptr_t)pieces) & 15) || ((uintptr_t)exponents & 3) || ((uintptr_t)out & 7)) return HB_BAD_ARGUMENT;
    if ((long long)pages * 2 * kv_heads * page_size > 0x7fffffffLL) return HB_UNSUPPORTED_SIZE;  // a row's number in the cache's tensor map
    if (q_stride > 0x7fffffffLL || out_stride > 0x7fffffffLL) return HB_UNSUPPORTED_SIZE;
    if (rows != 8 && rows != MOST_ROWS) return HB_UNSUPPORTED_SIZE;
    if (together && (together < 2 || together > MOST_TOGETHER || blocks % together || pieces || beside_tiles)) return HB_BAD_ARGUMENT;
    const int group = heads / kv_heads, gc = group < rows ? group : rows, chunks = (group + gc - 1) / gc;
    if ((long long)kv_heads * chunks > 65535) return HB_UNSUPPORTED_SIZE;
    const Args a{(const bf16*)q, (int)q_stride, (bf16*)out, (int)out_stride, (const signed char*)exponents, block_table, table_width, items, first_item, last, piece_start, own_start, pieces, (float2*)sums,
                 heads, kv_heads, page_size, pages, beside_tiles, together, gc, chunks, scale * 1.4426950408889634f, status};
    const auto launch = rows == 8 ? (exponents ? launch_strips<true, 1> : launch_strips<false, 1>) : (exponents ? launch_strips<true, 2> : launch_strips<false, 2>);
    if (int code = launch(a, cache, blocks, stream)) return code;
    return pieces ? hb_attention_pieces(pieces, sums, piece_start, out, out_stride, tokens, n_pieces, heads, stream) : 0;
}
