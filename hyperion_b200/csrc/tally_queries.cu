// The weights that many queries (a prompt, or its last tokens) give the slots that they see, summed over queries and over the query heads of a key/value head, added to the slots' weights:
//
//     y_vj = q_v . k_j scale log2(e),   m_v = max_j y_vj,   l_v = sum_j 2^(y_vj - m_v),   weights[j] += sum_v 2^(y_vj - m_v) / l_v
//
// v counts a request's (token, head) rows of a key/value head, token by token; token i of n sees the first length - n + i + 1 slots.  There is no result beside the weights, so values are not read.
//
// A weight is known only when its row's sum is, and a sum over rows has another owner than a row's, so the scores are made twice: the first walk goes along the slots and leaves m and 1 / l of every row,
// the second goes along the rows and adds up every slot's weights.  (Keeping them would move 8 bytes a score, against 2 d operations for making them again.)
//
// Both walks have one shape: a tile of 128 rows stays in shared memory (of Q; then of K), tiles of the other pass through a ring, and each pair is one product of 128 x 128 on the tensor cores (tcgen05) into
// one of two buffers of tensor memory.  The rows that stay are the product's lanes and what passes its columns, so one thread owns a row's maximum and sum, or a slot's sum, and nothing is exchanged.
// In the second walk a row's maximum and sum are part of the product: 16 more columns stand beside both tiles, 1 1 1 0 ... beside a slot and -(m + log2 l) / (scale log2 e) in three parts of bfloat16 beside a row,
// so that a thread takes 2^(c s) of what the product gives and adds it up.  (Read out of shared memory by all threads of a warp they cost more of its bandwidth than the products' operands: the second walk of three prompts 104 us, and 73 so.)
// A tile of Q has whole tokens: 128 / group of them with all heads of a key/value head, by one TMA box a panel.
//
// Where few rows would leave the device empty, the first walk's slots are cut, and its blocks leave (m, l) of every row and cut, which a small kernel puts together.  (By clusters of up to 16 cuts two requests' 8 queries of
// 1,000 slots take 11.0 us in place of 11.8, but 32 of 8,192 20.0 in place of 18.4 and 8 of 60,000 82 in place of 61.)  In the second walk a cluster's blocks share the tiles of Q that see a tile of slots, and read one
// another's sums in shared memory; where a request's rows are one tile, that stays, and the tiles of slots pass.  Nothing is added by atomics, so results do not depend on which block came first.
//
// Measured: three prompts of up to 2,047 tokens, 32 heads over 8 of 128, 123 us (both walks' products 0.6 PFLOP/s), of which either walk takes some 60.  In the loop a tile of 128 x 128 takes an SM
// 950 to 1,150 clocks: 576 of them are its products, 730 its exponentials on the special function unit (11 of 16 pairs), some 700 its instructions; blocks of two halves with a buffer each do not quite keep them all
// busy, and starts and ends of blocks cost another 15 %.  The last 32 of 8,192 tokens, 28 heads over 4: 18.6 us, three kernels' starts and trips to memory.  (With mma.sync and registers in place of tensor memory 890 and 49 us.)
//
// Slots beyond a request's length may hold anything: their scores are not looked at.  Every wait is bounded; one that runs out sets HB_STATUS_WAIT_EXPIRED and the block leaves, once the copies and products that it
// has on their way are done.
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
constexpr int BM = 128;                        // rows that stay, and rows that pass
constexpr int PANEL = BM * 128, PANELS = D / 64, TILE = PANELS * PANEL;  // bytes
constexpr int STAGES = D == 128 ? 2 : 4;       // of the ring: two blocks share an SM's memory
constexpr int MOST_SPANS = 16;                 // blocks that share the tiles of Q that pass a tile of slots, a cluster
constexpr int HALF = 4, PRODUCER = 2 * HALF, ISSUER = PRODUCER + 1, THREADS = 32 * (ISSUER + 1);  // warps that look at scores: four for each of the two buffers
constexpr int TMEM_COLS = 2 * BM;              // two blocks have all of an SM's
constexpr unsigned WAIT_LIMIT = HB_WAIT_LIMIT, LAST_WAIT_LIMIT = 1u << 24;
constexpr int BESIDE = 2 * BM * 16;            // bytes of a tile's 16 more columns: two groups of 8, rows of 16 bytes one behind the other (no swizzle)
constexpr size_t SMEM_BYTES = 1024 + (size_t)(TILE + BESIDE) * (1 + STAGES) + 2 * BM * 4 + 128;
static_assert(2 * (SMEM_BYTES + 1024) <= 228 * 1024, "an SM's shared memory");

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
__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, unsigned long long* bar, int x, int y, int z) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
                 ::"r"(smem_u32(dst)), "l"(map), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z) : "memory");
}

constexpr unsigned DESC_HIGH = (unsigned)(1024 >> 4) | (1u << 14) | (2u << 29);  // 8-row groups 1,024 bytes apart, sm_100 descriptor, 128-byte swizzle
constexpr unsigned IDESC = (1u << 4) | (1u << 7) | (1u << 10) | ((unsigned)(BM >> 3) << 17) | ((unsigned)(BM >> 4) << 24);  // float from bfloat16, both K-major, 128 x 128
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ unsigned low_k_major(const void* tile) { return ((smem_u32(tile) & 0x3FFFFu) >> 4) | (1u << 16); }
__device__ __forceinline__ void umma_commit_at(unsigned bar_addr) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar_addr) : "memory");
}
// The product of the 16 columns beside the tiles, added to what is there: two 8-column groups BM * 16 bytes apart, 8-row groups 128 bytes apart, no swizzle.
constexpr unsigned BESIDE_HIGH = (128u >> 4) | (1u << 14);
__device__ __forceinline__ unsigned beside_low(const void* tile) { return ((smem_u32(tile) & 0x3FFFFu) >> 4) | ((unsigned)(BM * 16 >> 4) << 16); }
__device__ __forceinline__ void umma_beside(unsigned tmem_d, unsigned a_low, unsigned b_low, unsigned idesc) {
    asm volatile(
        "{\n\t.reg .pred q;\n\t.reg .b64 da, db;\n\t"
        "setp.eq.b32 q, 0, 0;\n\t"
        "mov.b64 da, {%1, %4};\n\t"
        "mov.b64 db, {%2, %4};\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, q;\n\t}"
        ::"r"(tmem_d), "r"(a_low), "r"(b_low), "r"(idesc), "r"(BESIDE_HIGH) : "memory");
}
__device__ __forceinline__ bool elected() {  // one lane of the warp, all of which are here
    unsigned one;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(one));
    return one != 0;
}
// The product of a 64-entry panel of both tiles (4 of 16 entries); `first` = 0 starts a new one.
__device__ __forceinline__ void umma_s_panel(unsigned tmem_d, unsigned a_low, unsigned b_low, unsigned idesc, unsigned first) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t.reg .b64 da, db;\n\t.reg .b32 al, bl;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "setp.eq.b32 q, 0, 0;\n\t"
        "mov.b64 da, {%1, %5};\n\t"
        "mov.b64 db, {%2, %5};\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n\t"
        "add.u32 al, %1, 2;\n\t"
        "add.u32 bl, %2, 2;\n\t"
        "mov.b64 da, {al, %5};\n\t"
        "mov.b64 db, {bl, %5};\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, q;\n\t"
        "add.u32 al, %1, 4;\n\t"
        "add.u32 bl, %2, 4;\n\t"
        "mov.b64 da, {al, %5};\n\t"
        "mov.b64 db, {bl, %5};\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, q;\n\t"
        "add.u32 al, %1, 6;\n\t"
        "add.u32 bl, %2, 6;\n\t"
        "mov.b64 da, {al, %5};\n\t"
        "mov.b64 db, {bl, %5};\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, q;\n\t}"
        ::"r"(tmem_d), "r"(a_low), "r"(b_low), "r"(idesc), "r"(first), "r"(DESC_HIGH) : "memory");
}
// 32 consecutive columns of this thread's lane, on their way; arrived() says that they are there, and nothing that reads them can stand before it.
__device__ __forceinline__ void tmem_ld32(unsigned taddr, unsigned (&r)[32]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
                 : "r"(taddr));
}
__device__ __forceinline__ void arrived(unsigned (&r)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31]) :: "memory");
}
__device__ __forceinline__ float fast_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float max3(float a, float b, float c) {  // passes over a NaN, as fmaxf does
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// Two floats at a time.
struct Pair { float x, y; };
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
    Pair d;
    asm("{.reg .b64 a, b, c, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\tfma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}
__device__ __forceinline__ Pair add2(Pair a, Pair b) {
    Pair d;
    asm("{.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tadd.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}" : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ Pair mul2(Pair a, Pair b) {
    Pair d;
    asm("{.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmul.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}" : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ float max_nan(float a, float b) {
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}
// 2^y of a pair without the special function unit, which takes 8 clocks for a warp's 32 where the other units take half a one for each of these operations: y = n + f with n the nearest whole number (adding and
// taking away 1.5 * 2^23 rounds, and leaves n in the low bits), 2^f by the polynomial of degree 5 with the smallest relative error over [-1/2, 1/2] (7.5e-8; 2.1e-7 with its roundings), 2^n from its bits.  Below
// 2^-126 it is 0; a NaN stays one.  y at most 126.
__device__ __forceinline__ Pair polynomial_exp2(Pair y) {
    const Pair t{max_nan(y.x, -127.f), max_nan(y.y, -127.f)}, r = add2(t, Pair{12582912.f, 12582912.f}), n = add2(r, Pair{-12582912.f, -12582912.f}), f = fma2(n, Pair{-1.f, -1.f}, t);
    Pair p = fma2(f, Pair{1.3276472e-3f, 1.3276472e-3f}, Pair{9.675541e-3f, 9.675541e-3f});
    p = fma2(p, f, Pair{5.550713e-2f, 5.550713e-2f});
    p = fma2(p, f, Pair{0.2402212f, 0.2402212f});
    p = fma2(p, f, Pair{0.69314694f, 0.69314694f});
    p = fma2(p, f, Pair{1.0000001f, 1.0000001f});
    return mul2(p, Pair{__uint_as_float((__float_as_uint(r.x) << 23) + 0x3f800000u), __uint_as_float((__float_as_uint(r.y) << 23) + 0x3f800000u)});
}
// Of 16 pairs so many take the polynomial, spread evenly.  (Three prompts, none / 2 / 4 / 5 / 6: 132.3 / 126.0 / 123.3 / 122.9 / 126.5 us.)
constexpr int POLYNOMIAL = 5;
__device__ __forceinline__ Pair exp2_of(Pair y, int pair) { return (pair + 1) * POLYNOMIAL / 16 != pair * POLYNOMIAL / 16 ? polynomial_exp2(y) : Pair{fast_exp2(y.x), fast_exp2(y.y)}; }

// The blocks of a cluster.
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }
__device__ __forceinline__ float of_block(const float* p, int rank) {  // what another block of the cluster has at this place of its shared memory
    unsigned at;
    float v;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(p)), "r"(rank));
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
    return v;
}

struct Args {
    const int* block_table; int table_width;
    const int* starts;    // [requests + 1]
    const int* lengths;   // [requests]
    int tokens, most, longest;
    float* weights;       // [requests, kv_heads, capacity]
    int capacity;
    uint4* rows;          // [tokens * heads]: -(m + log2 l) / c in three parts of bfloat16, and zeros
    float2* cuts;         // [n_cuts, tokens * heads]: (m, l), where the slots are cut
    int n_cuts;
    int spans;            // blocks of a cluster, which share the tiles of Q that pass a tile of slots
    int heads, kv_heads, group, page_shift, pages;
    int per_tile;         // tokens of a tile of Q
    float scale_log2;
    int* status;
};
struct Request {
    int first, tokens, length, before;  // its queries, its slots; query i sees the first before + i + 1 of them
};
__device__ __forceinline__ Request request_of(const Args& a, int r, bool reports) {
    const int from = a.starts[r], to = a.starts[r + 1], length = a.lengths[r];
    if (0 <= from && from <= to && to <= a.tokens && to - from <= a.most && 0 <= length && length <= a.longest) return {from, to - from, length, length - (to - from)};
    // What is beyond the bounds or not there is left out; the queries that remain see what they would see without the bounds, up to `longest`.  (In 64 bits, which takes 0.3 us where all calls go through it.)
    if (reports) atomicOr(a.status, HB_STATUS_BAD_POSITION);
    const long long first = min(max(from, 0), a.tokens), tokens = min(max(min(to, a.tokens) - first, 0LL), (long long)a.most);
    const long long before = (long long)length - ((long long)to - from) + (first - from);  // beyond the next line's bounds every query sees nothing, or everything
    return {(int)first, (int)tokens, min(max(length, 0), a.longest), (int)min(max(before, -tokens), (long long)a.longest)};
}
// What stands beside a row: -(m + log2 l) / c in three parts, which together hold a float's 24 bits.  A row without a score that counts has -infinity, and gives nothing.
__device__ __forceinline__ unsigned half_word(float v) { return __bfloat16_as_ushort(__float2bfloat16_rn(v)); }
__device__ __forceinline__ uint4 beside_row(float m, float l, float c) {
    const float x = l == 0.f ? -INFINITY : -(m + log2f(l)) / c;
    const unsigned hi = half_word(x);
    unsigned mid = 0, lo = 0;
    if (fabsf(x) < INFINITY) {
        const float rest = x - __uint_as_float(hi << 16);
        mid = half_word(rest), lo = half_word(rest - __uint_as_float(mid << 16));
    }
    return make_uint4(hi | mid << 16, lo, 0, 0);
}
__device__ __forceinline__ int first_tile(const Args& a, int slot, int before) { return max(0, slot - before) / a.per_tile; }  // token slot - before is the first that sees the slot

// One walk, the first or the second (SECOND).  KEYS_STAY: block (span of the tiles of Q within tile of slots, key/value head, request), tiles of Q pass; else block (tile of Q and key/value head, cut, request), tiles of K pass.
// The second walk has the slots as the product's lanes either way: where a request's rows are one tile, that tile may stay and the slots pass.
template <bool KEYS_STAY, bool SECOND>
__global__ void __launch_bounds__(THREADS, 2) tally_walk_kernel(const __grid_constant__ CUtensorMap kv_map, const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap rows_map, const Args a) {
    extern __shared__ unsigned char smem_raw[];
    static_assert(SECOND || !KEYS_STAY, "rows stay in the first walk");
    unsigned char* stays = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    unsigned char* ring = stays + TILE;
    unsigned char* beside_stays = ring + STAGES * TILE;              // SECOND
    unsigned char* beside = beside_stays + BESIDE;                   // SECOND: [STAGES], or one for all slots' tiles
    float* theirs = reinterpret_cast<float*>(beside + STAGES * BESIDE);  // [2][BM]: what one half of the warps tells the other
    unsigned long long* full = reinterpret_cast<unsigned long long*>(theirs + 2 * BM);
    unsigned long long* empty = full + STAGES;
    unsigned long long* s_full = empty + STAGES;  // [2]
    unsigned long long* s_empty = s_full + 2;     // [2]
    unsigned long long* stays_full = s_empty + 2;
    unsigned long long* all_done = stays_full + 1;
    unsigned* tmem_slot = reinterpret_cast<unsigned*>(all_done + 1);
    volatile int* failed = reinterpret_cast<volatile int*>(tmem_slot + 1);

    constexpr bool SLOTS_PASS = SECOND && !KEYS_STAY;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, request = blockIdx.z;
    if (tid == 0) {
        for (int s = 0; s < STAGES; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
        for (int b = 0; b < 2; ++b) { mbar_init(&s_full[b], 1); mbar_init(&s_empty[b], HALF); }
        mbar_init(stays_full, 1), mbar_init(all_done, 1);
        *failed = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&kv_map) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&q_map) : "memory");
        if (SECOND) asm volatile("prefetch.tensormap [%0];" ::"l"(&rows_map) : "memory");
    }
    if (!KEYS_STAY) wait_for_previous_kernels();
    const int kvh = KEYS_STAY ? blockIdx.y : blockIdx.x % a.kv_heads, group = a.group;
    const Request r = request_of(a, request, !SECOND && blockIdx.x == 0 && blockIdx.y == 0 && tid == 0);
    const int before = r.before;
    const int q_tiles = (r.tokens + a.per_tile - 1) / a.per_tile;
    const int base = KEYS_STAY ? blockIdx.x / a.spans * BM : (int)(gridDim.x / a.kv_heads - 1 - blockIdx.x / a.kv_heads) * a.per_tile;  // the first slot, or the first token, that stays
    int from, to;  // tiles that pass
    if (KEYS_STAY) {
        from = first_tile(a, base, before), to = q_tiles;
        const int see = to - from;  // tiles that see any of the slots
        if (base >= r.length || see <= 0) {  // the same for all blocks of a cluster
            wait_for_previous_kernels();     // whoever comes next takes this kernel's end as the end of all
            return;
        }
        if (a.spans > 1) {
            const int span = blockIdx.x % a.spans;
            to = from + see * (span + 1) / a.spans, from += see * span / a.spans;  // at most 2^24 tiles: tokens * heads fit 31 bits
        }
    } else {
        if (base >= r.tokens) return;
        const int reach = min(r.length, max(0, before + min(base + a.per_tile, r.tokens))), n = (reach + BM - 1) / BM;  // slots that any of the tokens sees
        from = (int)((long long)n * blockIdx.y / a.n_cuts), to = (int)((long long)n * (blockIdx.y + 1) / a.n_cuts);
    }
    const int n_tiles = to - from;
    // rows of Q's tiles that no copy writes (beyond whole tokens)
    const int q_rows = a.per_tile * group;
    for (int e = tid; e < (BM - q_rows) * 8 * PANELS * (KEYS_STAY ? STAGES : 1); e += THREADS) {
        const int chunk = e & 7, row = q_rows + (e >> 3) % (BM - q_rows), panel = (e >> 3) / (BM - q_rows);
        reinterpret_cast<uint4*>((KEYS_STAY ? ring : stays) + panel * PANEL + row * 128)[chunk] = make_uint4(0, 0, 0, 0);
    }
    if (SECOND) {
        for (int e = tid; e < 2 * BM * (KEYS_STAY ? 1 + STAGES : 2); e += THREADS) {
            const int row = e % BM, second = e / BM & 1, tile = e / (2 * BM);  // the first tile is what stays
            const bool slots = KEYS_STAY == (tile == 0);
            uint4 x = make_uint4(0, 0, 0, 0);
            if (!second && slots) x = make_uint4(0x3f803f80u, 0x3f80u, 0, 0);  // 1 1 1 0 ...
            if (second || slots || row >= q_rows) reinterpret_cast<uint4*>(beside_stays)[e] = x;
        }
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncthreads();
    const int page_size = 1 << a.page_shift, pages_per_tile = BM >> a.page_shift;
    const int* table = a.block_table + (size_t)request * a.table_width;
    auto page_at = [&](int slot0) {  // this lane's page of the tile of K from slot0 on; -1: none
        const int k0 = slot0 + lane * page_size;
        if (lane >= pages_per_tile || k0 >= r.length) return -1;
        const int id = table[k0 >> a.page_shift];
        if (id >= 0 && id < a.pages) return id;
        atomicOr(a.status, HB_STATUS_BAD_PAGE);
        return -1;
    };
    auto fetch_keys = [&](unsigned char* tile, int page, unsigned long long* bar) {
        const unsigned valid = __popc(__ballot_sync(0xffffffffu, page >= 0));
        if (lane == 0) {
            if (valid) mbar_expect_tx(bar, valid * page_size * D * 2u); else mbar_arrive(bar);
        }
        __syncwarp();
        const int ops = pages_per_tile * PANELS;  // at most 32
        const int p = min(lane, ops - 1) / PANELS, h = lane % PANELS, id = __shfl_sync(0xffffffffu, page, p);
        if (lane < ops && id >= 0) tma_load_2d(tile + h * PANEL + p * page_size * 128, &kv_map, bar, h * 64, (id * 2 * a.kv_heads + kvh) << a.page_shift);
    };
    // The second walk's tile is on its way while the first one ends: its blocks are let in once all of the first walk's have waited, so what came before that one has finished.
    if (KEYS_STAY) {
        if (warp == PRODUCER && n_tiles > 0) fetch_keys(stays, page_at(base), stays_full);
        wait_for_previous_kernels();
    }
    // Tensor memory is taken only now that the kernels before have finished, and the next kernel is let in only once it is: a block further back or further on that holds some while it waits could wait for this one.
    if (warp == ISSUER) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    let_next_kernel_start();
    tc_fence_after();
    const unsigned tmem = *tmem_slot;

    if (warp == PRODUCER) {
        // ------------------------------------------------------------------ the whole warp
        auto fetch_queries = [&](unsigned char* tile, int token, unsigned long long* bar) {  // tokens beyond the request's own come along, or are filled with zeros
            if (lane == 0) {
                mbar_expect_tx(bar, (unsigned)((PANELS * 128 + (SECOND ? 16 : 0)) * q_rows));
                for (int h = 0; h < PANELS; ++h) tma_load_3d(tile + h * PANEL, &q_map, bar, h * 64, kvh * group, r.first + token);
                if (SECOND) tma_load_3d(KEYS_STAY ? beside + (tile - ring) / TILE * BESIDE : beside_stays, &rows_map, bar, 0, kvh * group, r.first + token);
            }
        };
        int sent = 0;
        if (n_tiles > 0) {
            if (!KEYS_STAY) fetch_queries(stays, base, stays_full);
            int page = KEYS_STAY ? 0 : page_at(from * BM);
            for (int i = 0; i < n_tiles; ++i, ++sent) {
                const int s = i % STAGES;
                if (!__all_sync(0xffffffffu, mbar_wait(&empty[s], ((i / STAGES) & 1) ^ 1, failed))) { *failed = 1; break; }
                if (KEYS_STAY) {
                    fetch_queries(ring + s * TILE, (from + i) * a.per_tile, &full[s]);
                } else {
                    fetch_keys(ring + s * TILE, page, &full[s]);
                    page = i + 1 < n_tiles ? page_at((from + i + 1) * BM) : -1;
                }
            }
            if (lane == 0) {
                mbar_last_wait(stays_full, 0);
                for (int k = max(0, sent - STAGES); k < sent; ++k) mbar_last_wait(&full[k % STAGES], (k / STAGES) & 1);
            }
            __syncwarp();
        }
    } else if (warp == ISSUER) {
        // ------------------------------------------------------------------ the warp stays together, so that descriptors are its common values; one elected lane issues
        const unsigned a_low = low_k_major(stays), b_low0 = low_k_major(ring);
        auto wait_for = [&](unsigned long long* bar, int phase) { return __all_sync(0xffffffffu, mbar_wait(bar, phase & 1, failed)) != 0; };
        bool ok = n_tiles == 0 || wait_for(stays_full, 0);
        for (int i = 0; i < n_tiles && ok; ++i) {
            const int s = i % STAGES, b = i & 1;
            ok = wait_for(&full[s], i / STAGES) && wait_for(&s_empty[b], (i >> 1) ^ 1);
            if (!ok) break;
            tc_fence_after();
            if (elected()) {
                const unsigned b_low = b_low0 + (unsigned)s * (TILE >> 4);
#pragma unroll
                for (int h = 0; h < PANELS; ++h) umma_s_panel(tmem + b * BM, (SLOTS_PASS ? b_low : a_low) + h * (PANEL >> 4), (SLOTS_PASS ? a_low : b_low) + h * (PANEL >> 4), IDESC, h ? 1u : 0u);
                if (SLOTS_PASS) umma_beside(tmem + b * BM, beside_low(beside), beside_low(beside_stays), IDESC);
                else if (KEYS_STAY) umma_beside(tmem + b * BM, beside_low(beside_stays), beside_low(beside) + (unsigned)s * (BESIDE >> 4), IDESC);
                umma_commit_at(smem_u32(&empty[s]));
                umma_commit_at(smem_u32(&s_full[b]));
            }
            __syncwarp();
        }
        if (!ok) *failed = 1;
        if (elected()) umma_commit_at(smem_u32(all_done));
        __syncwarp();
        mbar_last_wait(all_done, 0);
    } else {
        // ------------------------------------------------------------------ four warps a buffer: a thread has a lane of the product, 32 columns of it at a time
        const int half = warp / HALF, mine = (warp & 3) * 32 + lane;
        const unsigned lanes = tmem + half * BM + ((unsigned)((warp & 3) * 32) << 16);
        const float c = a.scale_log2;
        bool ok = true;
        [[maybe_unused]] float m = -INFINITY, l = 0.f;         // of this thread's row
        [[maybe_unused]] float sum = 0.f, rest = 0.f;          // of this thread's slot, and what its additions lost
        const int my_token = mine / group, my_head = kvh * group + mine - my_token * group;
        [[maybe_unused]] const int token = base + my_token;
        [[maybe_unused]] const int sees = token < r.tokens && mine < q_rows ? min(r.length, before + token + 1) : 0;
        [[maybe_unused]] const int all_see = min(r.length, before + base + 1);  // slots that every row of the tile sees
        for (int i = half; i < n_tiles; i += 2) {
            if (!__all_sync(0xffffffffu, mbar_wait(&s_full[half], (i >> 1) & 1, failed))) {
                *failed = 1, ok = false;
                break;
            }
            tc_fence_after();
            const int slot0 = KEYS_STAY ? base : (from + i) * BM, token0 = KEYS_STAY ? (from + i) * a.per_tile : base;
            // SECOND: the first row that sees this slot, and the rows that are the request's; whether all rows see all slots
            [[maybe_unused]] const int from_row = max(0, slot0 + mine - before - token0) * group, rows = min((r.tokens - token0) * group, q_rows);
            const bool all = SECOND ? slot0 + BM - 1 - before <= token0 && r.tokens - token0 >= a.per_tile : slot0 + BM <= all_see;
            // SECOND: a row that does not see this slot gives it nothing, whatever the row is, nor does one that is none, whose zeros a key's infinity has made a NaN of: the first columns, by 32, that need not be asked
            [[maybe_unused]] const int whole = all ? q_rows / 32 : 0;
            Pair part[2] = {{0.f, 0.f}, {0.f, 0.f}};
            if constexpr (SLOTS_PASS) {  // rows are few: of the product's columns those that are rows are looked at, 32 at a time
                float* weight = a.weights + ((size_t)request * a.kv_heads + kvh) * a.capacity + slot0 + mine;
                const float old = slot0 + mine < r.length ? *weight : 0.f;
                const int chunks = (rows + 31) / 32;
#pragma unroll 1
                for (int k = 0; k < chunks; ++k) {
                    unsigned v[32];
                    tmem_ld32(lanes + 32 * k, v);
                    arrived(v);
                    if (k + 1 == chunks) {
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&s_empty[half]);
                    }
                    if (k >= whole) {
#pragma unroll
                        for (int j = 0; j < 32; ++j)
                            if (32 * k + j < from_row || 32 * k + j >= rows) v[j] = 0xff800000u;
                    }
#pragma unroll
                    for (int j = 0; j < 32; j += 4)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const Pair y = fma2(Pair{__uint_as_float(v[j + 2 * e]), __uint_as_float(v[j + 2 * e + 1])}, Pair{c, c}, Pair{0.f, 0.f});
                            part[e] = add2(part[e], Pair{fast_exp2(y.x), fast_exp2(y.y)});
                        }
                }
                if (slot0 + mine < r.length) *weight = old + ((part[0].x + part[0].y) + (part[1].x + part[1].y));
                continue;
            }
            unsigned raw[2][32];
            tmem_ld32(lanes, raw[0]);
            arrived(raw[0]);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                unsigned (&v)[32] = raw[k & 1];
                if (k < 3) tmem_ld32(lanes + 32 * (k + 1), raw[(k + 1) & 1]);
                auto pair_at = [&](int j) { return Pair{__uint_as_float(v[j]), __uint_as_float(v[j + 1])}; };
                if constexpr (KEYS_STAY) {
                    if (k >= whole) {
#pragma unroll
                        for (int j = 0; j < 32; ++j)
                            if (32 * k + j < from_row || 32 * k + j >= rows) v[j] = 0xff800000u;
                    }
#pragma unroll
                    for (int j = 0; j < 32; j += 4)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const Pair y = fma2(pair_at(j + 2 * e), Pair{c, c}, Pair{0.f, 0.f});
                            part[e] = add2(part[e], exp2_of(y, j / 2 + e));
                        }
                } else {
                    if (!all) {
#pragma unroll
                        for (int j = 0; j < 32; ++j)
                            if (slot0 + 32 * k + j >= sees) v[j] = 0xff800000u;
                    }
                    float top = -INFINITY, other = -INFINITY;
#pragma unroll
                    for (int j = 0; j < 32; j += 4) {
                        top = max3(top, pair_at(j).x, pair_at(j).y), other = max3(other, pair_at(j + 2).x, pair_at(j + 2).y);
                    }
                    const float above = fmaxf(m, fmaxf(top, other) * c), low = above == -INFINITY ? 0.f : above;  // c is above 0
                    l *= m == -INFINITY ? 1.f : fast_exp2(m - low);  // nothing but zeros and NaN has been added up below -infinity
                    m = above;
                    part[0] = part[1] = Pair{0.f, 0.f};
#pragma unroll
                    for (int j = 0; j < 32; j += 4)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const Pair y = fma2(pair_at(j + 2 * e), Pair{c, c}, Pair{-low, -low});
                            part[e] = add2(part[e], exp2_of(y, j / 2 + e));
                        }
                    l += (part[0].x + part[0].y) + (part[1].x + part[1].y);
                }
                if (k < 3) arrived(raw[(k + 1) & 1]);
                if (k == 2) {
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&s_empty[half]);
                }
            }
            if constexpr (KEYS_STAY) {
                // added up with what is lost: a slot that thousands of rows see would be off by more than all else
                const float y = (part[0].x + part[0].y) + (part[1].x + part[1].y) - rest, t = sum + y;
                rest = (t - sum) - y, sum = t;
            }
        }
        if constexpr (!SLOTS_PASS) {
            // the second half's sums come to the first
            if (half == 1) theirs[mine] = KEYS_STAY ? sum : m, theirs[BM + mine] = KEYS_STAY ? rest : l;
            asm volatile("bar.sync 3, %0;" ::"n"(64 * HALF) : "memory");
            if (half == 0 && ok) {
                if constexpr (KEYS_STAY) {
                    sum += theirs[mine] - (rest + theirs[BM + mine]);
                    if (a.spans > 1) theirs[mine] = sum;
                    else if (base + mine < r.length) a.weights[((size_t)request * a.kv_heads + kvh) * a.capacity + base + mine] += sum;
                } else if (mine < q_rows && token < r.tokens) {
                    const float other = theirs[mine], above = fmaxf(m, other);
                    l = (m == -INFINITY ? l : l * fast_exp2(m - above)) + (other == -INFINITY ? theirs[BM + mine] : theirs[BM + mine] * fast_exp2(other - above));
                    const size_t at = (size_t)(r.first + token) * a.heads + my_head;
                    if (a.n_cuts == 1) a.rows[at] = beside_row(above, l, c);
                    else a.cuts[(size_t)blockIdx.y * a.tokens * a.heads + at] = make_float2(above, l);
                }
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (tid == 0 && *failed) atomicOr(a.status, HB_STATUS_WAIT_EXPIRED | HB_STATUS_IN_TALLY_QUERIES);
    if (warp == ISSUER) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM_COLS) : "memory");
    }
    if constexpr (KEYS_STAY) {
        // The spans' sums of a slot, in their order.  Tensor memory has been given back, so that no block has some while it waits for another.
        if (a.spans > 1) {
            const int rank = blockIdx.x % a.spans, slot = rank + tid * a.spans;  // whose sums this thread adds up
            const bool adds = slot < BM && base + slot < r.length;
            float* weight = a.weights + ((size_t)request * a.kv_heads + kvh) * a.capacity + base + slot;
            const float old = adds ? *weight : 0.f;
            cluster_arrive(), cluster_wait();
            if (adds) {
                float part[MOST_SPANS], sum = 0.f;
#pragma unroll
                for (int k = 0; k < MOST_SPANS; ++k) part[k] = k < a.spans ? of_block(theirs + slot, k) : 0.f;
#pragma unroll
                for (int k = 0; k < MOST_SPANS; ++k) sum += part[k];
                *weight = old + sum;
            }
            cluster_arrive(), cluster_wait();  // the sums have been read
        }
    }
}

// Puts the cuts of a row together: `lanes` threads of a warp a row, a power of two, so that all of a row's cuts are on their way at once (32 cuts by one thread a row took 7 us).
__global__ void __launch_bounds__(256) tally_cuts_kernel(const Args a, int lanes) {
    let_next_kernel_start();
    wait_for_previous_kernels();
    const int n = a.tokens * a.heads, at = (blockIdx.x * 256 + threadIdx.x) / lanes, mine = threadIdx.x % lanes;
    float top = -INFINITY, all = 0.f;
    for (int c = mine; at < n && c < a.n_cuts; c += lanes) {
        const float2 ml = a.cuts[(size_t)c * n + at];
        const float above = fmaxf(top, ml.x);
        all = above == -INFINITY ? all + ml.y : fmaf(ml.x == -INFINITY ? 0.f : fast_exp2(ml.x - above), ml.y, all * (top == -INFINITY ? 0.f : fast_exp2(top - above)));
        top = above;
    }
    float above = top;
    for (int offset = 1; offset < lanes; offset <<= 1) above = fmaxf(above, __shfl_xor_sync(0xffffffffu, above, offset));
    if (top != -INFINITY) all *= fast_exp2(top - above);
    for (int offset = 1; offset < lanes; offset <<= 1) all += __shfl_xor_sync(0xffffffffu, all, offset);
    if (mine == 0 && at < n) a.rows[at] = beside_row(above, all, a.scale_log2);
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
int encoded(CUtensorMap* map, const void* base, int rank, const cuuint64_t* dims, const cuuint64_t* strides, const cuuint32_t* box, CUtensorMapSwizzle swizzle = CU_TENSOR_MAP_SWIZZLE_128B) {
    EncodeTiled encode = encode_tiled();
    if (!encode) return HB_BAD_ARGUMENT;
    const cuuint32_t elem[3] = {1, 1, 1};
    return encode(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, rank, const_cast<void*>(base), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS ? 0 : HB_BAD_ARGUMENT;
}
template <bool KEYS_STAY, bool SECOND>
int launch_walk(const CUtensorMap& kv_map, const CUtensorMap& q_map, const CUtensorMap& rows_map, const Args& a, dim3 grid, int together, cudaStream_t stream) {  // blocks of a cluster, along x
    static std::atomic<unsigned long long> allowed{0};
    if (const cudaError_t error = allow_shared((const void*)tally_walk_kernel<KEYS_STAY, SECOND>, SMEM_BYTES, allowed)) return (int)error;
    static std::atomic<unsigned long long> wide{0};
    if (together > 8)
        if (const cudaError_t error = allow_wide_clusters((const void*)tally_walk_kernel<KEYS_STAY, SECOND>, wide)) return (int)error;
    cudaLaunchConfig_t config = {};
    config.gridDim = grid, config.blockDim = dim3(THREADS), config.dynamicSmemBytes = SMEM_BYTES, config.stream = stream;
    cudaLaunchAttribute attributes[2];
    attributes[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attributes[0].val.programmaticStreamSerializationAllowed = overlap_launches() ? 1 : 0;
    attributes[1].id = cudaLaunchAttributeClusterDimension;
    attributes[1].val.clusterDim = {(unsigned)together, 1, 1};
    config.attrs = attributes, config.numAttrs = together > 1 ? 2 : 1;
    return (int)cudaLaunchKernelEx(&config, tally_walk_kernel<KEYS_STAY, SECOND>, kv_map, q_map, rows_map, a);
}
}  // namespace

// Into how many cuts the first walk's slots go: as many as give the device two blocks an SM, of two tiles at least, and none up to four tiles, where the kernel that puts cuts together would cost more than it saves.  (us,
// 28 heads over 4 of 128, tiles a cut at least 1 / 2 / 4: 8 queries of 300 slots, three tiles, 10.9 / 11.3 / 10.6 where 4 leaves one cut; 16 of 1,000 10.8 / 11.5 / 13.5; 32 of 8,192 21.6 / 20.6 / 19.0; 14 over 2 of 64, 32 of
// 8,192 19.4 / 14.8 / 14.6; four requests' 32 of 2,048 14.2 / 12.4 / 13.6.)
static int cuts_for(int requests, int most, int longest, int heads, int kv_heads, int sms) {
    const int per_tile = BM / (heads / kv_heads), tiles = (longest + BM - 1) / BM;
    const long long blocks = (long long)((most + per_tile - 1) / per_tile) * kv_heads * requests, wanted = 2LL * sms / (blocks ? blocks : 1), most_cuts = tiles <= 4 ? 1 : (tiles + 1) / 2;
    return (int)(wanted < 1 ? 1 : wanted < most_cuts ? wanted : most_cuts);
}
// Blocks of the second walk that share the tiles of Q that pass a tile of slots.  A block takes the time of its tiles and of some three more, for its start, and longer the more blocks an SM has, from 0.7 on: of some sizes the one
// with the smallest such product.  Even ones, because an SM holds two, and no 10 to 14, of which few fit a group of SMs.  (us, one / two / four / six / eight / 16 blocks, the one that is taken in brackets: 14 heads over 2 of
// 64, a prompt of 300 tokens 21.9 / 16.9 / 13.4 / 12.5 / 11.7 / [11.1], of 895 43.7 / 30.1 / 23.0 / 20.4 / [18.7] / 19.7; 28 over 4 of 128, 500 tokens 32.0 / 23.0 / 18.6 / [16.6] / 17.5 / 20.8, three prompts of 700 46.2 /
// 35.2 / [34.3] / 36.2 / 39.1 / 56.5; 32 over 8 of 128, three of 2,047 127.5 / [123.5] / 135.4 / 153.9 / 173.5 / 266.5.  Over 85 sizes it comes within 1 % of the best on average.)
static int spans_for(int requests, int most, int longest, int heads, int kv_heads, int sms) {
    const int per_tile = BM / (heads / kv_heads), tiles = (most + per_tile - 1) / per_tile;
    const float blocks = (float)((longest + BM - 1) / BM) * (float)kv_heads * (float)requests;
    int best = 1;
    float least = INFINITY;
    for (int n : {1, 2, 4, 6, 8, MOST_SPANS}) {
        if (n > tiles) break;
        const float crowd = blocks * (float)n / (float)sms - 0.7f, cost = ((float)tiles / (float)n + 3.f) * (1.f + 0.8f * (crowd > 0.f ? crowd : 0.f));
        if (cost < least) least = cost, best = n;
    }
    return best;
}
// Bytes of scratch that hb_tally_queries takes.
HB_EXPORT long long hb_tally_queries_scratch(int tokens, int requests, int most, int longest, int heads, int kv_heads, int sms) {
    if (tokens <= 0 || requests <= 0 || most <= 0 || longest <= 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads || heads / kv_heads > BM || sms <= 0) return 0;
    const int cuts = cuts_for(requests, most, longest, heads, kv_heads, sms);
    return 16LL * tokens * heads + (cuts > 1 ? 8LL * tokens * heads * cuts : 0);
}
// q [tokens, heads * D] with rows q_stride apart, request r's from starts[r] to starts[r + 1] - 1, at most `most`, the last of which stands in its last slot; cache [pages, 2, kv_heads, page_size, D];
// lengths [requests], at most `longest`, which table and capacity hold; weights [requests, kv_heads, capacity].  scratch: hb_tally_queries_scratch bytes on a 16-byte boundary.
HB_EXPORT int hb_tally_queries(const void* q, long long q_stride, int tokens, const void* cache, const int* block_table, int table_width, const int* starts, const int* lengths, int requests, int most,
                               int longest, float* weights, int capacity, int heads, int kv_heads, int page_size, int pages, float scale, int sms, void* scratch, int* status, cudaStream_t stream) {
    if (requests <= 0 || tokens <= 0) return 0;
    if (!q || !cache || !block_table || !starts || !lengths || !weights || !scratch || !status) return HB_BAD_ARGUMENT;
    if (kv_heads <= 0 || heads <= 0 || heads % kv_heads || pages <= 0 || table_width <= 0 || longest <= 0 || most <= 0 || capacity < longest || sms <= 0 || q_stride % 8 || !(scale >= 0x1p-100f && scale <= 0x1p127f)) return HB_BAD_ARGUMENT;
    if (page_size < 8 || page_size > 64 || (page_size & (page_size - 1)) || heads / kv_heads > BM) return HB_UNSUPPORTED_SIZE;
    if ((((uintptr_t)q | (uintptr_t)cache) & 15) || ((uintptr_t)scratch & 15) || (long long)table_width * page_size < longest) return HB_BAD_ARGUMENT;
    const int group = heads / kv_heads, per_tile = BM / group;
    if (q_stride > 0x7fffffffLL || (long long)tokens * heads > 0x7fffffffLL - 256 || (long long)longest + tokens > 0x7fffffff - BM || requests > 65535 || kv_heads > 65535) return HB_UNSUPPORTED_SIZE;
    if ((long long)pages * 2 * kv_heads * page_size > 0x7fffffffLL) return HB_UNSUPPORTED_SIZE;  // a row's number in the cache's tensor map
    const long long row_blocks = (long long)((most + per_tile - 1) / per_tile) * kv_heads;
    if (row_blocks > 0x7fffffffLL || sms > 16384) return HB_UNSUPPORTED_SIZE;
    const int cuts = cuts_for(requests, most, longest, heads, kv_heads, sms), spans = spans_for(requests, most, longest, heads, kv_heads, sms), slot_tiles = (longest + BM - 1) / BM;
    if ((long long)slot_tiles * spans > 0x7fffffffLL) return HB_UNSUPPORTED_SIZE;
    CUtensorMap kv_map, q_map, rows_map;
    const cuuint64_t kv_dims[2] = {(cuuint64_t)D, (cuuint64_t)pages * 2 * kv_heads * page_size}, kv_strides[1] = {(cuuint64_t)D * 2};
    const cuuint32_t kv_box[2] = {64, (cuuint32_t)page_size};
    if (int code = encoded(&kv_map, cache, 2, kv_dims, kv_strides, kv_box)) return code;
    // a single row has no stride of its own
    const cuuint64_t q_dims[3] = {(cuuint64_t)D, (cuuint64_t)heads, (cuuint64_t)tokens}, q_strides[2] = {(cuuint64_t)D * 2, (cuuint64_t)(tokens > 1 ? q_stride : (long long)heads * D) * 2};
    const cuuint32_t q_box[3] = {64, (cuuint32_t)group, (cuuint32_t)per_tile};
    if (int code = encoded(&q_map, q, 3, q_dims, q_strides, q_box)) return code;
    uint4* rows = (uint4*)scratch;
    const cuuint64_t rows_dims[3] = {8, (cuuint64_t)heads, (cuuint64_t)tokens}, rows_strides[2] = {16, (cuuint64_t)heads * 16};
    const cuuint32_t rows_box[3] = {8, (cuuint32_t)group, (cuuint32_t)per_tile};
    if (int code = encoded(&rows_map, rows, 3, rows_dims, rows_strides, rows_box, CU_TENSOR_MAP_SWIZZLE_NONE)) return code;
    float2* cut_sums = (float2*)(rows + (size_t)tokens * heads);
    const Args a{block_table, table_width, starts, lengths, tokens, most, longest, weights, capacity, rows, cut_sums, cuts, spans, heads, kv_heads, group, __builtin_ctz(page_size), pages, per_tile,
                 scale * 1.4426950408889634f, status};
    if (int code = launch_walk<false, false>(kv_map, q_map, rows_map, a, dim3((unsigned)row_blocks, cuts, requests), 1, stream)) return code;
    if (cuts > 1) {
        int lanes = 2;
        while (lanes < 32 && lanes < cuts) lanes *= 2;
        const long long threads = (long long)tokens * heads * lanes;
        if (threads > 0x7fffffffLL - 256) return HB_UNSUPPORTED_SIZE;
        if (int code = launch_after_previous(tally_cuts_kernel, dim3((unsigned)((threads + 255) / 256)), dim3(256), 0, stream, a, lanes)) return code;
    }
    // Where a request's rows are one tile, a block of the second walk goes on from tile of slots to tile of slots, if there are more of those than SMs (us, by a block each / so: three queries of 16,384 slots, 14 heads over 2 of 64,
    // 256 tiles, 14.3 / 12.2, 28 over 4 of 128, 512 tiles, 22.9 / 17.0, 16 over 16 of 64, 2,048 tiles, 55.6 / 25.4; five of 60,000, 32 over 8, 3,752 tiles, 103 / 52; eight requests' five of 300, 28 over 4, 96 tiles, 11.6 /
    // 13.2).  More tiles of rows one after the other gain nothing up to some 700 tiles of slots.
    if (row_blocks == kv_heads && (long long)slot_tiles * kv_heads * requests > sms) return launch_walk<false, true>(kv_map, q_map, rows_map, a, dim3(kv_heads, cuts, requests), 1, stream);
    return launch_walk<true, true>(kv_map, q_map, rows_map, a, dim3(slot_tiles * spans, kv_heads, requests), spans, stream);
}
HB_EXPORT int hb_tally_queries_packed(const void* arguments) { return call_packed(&hb_tally_queries, arguments); }
