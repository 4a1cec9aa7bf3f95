// Attention behind shared positions on the 5th-generation tensor cores: items of many rows (attention_shared.cu has the items, the pieces they leave and the kernel
// for few rows), over paged caches of bfloat16 and of 8-bit records (cache8.cu), head sizes 64 and 128 (HB_HEAD_DIM), pages of 8 to 64 tokens.
//
// An item is up to 256 (token, head) rows of one key/value head and a range of keys: all of a group's tokens over a share of the positions that they
// hold in common, or a portion of a prompt over its own.  One block per SM holds all of the SM's tensor memory and takes its share of the items; two
// halves of 128 rows (H and L) walk the same tiles of 128 keys, so that the tensor core runs one half's products under the other half's softmax:
//   warp 0       fetches: over bfloat16 caches one cp.async.bulk.tensor per page and 64-column panel of K and of V, over operands one plain copy of each, and the queries as
//                one 3-D box per panel;
//   warp 1       issues S_x = Q_x K^T (M 128, N 128) and O_x += P_x V (P from tensor memory, V MN-major), each half's next S right behind its last product;
//   warps 4-11   softmax, a row per thread: running maximum and sum in float, O rescaled only when the maximum has grown by much.
// 8-bit records are made into operands before (shared_operands_kernel).
//
// Weights go to the second product in two parts, cut off to bfloat16 and what that left over: rounded once they would cost the result as
// much as its own rounding does.  8-bit values are bfloat16 numbers as they are (code * 2^e).  (As float16, which holds codes exactly and weights in one part, a tile took a tenth less: 256 requests behind
// 16,384 positions 128 us against 146, a portion of 1,000 tokens of 5,000 66 against 71.  But weights below 2^-25 of the largest were lost and those below 2^-14 cut short, and behind a
// key that takes nearly all of a row's weight and brings nothing to an entry, the entry is made of thousands of those.)  A row of S is 128 float columns of tensor memory and the two
// parts of its P are 2 x 64, so P takes exactly the place of the S it was made from, 32 keys at a time; the softmax reads S twice (for the maximum, then for the weights), 32
// columns under way while it works on 32.  P is handed over in two halves of the tile's keys, so that the product of the first runs under the making of the second.
// What bounds it is the chain of a half: from the arrival of S 2,750 clocks until the last weights are handed over (of which 1,024 are the special function unit's for 128 columns,
// which the other half's want as well), then 1,390 for the rest of O += P V, the next S and its arrival.  4,100 clocks a tile, of which the tensor core is busy for 3,072.
// Tried and dropped, with weights as float16 and 3,600 clocks a tile: weights by the maximum so far with one reading of S (3,150 clocks as long as no maximum is outgrown, 5,000 when one of
// 256 rows' is, and one often is); a part of the exponentials by a polynomial (no faster); two threads a row (4,700); an issuer for each half (the halves fall into step: 4,700).
//
// Slots beyond an item's range may hold anything: their scores are replaced, and their values are zeros before a product reads them (operands are made so; over
// bfloat16 the fetching warp clears them in the item's first and last tile).  Every mbarrier wait is bounded (HB_WAIT_LIMIT looks); a wait that runs out sets
// HB_STATUS_WAIT_EXPIRED, all roles leave their loops, what the block has on its way (copies, products) is waited for, tensor memory is freed and the block returns.
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
constexpr int BM = 128;                       // rows of one half = tensor-memory lanes
constexpr int ROWS = 2 * BM;                  // rows of an item
constexpr int BN = 128;                       // keys per tile
constexpr int PANELS = D / 64;
constexpr int KV_PANEL = BN * 64;             // elements of a 128-key x 64-column panel (16 KB)
constexpr int Q_PANEL = ROWS * 64;            // elements of a 256-row x 64-column panel of Q (32 KB)
constexpr int TILE_BYTES = PANELS * KV_PANEL * 2;
constexpr int STAGES = 2;                     // of K tiles and of V tiles
constexpr int TMEM_COLS = 512;                // S_H [0,128) S_L [128,256) O_H [256,256+D) O_L [384,384+D); P_x over S_x
constexpr int O_COL = 256;
constexpr int ITEM_WORDS = 7;                 // first token, tokens, table row, first key, last key + 1, number of the piece (with OWN_PIECE: among those of its own positions), first operand tile
constexpr int OWN_PIECE = 1 << 30;
enum Source : int { BFLOAT16 = 0, OPERANDS = 1 };  // what the tiles come from: a bfloat16 cache, or operands made of an 8-bit one
constexpr unsigned WAIT_LIMIT = HB_WAIT_LIMIT, LAST_WAIT_LIMIT = 1u << 24;

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
__device__ __forceinline__ void bulk_load(void* dst, const void* src, unsigned bytes, unsigned long long* bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)), "l"(src), "r"(bytes), "r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// The lane that issues the products is one thread, and a lone thread runs a few cycles per instruction: descriptor
// arithmetic between two products is time the tensor cores stand idle. So descriptors are kept as 32-bit low words that
// are only added to (the high word is the same for K-major and MN-major tiles with the 128-byte swizzle and 8-row groups
// 1,024 bytes apart), and four products are issued from one statement.
constexpr unsigned DESC_HIGH = (unsigned)(1024 >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ unsigned low_k_major(const void* tile) { return ((smem_u32(tile) & 0x3FFFFu) >> 4) | (1u << 16); }
__device__ __forceinline__ unsigned low_mn_major(const void* tile, unsigned panel_bytes) { return ((smem_u32(tile) & 0x3FFFFu) >> 4) | ((panel_bytes >> 4) << 16); }

// S = Q K^T over one 64-column panel of the head (4 products of 16 columns); `first` = 0 starts a new S.
__device__ __forceinline__ void umma_s_panel(unsigned tmem_d, unsigned q_low, unsigned k_low, unsigned idesc, unsigned first) {
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
        ::"r"(tmem_d), "r"(q_low), "r"(k_low), "r"(idesc), "r"(first), "r"(DESC_HIGH) : "memory");
}
// O += P V over 32 keys: the upper parts of P (8 columns per 16 keys), then the lower ones, V MN-major (16 keys = two 8-key groups = 2,048 bytes = 128 units of
// the descriptor's address field).
__device__ __forceinline__ void umma_pv_32(unsigned tmem_o, unsigned tmem_p, unsigned v_low, unsigned idesc, unsigned first) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t.reg .b64 da, db;\n\t.reg .b32 bl, pa;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "setp.eq.b32 q, 0, 0;\n\t"
        "mov.b64 da, {%2, %5};\n\t"
        "add.u32 bl, %2, 128;\n\t"
        "mov.b64 db, {bl, %5};\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], da, %3, p;\n\t"
        "add.u32 pa, %1, 8;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [pa], db, %3, q;\n\t"
        "add.u32 pa, %1, 16;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [pa], da, %3, q;\n\t"
        "add.u32 pa, %1, 24;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [pa], db, %3, q;\n\t}"
        ::"r"(tmem_o), "r"(tmem_p), "r"(v_low), "r"(idesc), "r"(first), "r"(DESC_HIGH) : "memory");
}
__device__ __forceinline__ void umma_commit_at(unsigned bar_addr) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar_addr) : "memory");
}
// float accumulator, both operands bfloat16, A K-major, M 128, N n; B MN-major when b_mn.
__device__ __forceinline__ unsigned idesc_for(int n, bool b_mn) {
    return (1u << 4) | (1u << 7) | (1u << 10) | (b_mn ? (1u << 16) : 0u) | ((unsigned)(n >> 3) << 17) | ((unsigned)(BM >> 4) << 24);
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
__device__ __forceinline__ void tmem_st32(unsigned taddr, const unsigned (&r)[32]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};"
                 :: "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]), "r"(taddr)
                 : "memory");
}
// 2^x by the hardware approximation (inputs are <= OUTGROWN; -inf gives 0).
__device__ __forceinline__ float fast_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ unsigned pack_bf16x2(float lo, float hi) {
    unsigned w;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(hi), "f"(lo));
    return w;
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
__device__ __forceinline__ bool elected() {  // one lane of the warp, all of which are here
    unsigned one;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(one));
    return one != 0;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ float value_of_half(unsigned short h) {
    float f;
    asm("cvt.f32.f16 %0, %1;" : "=f"(f) : "h"(h));
    return f;
}

struct Args {
    const unsigned char* operands;  // [tiles, kv_heads, 2, TILE_BYTES]
    bf16* out; int out_stride;
    const int* block_table; int table_width;
    const int* items;
    const int* first_item;          // [blocks + 1]: block b takes items first_item[b] .. first_item[b + 1] - 1
    const int* last;                // [tokens]: the last position a token sees, -1 for none
    const int* piece_start;         // [tokens + 1]
    const int* own_start;           // [tokens]
    float* pieces;                  // [pieces, heads, D], or null: rows have one piece each and are stored at once
    float2* sums;                   // [pieces, heads]: (m, l)
    int heads, kv_heads, page_size, pages;
    int gc, chunks;                 // heads of an item, items of a key/value head's group
    float scale_log2;
    int* status;
};

// How far (in powers of two) a maximum may be outgrown before the row is rescaled.  A stale maximum changes no result (numerator and denominator use the same
// one) as long as nothing overflows: weights are bfloat16, their sums float, and values end below 2^49.  A row that outgrows its own makes its half of the tile wait while O is scaled.
constexpr float OUTGROWN = 32.f;

constexpr int Q_BYTES = PANELS * Q_PANEL * 2;
constexpr int THREADS = 32 * 12;
constexpr int DESK = 32 * 32;                 // floats a softmax warp has in shared memory for 32 columns of its rows on their way out
constexpr size_t SMEM_USED = 1024 + (size_t)Q_BYTES + (size_t)2 * STAGES * TILE_BYTES + 8 * DESK * 4 + 256;
static_assert(SMEM_USED <= 227 * 1024, "an SM's shared memory");
// more than half of an SM's shared memory, so that one block is all an SM takes: the block holds all of its tensor memory
constexpr size_t SMEM_BYTES = SMEM_USED > 120 * 1024 ? SMEM_USED : 120 * 1024;

// Sixteen codes times 2^e as bfloat16, which holds them exactly.
__device__ __forceinline__ void widen(const uint4& codes, int e, unsigned (&wide)[8]) {
    const unsigned words[4] = {codes.x, codes.y, codes.z, codes.w};
    const float f = __uint_as_float((unsigned)(127 + e) << 23);
    const Pair factor{f, f};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        unsigned h0, h1;
        asm("{.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\tcvt.rn.f16x2.e4m3x2 %1, hi;\n\t}" : "=r"(h0), "=r"(h1) : "r"(words[k]));
        const Pair v0 = mul2(Pair{value_of_half((unsigned short)h0), value_of_half((unsigned short)(h0 >> 16))}, factor);
        const Pair v1 = mul2(Pair{value_of_half((unsigned short)h1), value_of_half((unsigned short)(h1 >> 16))}, factor);
        wide[2 * k] = pack_bf16x2(v0.x, v0.y), wide[2 * k + 1] = pack_bf16x2(v1.x, v1.y);
    }
}

struct Item {
    int tok0, ntok, key_lo, key_hi, piece, operand, start, n_tiles, halves;
    const int* table;
};

template <Source FROM>
__global__ void __launch_bounds__(THREADS, 1) attention_shared_kernel(const __grid_constant__ CUtensorMap kv_map, const __grid_constant__ CUtensorMap q_map, const Args a) {
    extern __shared__ unsigned char smem_raw[];
    unsigned char* base = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    unsigned char* k_ring = base;
    unsigned char* v_ring = k_ring + (size_t)STAGES * TILE_BYTES;
    unsigned char* qs = v_ring + (size_t)STAGES * TILE_BYTES;
    float* desks = reinterpret_cast<float*>(qs + Q_BYTES);  // [8][DESK]
    unsigned long long* k_full = reinterpret_cast<unsigned long long*>(desks + 8 * DESK);
    unsigned long long* k_empty = k_full + 2;
    unsigned long long* v_full = k_empty + 2;
    unsigned long long* v_empty = v_full + 2;
    unsigned long long* s_full = v_empty + 2;    // [2]: per half
    unsigned long long* p_full = s_full + 2;     // [2][2]: the P of the tile's upper keys, of its lower ones
    unsigned long long* o_done = p_full + 4;     // [2]: the item's last product
    unsigned long long* q_full = o_done + 2;
    unsigned long long* q_empty = q_full + 1;
    unsigned long long* edge_full = q_empty + 1;  // bfloat16: a V tile whose slots beyond the range are cleared before it is announced
    unsigned long long* all_done = edge_full + 1;  // every product that was issued
    unsigned* tmem_slot = reinterpret_cast<unsigned*>(all_done + 1);
    volatile int* failed = reinterpret_cast<volatile int*>(tmem_slot + 1);

    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (tid == 0) {
        for (int s = 0; s < 2; ++s) {
            mbar_init(&k_full[s], 1);
            mbar_init(&k_empty[s], 1);
            mbar_init(&v_full[s], 1);
            mbar_init(&v_empty[s], 1);
            mbar_init(&s_full[s], 1);
            mbar_init(&p_full[2 * s], 4);
            mbar_init(&p_full[2 * s + 1], 4);
            mbar_init(&o_done[s], 1);
        }
        mbar_init(q_full, 1);
        mbar_init(q_empty, 1);
        mbar_init(edge_full, 1);
        mbar_init(all_done, 1);
        *failed = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&kv_map) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&q_map) : "memory");
    }
    // rows of Q that no copy writes (beyond tokens x heads of an item) are computed like the others and never stored
    for (int e = tid; e < Q_BYTES / 16; e += THREADS) reinterpret_cast<uint4*>(qs)[e] = make_uint4(0, 0, 0, 0);
    const int first_item = a.first_item[blockIdx.x], end_item = a.first_item[blockIdx.x + 1];  // written with the plan, long before, like the items
    wait_for_previous_kernels();
    // All of the SM's tensor memory, and only now: a block of a kernel further back in the stream that has yet to start on this SM can no longer want any.
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    tc_fence_before();
    __syncthreads();
    // Only now: the strip kernel of the same step takes its start as the sign that all that came before has finished, and a kernel behind that takes tensor memory before it waits for
    // this one must find it taken, not take what this block still has to ask for.
    let_next_kernel_start();
    tc_fence_after();
    const unsigned tmem = *tmem_slot;
    const int shift = 31 - __clz(a.page_size);
    const int group = a.heads / a.kv_heads, kvh = blockIdx.y / a.chunks, chunk = blockIdx.y - kvh * a.chunks;
    const int first_head = kvh * group + chunk * a.gc, heads_here = min(a.gc, group - chunk * a.gc);

    // The roles run through the block's items each at its own pace, held together by the barriers of the data alone.  A wait by parity tells "this phase is over"
    // only to a thread that is at most one phase behind: every barrier's waiter is the one whose own arrival, on the barrier's counterpart, lets the next
    // phase begin, or it looks at the barrier once per phase.
    auto read_item = [&](int index) {
        Item it;
        const int* words = a.items + (size_t)index * ITEM_WORDS;
        it.tok0 = words[0], it.ntok = words[1], it.key_lo = words[3], it.key_hi = words[4], it.piece = words[5], it.operand = words[6];
        it.table = a.block_table + (size_t)words[2] * a.table_width;
        it.start = it.key_lo / BN * BN;
        it.n_tiles = it.key_hi > it.key_lo ? (it.key_hi - it.start + BN - 1) / BN : 0;
        it.halves = it.ntok * a.gc > BM ? 2 : 1;
        return it;
    };
    auto fail = [&] { *failed = 1; };

    if (warp == 0) {
        // ------------------------------------------------------------------ producer (the whole warp)
        const int pages_per_tile = BN >> shift, tokens_per_item = ROWS / a.gc;
        bool alive = true;
        int g = 0, edges = 0, round = 0;  // g: tiles so far
        int k_sent = 0, v_sent = 0, q_sent = 0, edges_sent = 0;  // phases of the barriers that lane 0 has set going
        for (int index = first_item; index < end_item && alive; ++index, ++round) {
            const Item it = read_item(index);
            if (lane == 0) {  // the queries: tokens beyond the item's own come along, or are filled with zeros
                if (!mbar_wait(q_empty, (round & 1) ^ 1, failed)) alive = false;
                if (alive) {
                    mbar_expect_tx(q_full, (unsigned)(PANELS * 128 * a.gc * tokens_per_item));
                    ++q_sent;
                    for (int h = 0; h < PANELS; ++h) tma_load_3d(qs + h * Q_PANEL * 2, &q_map, q_full, h * 64, first_head, it.tok0);
                }
            }
            alive = __shfl_sync(0xffffffffu, alive ? 1 : 0, 0) != 0;
            for (int t = 0; t < it.n_tiles && alive; ++t, ++g) {
                const int tile_base = it.start + t * BN;
                if constexpr (FROM == OPERANDS) {  // two plain copies: they stand there as the products read them
                    if (lane == 0) {
                        const unsigned char* from = a.operands + ((size_t)(it.operand + t) * a.kv_heads + kvh) * (2 * TILE_BYTES);
                        for (int which = 0; which < 2 && alive; ++which) {
                            const int s = g & 1, turn = g >> 1;
                            if (!mbar_wait(which ? &v_empty[s] : &k_empty[s], (turn & 1) ^ 1, failed)) { alive = false; break; }
                            mbar_expect_tx(which ? &v_full[s] : &k_full[s], TILE_BYTES);
                            ++(which ? v_sent : k_sent);
                            bulk_load((which ? v_ring : k_ring) + (size_t)s * TILE_BYTES, from + which * TILE_BYTES, TILE_BYTES, which ? &v_full[s] : &k_full[s]);
                        }
                    }
                    alive = __shfl_sync(0xffffffffu, alive ? 1 : 0, 0) != 0;
                    continue;
                }
                int my_page = -1;
                const int k0 = tile_base + lane * a.page_size;
                if (lane < pages_per_tile && k0 < it.key_hi && k0 + a.page_size > it.key_lo) {
                    const int block = k0 >> shift;
                    const int id = block < a.table_width ? __ldg(it.table + block) : -1;
                    if (id >= 0 && id < a.pages) my_page = id;
                    else atomicOr(a.status, HB_STATUS_BAD_PAGE);
                }
                const unsigned valid = __popc(__ballot_sync(0xffffffffu, my_page >= 0));
                const bool edge = tile_base < it.key_lo || tile_base + BN > it.key_hi;
                for (int which = 0; which < 2 && alive; ++which) {  // the K tile, then the V tile
                    const int s = g & 1, turn = g >> 1;
                    unsigned long long* empty = which ? &v_empty[s] : &k_empty[s];
                    unsigned long long* full = which ? (edge ? edge_full : &v_full[s]) : &k_full[s];
                    int ok = 1;
                    if (lane == 0) ok = mbar_wait(empty, (turn & 1) ^ 1, failed) ? 1 : 0;
                    ok = __shfl_sync(0xffffffffu, ok, 0);
                    if (!ok) { alive = false; break; }
                    if (lane == 0) {
                        const unsigned page_bytes = (unsigned)a.page_size * D * 2u;
                        if (valid) mbar_expect_tx(full, valid * page_bytes); else mbar_arrive(full);
                        ++(which ? (edge ? edges_sent : v_sent) : k_sent);
                    }
                    __syncwarp();
                    unsigned char* stage = which ? v_ring + (size_t)s * TILE_BYTES : k_ring + (size_t)s * TILE_BYTES;
                    const int ops = pages_per_tile * PANELS;
                    for (int op0 = 0; op0 < ops; op0 += 32) {
                        const int op = op0 + lane, p = min(op, ops - 1) / PANELS, h = op % PANELS;
                        const int from = __shfl_sync(0xffffffffu, my_page, p);
                        if (op < ops && from >= 0)
                            tma_load_2d(stage + h * KV_PANEL * 2 + p * a.page_size * 128, &kv_map, full, h * 64, ((from * 2 + which) * a.kv_heads + kvh) * a.page_size);
                    }
                    if (which && edge) {
                        ok = mbar_wait(edge_full, edges & 1, failed) ? 1 : 0;
                        ++edges;
                        if (!__all_sync(0xffffffffu, ok)) { alive = false; break; }
                        for (int e = lane; e < BN * 8 * PANELS; e += 32) {
                            const int row = (e >> 3) & (BN - 1), pos = tile_base + row;
                            if (pos < it.key_lo || pos >= it.key_hi) reinterpret_cast<uint4*>(stage)[e] = make_uint4(0, 0, 0, 0);
                        }
                        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&v_full[s]), ++v_sent;
                    }
                }
            }
        }
        if (!alive) fail();
        if (lane == 0) {  // all that was sent arrives before the block leaves
            for (int t = max(0, k_sent - 2); t < k_sent; ++t) mbar_last_wait(&k_full[t & 1], (t >> 1) & 1);
            for (int t = max(0, v_sent - 2); t < v_sent; ++t) mbar_last_wait(&v_full[t & 1], (t >> 1) & 1);
            if (q_sent) mbar_last_wait(q_full, (q_sent - 1) & 1);
            if (edges_sent) mbar_last_wait(edge_full, (edges_sent - 1) & 1);
        }
        __syncwarp();
    } else if (warp == 1) {
        // ------------------------------------------------------------------ tensor-core issuer: the warp stays together, so that descriptors are its common values
        // (uniform registers); one elected lane issues.  Under `if (lane == 0)` every product took 65 clocks to
        // issue, as long as it runs, and the waits came on top (a tile a tenth slower).
        const unsigned idesc_s = idesc_for(BN, false), idesc_o = idesc_for(D, true);
        const unsigned q_low0 = low_k_major(qs), k_low0 = low_k_major(k_ring), v_low0 = low_mn_major(v_ring, KV_PANEL * 2);
        auto wait_for = [&](unsigned long long* bar, int phase) { return __all_sync(0xffffffffu, mbar_wait(bar, phase & 1, failed)) != 0; };
        auto issue_s = [&](int x, int g) {  // S_x = Q_x K(g)^T
            const unsigned k_low = k_low0 + (unsigned)(g & 1) * (TILE_BYTES >> 4), q_low = q_low0 + (unsigned)x * (BM * 128 >> 4);
            if (elected()) {
                umma_s_panel(tmem + x * BN, q_low, k_low, idesc_s, 0u);
#pragma unroll
                for (int h = 1; h < PANELS; ++h) umma_s_panel(tmem + x * BN, q_low + h * (Q_PANEL * 2 >> 4), k_low + h * (KV_PANEL * 2 >> 4), idesc_s, 1u);
                umma_commit_at(smem_u32(&s_full[x]));
            }
        };
        auto issue_pv = [&](int x, int g, int part, unsigned accumulate) {  // O_x (+)= P_x V(g) over the upper (part 0) or the lower 64 keys
            const unsigned at = part ? 0u : 64u, v_low = v_low0 + (unsigned)(g & 1) * (TILE_BYTES >> 4) + at * 8, o = tmem + O_COL + x * BM, p = tmem + x * BN + at;
            if (elected()) {
                umma_pv_32(o, p, v_low, idesc_o, accumulate);
                umma_pv_32(o, p + 32, v_low + 256, idesc_o, 1u);
            }
        };
        auto commit = [&](unsigned long long* bar) {
            if (elected()) umma_commit_at(smem_u32(bar));
        };
        bool ok = true;
        int g = 0, mine[2] = {0, 0}, round = 0;  // tiles so far, and those that a half had a part in
        for (int index = first_item; index < end_item && ok; ++index, ++round) {
            const Item it = read_item(index);
            if (!wait_for(q_full, round)) { ok = false; break; }
            if (it.n_tiles == 0) { commit(q_empty); continue; }
            if (!wait_for(&k_full[g & 1], g >> 1)) { ok = false; break; }
            tc_fence_after();
            // S_x of the first tile lands in the columns that the last product of the item before read its P from: products of one thread run in the
            // order of their issue
            for (int x = 0; x < it.halves; ++x) issue_s(x, g);
            commit(&k_empty[g & 1]);
            if (it.n_tiles == 1) commit(q_empty);
            for (int j = 0; j < it.n_tiles && ok; ++j, ++g) {
                const bool more = j + 1 < it.n_tiles;
                if (!wait_for(&v_full[g & 1], g >> 1) || (more && !wait_for(&k_full[(g + 1) & 1], (g + 1) >> 1))) { ok = false; break; }  // while the softmax is busy
                for (int x = 0; x < it.halves && ok; ++x) {
                    for (int part = 0; part < 2 && ok; ++part) {
                        if (!wait_for(&p_full[2 * x + part], mine[x])) { ok = false; break; }
                        tc_fence_after();
                        issue_pv(x, g, part, j > 0 || part > 0 ? 1u : 0u);
                    }
                    if (!ok) break;
                    if (more) issue_s(x, g + 1);
                    else commit(&o_done[x]);
                    ++mine[x];
                }
                if (!ok) break;
                commit(&v_empty[g & 1]);
                if (more) commit(&k_empty[(g + 1) & 1]);
                if (j + 2 == it.n_tiles) commit(q_empty);
            }
        }
        if (!ok) fail();
        commit(all_done);  // the products and the arrivals that tell of them, before tensor memory is freed
        mbar_last_wait(all_done, 0);
        __syncwarp();
    } else if (warp >= 4) {
        // ------------------------------------------------------------------ softmax: thread = row = tensor-memory lane of its half
        const int x = (warp - 4) >> 2, quarter = warp & 3, r = quarter * 32 + lane, v = x * BM + r;
        const unsigned lane_addr = tmem + ((unsigned)(quarter * 32) << 16);
        const unsigned s_addr = lane_addr + x * BN, o_addr = lane_addr + O_COL + x * BM;
        float* desk = desks + (warp - 4) * DESK;
        const float scale = a.scale_log2;
        const Pair scale2{scale, scale}, minus_one{-1.f, -1.f};
        int hx = 0, mine = 0;  // tiles this half has seen, items it has had a part in
        bool ok = true;
        for (int index = first_item; index < end_item && ok; ++index) {
            const Item it = read_item(index);
            if (x >= it.halves) continue;
            const int tok = v / a.gc, hh = v - tok * a.gc;
            const bool row_valid = tok < it.ntok && hh < heads_here;
            // a row that is no one's is computed like the item's last token and never stored: it takes the same way through the code as its neighbours
            const int token = it.tok0 + min(tok, it.ntok - 1), hi = min(it.key_hi - 1, a.last[token]);
            int piece_at = 0;
            if (row_valid && a.pieces) piece_at = (it.piece & OWN_PIECE ? a.own_start : a.piece_start)[token] + (it.piece & (OWN_PIECE - 1));
            float m = -INFINITY, l = 0.f;
            for (int j = 0; j < it.n_tiles; ++j) {
                const int h = hx + j;
                if (!mbar_wait(&s_full[x], h & 1, failed)) { ok = false; break; }
                tc_fence_after();
                const int tile_base = it.start + j * BN, last_visible = hi - tile_base, first_visible = it.key_lo - tile_base;
                unsigned s0[32], s1[32];  // of this row's S, 32 columns at hand and 32 on their way
                auto hand_over = [&](int which) {
                    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&p_full[2 * x + which]);
                };
                float part[2] = {-INFINITY, -INFINITY};
                auto look = [&](unsigned (&s)[32]) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) part[i & 1] = max3(part[i & 1], __uint_as_float(s[2 * i]), __uint_as_float(s[2 * i + 1]));
                };
                const bool whole = __all_sync(0xffffffffu, last_visible >= BN - 1 && first_visible <= 0);
                // The loops below are kept short on purpose: the roles of a block run different code on the same schedulers, and straight-line code is bound by
                // the fetching of instructions (256 requests behind 16,384 positions took 19 % longer with every loop unrolled and masks in each of them).
                if (!whole) {  // what a row does not see is replaced where it stands; one way for the whole warp
#pragma unroll 1
                    for (int c = 0; c < BN; c += 32) {
                        tmem_ld32(s_addr + c, s0), arrived(s0);
#pragma unroll
                        for (int i = 0; i < 32; ++i) s0[i] = (c + i <= last_visible && c + i >= first_visible) ? s0[i] : 0xff800000u;
                        tmem_st32(s_addr + c, s0);
                    }
                    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                }
                tmem_ld32(s_addr, s0), arrived(s0);
#pragma unroll 1
                for (int c = 0; c < BN; c += 64) {
                    tmem_ld32(s_addr + c + 32, s1), look(s0), arrived(s1);
                    if (c == 0) tmem_ld32(s_addr + 64, s0);
                    look(s1);
                    if (c == 0) arrived(s0);
                }
                const float seen = max3(part[0], part[1], -INFINITY) * scale, m_new = fmaxf(m, seen);  // the scale is positive: the largest score stays the largest
                const bool outgrown = __any_sync(0xffffffffu, m > -INFINITY && m_new - m > OUTGROWN);  // one row's is taken as the occasion for all of the warp's
                float alpha = 1.f;
                if (!(seen < INFINITY)) {
                    m = __uint_as_float(0x7fffffffu);  // a NaN or an infinity among the scores: the row's softmax is no number, and stays none
                } else if (m == -INFINITY) {
                    m = m_new;  // nothing seen so far: the row of O holds zeros (or is overwritten by the first product)
                } else if (outgrown) {
                    alpha = exp2f(m - m_new);
                    m = m_new;
                }
                // The products of the tiles before were issued before this S was, and this S has arrived: O stands still.
                if (j > 0 && outgrown) {
#pragma unroll 1
                    for (int c = 0; c < D; c += 32) {
                        tmem_ld32(o_addr + c, s0), arrived(s0);
#pragma unroll
                        for (int i = 0; i < 32; ++i) s0[i] = __float_as_uint(__uint_as_float(s0[i]) * alpha);
                        tmem_st32(o_addr + c, s0);
                    }
                }
                const float minus_m = m == -INFINITY ? 0.f : -m;
                const Pair minus_m2{minus_m, minus_m};
                Pair sum[2] = {{0.f, 0.f}, {0.f, 0.f}};
                auto weigh = [&](const unsigned (&s)[32], int c) {  // P of 32 columns as bfloat16 in two parts, over the columns that they came from
                    unsigned w[32];
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const Pair z = fma2(Pair{__uint_as_float(s[2 * i]), __uint_as_float(s[2 * i + 1])}, scale2, minus_m2), p{fast_exp2(z.x), fast_exp2(z.y)};
                        sum[i & 1] = add2(sum[i & 1], p);
                        w[i] = __byte_perm(__float_as_uint(p.x), __float_as_uint(p.y), 0x7632);
                        const Pair rest = fma2(Pair{__uint_as_float(__float_as_uint(p.x) & 0xffff0000u), __uint_as_float(__float_as_uint(p.y) & 0xffff0000u)}, minus_one, p);
                        w[16 + i] = pack_bf16x2(rest.x, rest.y);
                    }
                    tmem_st32(s_addr + c, w);
                };
#pragma unroll 1
                for (int c = 64; c >= 0; c -= 64) {  // columns 96 to 127 are still at hand
                    tmem_ld32(s_addr + c, s0), weigh(s1, c + 32), arrived(s0);
                    if (c) tmem_ld32(s_addr + c - 32, s1);
                    weigh(s0, c);
                    hand_over(c ? 0 : 1);
                    if (c) arrived(s1);
                }
                l = l * alpha + ((sum[0].x + sum[0].y) + (sum[1].x + sum[1].y));
            }
            if (ok && it.n_tiles > 0) ok = mbar_wait(&o_done[x], mine++ & 1, failed);
            ok = __all_sync(0xffffffffu, ok);
            tc_fence_after();
            if (ok) {
                if (m == -INFINITY) l = 0.f;  // a row that sees nothing: what exp2_pair gave for it is none of its weights
                const float inv = a.pieces ? 1.f : (l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l));  // a row that sees nothing is zeros; a NaN stays one
                // Rows leave through shared memory, 32 columns of 32 rows at a time: eight lanes then store 128 bytes of a row side by side, where a thread storing its own row
                // would touch 32 lines with every instruction.  Some 6,000 clocks an item either way, 32 bytes a clock: what an SM stores.
                const long long row_at = !row_valid ? -1 : a.pieces ? ((long long)piece_at * a.heads + first_head + hh) * D : (long long)token * a.out_stride + (long long)(first_head + hh) * D;
                if (row_valid && a.pieces) a.sums[(size_t)piece_at * a.heads + first_head + hh] = make_float2(m, l);
#pragma unroll 1
                for (int c = 0; c < D; c += 32) {
                    unsigned o[32];
                    if (it.n_tiles > 0) {
                        tmem_ld32(o_addr + c, o), arrived(o);
                    } else {
#pragma unroll
                        for (int i = 0; i < 32; ++i) o[i] = 0u;
                    }
                    float4* line = reinterpret_cast<float4*>(desk) + lane * 8;
#pragma unroll
                    for (int i = 0; i < 8; ++i)  // 16-byte pieces, turned about by the row so that neither way meets a bank twice
                        line[i ^ (lane & 7)] = make_float4(__uint_as_float(o[4 * i]) * inv, __uint_as_float(o[4 * i + 1]) * inv, __uint_as_float(o[4 * i + 2]) * inv, __uint_as_float(o[4 * i + 3]) * inv);
                    __syncwarp();
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const int row = i * 4 + (lane >> 3), at = lane & 7;
                        const long long to = __shfl_sync(0xffffffffu, row_at, row);
                        const float4 out = reinterpret_cast<const float4*>(desk)[row * 8 + (at ^ (row & 7))];
                        if (to >= 0) {
                            const float w[4] = {out.x, out.y, out.z, out.w};
                            if (a.pieces) store4(a.pieces + to + c + 4 * at, w);
                            else store4(a.out + to + c + 4 * at, w);
                        }
                    }
                    __syncwarp();
                }
                // the row is out of tensor memory before this thread hands over the next item's first P, and only then is O written anew
                tc_fence_before();
            }
            hx += it.n_tiles;
        }
        if (!ok) fail();
    }
    tc_fence_before();
    __syncthreads();
    if (tid == 0 && *failed) atomicOr(a.status, HB_STATUS_WAIT_EXPIRED | HB_STATUS_IN_ATTENTION_SHARED);
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM_COLS) : "memory");
    }
}

// Operands of 8-bit records: a block makes one tile of K or of V of one key/value head, in the layout of the attention's shared memory, so that every run of tokens that
// walks it fetches it by a plain copy and converts nothing.  Bound by what the device writes to L2: 16,384 positions of 4 heads of 128 in 12 us (67 MB, 5.6 TB/s).  (Conversion inside the attention, by eight more warps between the
// copies and the products, was built first: it held a block back from 4,200 to 5,600 clocks a tile, for every run anew: 256
// requests behind 16,384 positions, eight runs, 162 us against 154, 64 requests behind 4,096, two runs, 35.6 against 39.4, with the slower softmax of then.)
constexpr int OPERAND_THREADS = 256;
__global__ void __launch_bounds__(OPERAND_THREADS) shared_operands_kernel(const unsigned char* __restrict__ codes, const signed char* __restrict__ exponents, const int* __restrict__ block_table,
                                                                          int table_width, const int4* __restrict__ tiles, unsigned char* __restrict__ operands,
                                                                          int page_size, int pages, int* status) {
    let_next_kernel_start();
    const int4 tile = tiles[blockIdx.x];  // table row, first position, first key and last key + 1 of the range; written with the plan, long before
    wait_for_previous_kernels();
    const int kvh = blockIdx.y, kv_heads = gridDim.y, which = blockIdx.z, tid = threadIdx.x, base = tile.y, lo = tile.z, hi = tile.w, shift = 31 - __clz(page_size);
    const int* table = block_table + (size_t)tile.x * table_width;
    auto record = [&](int pos) -> long long {  // -1: not in the range, or without a page
        const int block = pos >> shift, page = pos >= lo && pos < hi && block < table_width ? table[block] : -1;
        return page >= 0 && page < pages ? (((long long)page * 2 + which) * kv_heads + kvh) * page_size + (pos & (page_size - 1)) : -1;
    };
    constexpr int CHUNKS = D / 16, UNITS = BN * CHUNKS / OPERAND_THREADS, STEP = OPERAND_THREADS / CHUNKS;  // a thread's chunks of 16 codes, of rows STEP apart
    const int chunk = tid % CHUNKS, row0 = tid / CHUNKS;
    long long from[UNITS];
    uint4 raw[UNITS];
    int e[UNITS];
#pragma unroll
    for (int u = 0; u < UNITS; ++u) from[u] = record(base + row0 + u * STEP);
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
        const long long at = max(from[u], 0ll);
        raw[u] = *reinterpret_cast<const uint4*>(codes + at * D + chunk * 16);
        e[u] = min(max((int)exponents[at], -40), 40);
    }
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
        const int pos = base + row0 + u * STEP;
        if (chunk == 0 && kvh == 0 && which == 0 && from[u] < 0 && pos >= lo && pos < hi) atomicOr(status, HB_STATUS_BAD_PAGE);
    }
    unsigned char* out = operands + (((size_t)blockIdx.x * kv_heads + kvh) * 2 + which) * TILE_BYTES;
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
        const int row = row0 + u * STEP;
        unsigned wide[8];
        widen(raw[u], e[u], wide);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int oc = 2 * chunk + half;
            uint4 w = make_uint4(wide[4 * half], wide[4 * half + 1], wide[4 * half + 2], wide[4 * half + 3]);
            if (from[u] < 0) w = make_uint4(0, 0, 0, 0);
            *reinterpret_cast<uint4*>(out + (oc >> 3) * (KV_PANEL * 2) + row * 128 + (((oc & 7) ^ (row & 7)) << 4)) = w;
        }
    }
}

typedef CUresult (*EncodeTiled)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiled encode_tiled() {
    static EncodeTiled fn = nullptr;
    if (!fn) {
        void* found = nullptr;
        cudaDriverEntryPointQueryResult result;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &found, cudaEnableDefault, &result) == cudaSuccess &&
            result == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<EncodeTiled>(found);
    }
    return fn;
}

template <Source FROM>
int launch(const Args& a, int blocks, const void* q, int q_stride, int n_tokens, const void* cache, cudaStream_t stream) {
    EncodeTiled encode = encode_tiled();
    if (!encode) return HB_BAD_ARGUMENT;
    CUtensorMap map, q_map;
    const cuuint32_t elem[3] = {1, 1, 1};
    // the queries as (column, head, token): an item's box is 64 columns of gc heads of its tokens
    const cuuint64_t q_dims[3] = {(cuuint64_t)D, (cuuint64_t)a.heads, (cuuint64_t)n_tokens};
    const cuuint64_t q_strides[2] = {(cuuint64_t)D * 2, (cuuint64_t)q_stride * 2};
    const cuuint32_t q_box[3] = {64, (cuuint32_t)a.gc, (cuuint32_t)(ROWS / a.gc)};
    if (encode(&q_map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(q), q_dims, q_strides, q_box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
        return HB_BAD_ARGUMENT;
    if constexpr (FROM == BFLOAT16) {  // the cache as a matrix [pages * 2 * kv_heads * page_size, D], fetched in boxes of a page's rows and 64 columns
        const cuuint64_t dims[2] = {(cuuint64_t)D, (cuuint64_t)a.pages * 2 * a.kv_heads * a.page_size};
        const cuuint64_t strides[1] = {(cuuint64_t)D * 2};
        const cuuint32_t box[2] = {64, (cuuint32_t)a.page_size};
        if (encode(&map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(cache), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                   CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
            return HB_BAD_ARGUMENT;
    } else {
        map = q_map;  // operands are fetched without one
    }
    static const cudaError_t configured = cudaFuncSetAttribute(attention_shared_kernel<FROM>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)SMEM_BYTES);
    if (configured != cudaSuccess) return (int)configured;
    return launch_after_previous(attention_shared_kernel<FROM>, dim3(blocks, a.kv_heads * a.chunks), dim3(THREADS), SMEM_BYTES, stream, map, q_map, a);
}
}  // namespace

// tiles [n_tiles, 4]: table row, first position, first key and last key + 1 of the tile's range.  operands: n_tiles * kv_heads * 4 * 128 * D bytes.
HB_EXPORT int hb_shared_operands(const void* codes, const void* exponents, const int* block_table, int table_width, const int* tiles, int n_tiles, void* operands, int kv_heads,
                                 int page_size, int pages, int* status, cudaStream_t stream) {
    if (n_tiles <= 0) return 0;
    if (!codes || !exponents || !block_table || !tiles || !operands || !status || table_width <= 0 || kv_heads <= 0 || pages <= 0) return HB_BAD_ARGUMENT;
    if (page_size < 8 || page_size > 64 || (page_size & (page_size - 1)) || kv_heads > 65535) return HB_UNSUPPORTED_SIZE;
    if (((uintptr_t)codes | (uintptr_t)operands) & 15) return HB_BAD_ARGUMENT;
    if ((uintptr_t)tiles & 15) return HB_BAD_ARGUMENT;
    return launch_after_previous(shared_operands_kernel, dim3(n_tiles, kv_heads, 2), dim3(OPERAND_THREADS), 0, stream, (const unsigned char*)codes, (const signed char*)exponents, block_table,
                                 table_width, (const int4*)tiles, (unsigned char*)operands, page_size, pages, status);
}

// cache: [pages, 2, kv_heads, page_size, D] in bfloat16 (exponents and operands null), or e4m3 codes with exponents and the operands that hb_shared_operands has made of them.
// items: see ITEM_WORDS; first_item [blocks + 1]; an item has at most 256 / min(heads / kv_heads, 256) tokens.  pieces, sums null: one piece a row.
HB_EXPORT int hb_attention_shared_tiles(const void* q, long long q_stride, int n_tokens, void* out, long long out_stride, const void* cache, const void* exponents, const int* block_table,
                                        int table_width, const int* items, const int* first_item, int blocks, const void* operands, int operand_tiles, const int* last, const int* piece_start, const int* own_start, float* pieces, float* sums, int heads,
                                        int kv_heads, int page_size, int pages, float scale, int* status, cudaStream_t stream) {
    if (blocks <= 0) return 0;
    if (!q || !out || !cache || !block_table || !items || !first_item || !last || !piece_start || !own_start || !status || (!pieces != !sums)) return HB_BAD_ARGUMENT;
    if (kv_heads <= 0 || heads <= 0 || heads % kv_heads || pages <= 0 || table_width <= 0 || n_tokens <= 0 || q_stride % 8 || out_stride % 4) return HB_BAD_ARGUMENT;
    if (!(scale > 0.f)) return HB_BAD_ARGUMENT;  // the row maximum is taken before the scores are scaled
    if (page_size < 8 || page_size > 64 || (page_size & (page_size - 1))) return HB_UNSUPPORTED_SIZE;
    if ((((uintptr_t)q | (uintptr_t)cache) & 15) || ((uintptr_t)pieces & 31) || ((uintptr_t)exponents & 3) || ((uintptr_t)out & 7)) return HB_BAD_ARGUMENT;
    if ((long long)pages * 2 * kv_heads * page_size > 0x7fffffffLL) return HB_UNSUPPORTED_SIZE;  // a row's number in the cache's tensor map
    if (q_stride > 0x7fffffffLL || out_stride > 0x7fffffffLL) return HB_UNSUPPORTED_SIZE;
    const int group = heads / kv_heads, gc = group < ROWS ? group : ROWS, chunks = (group + gc - 1) / gc;
    if ((long long)kv_heads * chunks > 65535) return HB_UNSUPPORTED_SIZE;
    if (!operands != !exponents || (operands && (operand_tiles <= 0 || ((uintptr_t)operands & 15)))) return HB_BAD_ARGUMENT;
    const Args a{(const unsigned char*)operands, (bf16*)out, (int)out_stride, block_table, table_width, items, first_item, last, piece_start, own_start, pieces, (float2*)sums,
                 heads, kv_heads, page_size, pages, gc, chunks, scale * 1.4426950408889634f, status};
    if (operands) return launch<OPERANDS>(a, blocks, q, (int)q_stride, n_tokens, cache, stream);
    return launch<BFLOAT16>(a, blocks, q, (int)q_stride, n_tokens, cache, stream);
}
