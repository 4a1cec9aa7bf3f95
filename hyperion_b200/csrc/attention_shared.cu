// Attention of a step's queries over paged caches in which groups of requests share their first positions, for caches of bfloat16 and of
// 8-bit records (cache8.cu), head sizes 64 and 128 (HB_HEAD_DIM) and pages of 8 to 64 tokens.
//
// The host cuts the step into items: (tokens that stand together, a table row, a range of keys).  A group's shared positions are one range
// for all of its tokens, so they are fetched once for all of them; what a request holds beyond them is a range for its own tokens; either may
// be cut further so that the device is filled.  An item leaves for each of its (token, head) rows a piece
//     m,  l = sum_j 2^(y_j - m),  o = sum_j 2^(y_j - m) v_j          y_j = score_j * scale * log2(e)
// and the pieces of a row are put together afterwards, in the order of the ranges: with M = max m, out = sum 2^(m - M) o / sum 2^(m - M) l.
// A step whose rows have one piece each is stored at once.
//
// This file has the strip kernel, for items of few rows: it is bound by the bytes of the keys and values.  One lane of a producer warp per
// page fetches K and V by TMA (one box a page and 128-byte panel, no multicast) into a ring of 64-key stages; each of four warps takes 16 of a
// stage's keys for all 16 rows, S = Q K^T and O += P V by mma.sync m16n8k16, and at the end the warps' results are put together in shared memory.
//
// 8-bit records meet the tensor cores as float16, which holds every e4m3 code: one conversion instruction for two codes and nothing else per
// entry.  The exponents are kept out of the entries: a key's multiplies its score, and a value's goes into the softmax's exponent,
//     z_j = y_j + e_j,  P_j = 2^(z_j - m),  o = sum P_j code_j,  l = sum P_j 2^-e_j,
// with m the maximum of z.  Which entry of a head a lane's fragment holds does not matter to Q K^T as long as it is the same one in Q and K, so a
// lane takes 16 bytes of a key at once (entries 16 c to 16 c + 15 of chunk c), and Q's fragments are loaded to match; the columns of P V come
// out in another order than they are stored in, and are stored where they belong.
//
// Where the values' exponents lie far apart (a value 2^12 times smaller than another one of its range), a weight that counts can be too small for float16
// beside the other's: such a stage's weights are multiplied in lots by their size.
//
// Over a bfloat16 cache the weights are taken in two parts, rounded to bfloat16 and what that left over: rounded once they would cost the result as much as
// its own rounding does (1.4 times the error in all), and float16, whose rounding does not show, does not hold every bfloat16 value.
//
// Slots beyond a range's end may hold anything: their scores are replaced and their values are read as zeros.  Every mbarrier wait is
// bounded; one that runs out sets HB_STATUS_WAIT_EXPIRED and the block leaves.
#include <cuda.h>
#include <cuda_fp16.h>

#include "common.cuh"

#ifndef HB_HEAD_DIM
#define HB_HEAD_DIM 128
#endif

namespace {
typedef __nv_bfloat16 bf16;
constexpr int D = HB_HEAD_DIM;
static_assert(D == 64 || D == 128, "head sizes 64 and 128");
constexpr int BN = 64;          // keys of a stage
constexpr int ROWS = 16;        // (token, head) rows of a strip
constexpr int WARPS = 4;        // that compute; one more fetches
constexpr int THREADS = 32 * (WARPS + 1);
constexpr int ITEM_WORDS = 6;   // first token, tokens, table row, first key, last key + 1, number of the piece
constexpr unsigned WAIT_LIMIT = 1u << 24;
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
__device__ __forceinline__ bool mbar_wait(unsigned long long* bar, unsigned parity, volatile int* failed) {
    const unsigned addr = smem_u32(bar);
    for (unsigned spin = 0; spin < WAIT_LIMIT; ++spin) {
        unsigned done;
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
            "selp.b32 %0, 1, 0, p;\n\t}"
            : "=r"(done) : "r"(addr), "r"(parity) : "memory");
        if (done) return true;
        if ((spin & 1023) == 1023 && *failed) return false;
    }
    return false;
}
__device__ __forceinline__ void tma_load_2d(void* dst, const CUtensorMap* map, unsigned long long* bar, int x, int y) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
                 ::"r"(smem_u32(dst)), "l"(map), "r"(smem_u32(bar)), "r"(x), "r"(y) : "memory");
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
__device__ __forceinline__ float fast_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float((unsigned)(127 + e) << 23); }  // -126 <= e <= 127

template <bool E8>
struct Shape {
    static constexpr int BYTES = E8 ? 1 : 2;                  // of an entry
    static constexpr int TILE = BN * D * BYTES;               // one K or V tile
    static constexpr int PANEL_BYTES = D * BYTES < 128 ? D * BYTES : 128;  // of a row, in one box
    static constexpr int PANELS = D * BYTES / PANEL_BYTES;
    static constexpr int STAGE = 2 * TILE + (E8 ? 128 : 0);   // K, V, and the exponents of both
    static constexpr int STAGES = E8 ? (D == 128 ? 6 : 8) : (D == 128 ? 3 : 5);
    static constexpr int PER_CHUNK = 16 / BYTES;              // entries of 16 bytes
    static constexpr int CHUNKS = D / PER_CHUNK;              // of a row
    static constexpr int STEPS = PER_CHUNK / 4;               // products of 16 entries that one chunk a lane feeds
    static constexpr size_t SMEM = 1024 + (size_t)STAGES * STAGE + 2 * STAGES * 8 + 16;
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
    const int* last;         // [tokens]: the last position a token sees, -1 for none
    const int* piece_start;  // [tokens + 1]
    float* pieces;           // [pieces, heads, D], or null: rows have one piece each and are stored at once
    float2* sums;            // [pieces, heads]: (m, l)
    int heads, kv_heads, page_size, pages;
    int gc, chunks;          // heads of a strip, strips of a key/value head's group
    float scale_log2;
    int* status;
};

template <bool E8>
__global__ void __launch_bounds__(THREADS) attention_strip_kernel(const __grid_constant__ CUtensorMap kv_map, const Args a) {
    typedef Shape<E8> S;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* ring = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    // the tiles of all stages, then the exponents of all stages
    unsigned char* exps = ring + (size_t)S::STAGES * 2 * S::TILE;
    unsigned long long* full = reinterpret_cast<unsigned long long*>(exps + (E8 ? S::STAGES * 128 : 0));
    unsigned long long* empty = full + S::STAGES;
    volatile int* failed = reinterpret_cast<volatile int*>(empty + S::STAGES);

    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (tid == 0) {
        for (int s = 0; s < S::STAGES; ++s) { mbar_init(&full[s], E8 ? 33 : 1); mbar_init(&empty[s], WARPS); }
        *failed = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    let_next_kernel_start();
    wait_for_previous_kernels();
    const int* item = a.items + (size_t)blockIdx.x * ITEM_WORDS;
    const int tok0 = item[0], ntok = item[1], key_lo = item[3], key_hi = item[4], piece = item[5];
    const int* table = a.block_table + (size_t)item[2] * a.table_width;
    const int kvh = blockIdx.y / a.chunks, chunk = blockIdx.y - kvh * a.chunks;
    const int group = a.heads / a.kv_heads, first_head = kvh * group + chunk * a.gc, heads_here = min(a.gc, group - chunk * a.gc);
    const int start = key_lo / BN * BN, n_tiles = key_hi > key_lo ? (key_hi - start + BN - 1) / BN : 0;

    if (warp == WARPS) {
        // ------------------------------------------------------------------ producer (the whole warp)
        const int shift = 31 - __clz(a.page_size), pages_per_tile = BN >> shift, tiles_per_look = 32 / pages_per_tile;
        constexpr int OPS_PER_PAGE = 2 * S::PANELS;
        const int ops = pages_per_tile * OPS_PER_PAGE;
        const unsigned page_bytes = 2u * a.page_size * D * S::BYTES;
        if (lane == 0) asm volatile("prefetch.tensormap [%0];" ::"l"(&kv_map) : "memory");
        int looked = -1;
        for (int it = 0; it < n_tiles; ++it) {
            const int s = it % S::STAGES, round = it / S::STAGES;
            if (it % tiles_per_look == 0) {  // a page number per lane, for the next tiles
                const int block = ((start + it * BN) >> shift) + lane;
                looked = block < a.table_width ? __ldg(table + block) : -1;
            }
            int ok = 1;
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
            unsigned char* stage = ring + (size_t)s * 2 * S::TILE;
            if constexpr (E8) {  // the exponents of four keys or values a lane
                const int which = lane >> 4, key = (lane & 15) * 4;
                const int from = __shfl_sync(0xffffffffu, page, key >> shift);
                if (from >= 0) {
                    const signed char* src = a.exponents + (((size_t)from * 2 + which) * a.kv_heads + kvh) * a.page_size + (key & (a.page_size - 1));
                    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(exps + s * 128 + lane * 4)), "l"(src) : "memory");
                }
                asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(&full[s])) : "memory");
            }
            for (int op0 = 0; op0 < ops; op0 += 32) {
                const int op = op0 + lane;
                const int p = min(op, ops - 1) / OPS_PER_PAGE, rest = op % OPS_PER_PAGE, which = rest / S::PANELS, panel = rest - which * S::PANELS;
                const int from = __shfl_sync(0xffffffffu, page, p);
                if (op < ops && from >= 0)
                    tma_load_2d(stage + which * S::TILE + panel * (BN * S::PANEL_BYTES) + p * a.page_size * S::PANEL_BYTES, &kv_map, &full[s],
                                panel * (S::PANEL_BYTES / S::BYTES), ((from * 2 + which) * a.kv_heads + kvh) * a.page_size);
            }
        }
        return;
    }
    // ---------------------------------------------------------------------- consumers
    const int t = lane & 3, g = lane >> 2;
    unsigned qf[D / 16][4];
    float row_scale[2];
    int hi[2];  // the last key a row sees
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        const int v = g + r * 8, tok = v / a.gc, hh = v - tok * a.gc;
        const bool valid = tok < ntok && hh < heads_here;
        hi[r] = valid ? min(key_hi - 1, a.last[tok0 + tok]) : -1;
        const bf16* src = a.q + (size_t)(tok0 + (valid ? tok : 0)) * a.q_stride + (size_t)(first_head + (valid ? hh : 0)) * D;
        uint4 raw[D / 32];  // this lane's quarter of the row: chunks t, t + 4, ... of PER_CHUNK entries
        constexpr int PIECES = S::PER_CHUNK / 8;
#pragma unroll
        for (int i = 0; i < D / 32; ++i)
            raw[i] = valid ? *reinterpret_cast<const uint4*>(src + (t + 4 * (i / PIECES)) * S::PER_CHUNK + (i % PIECES) * 8) : make_uint4(0, 0, 0, 0);
        const unsigned* words = reinterpret_cast<const unsigned*>(raw);
        float factor = 1.f;
        if constexpr (E8) {
            // As float16 with the row's largest entry between 2^13 and 2^14: an entry of eight bits keeps them all down to 2^-27 of the largest.
            float largest = 0.f;
#pragma unroll
            for (int i = 0; i < D / 8; ++i) largest = fmaxf(largest, fmaxf(fabsf(__uint_as_float(words[i] << 16)), fabsf(__uint_as_float(words[i] & 0xffff0000u))));
            largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, 1));
            largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, 2));
            const int e = min(max((int)(__float_as_uint(largest) >> 23) - 127 - 13, -126), 126);
            factor = power_of_two(-e);
            row_scale[r] = a.scale_log2 * power_of_two(e);
        } else {
            row_scale[r] = a.scale_log2;
        }
#pragma unroll
        for (int i = 0; i < D / 8; ++i) {  // word i: entries 2 i, 2 i + 1 of the quarter; product i / 2, fragment register (i & 1) * 2 + r
            unsigned w = words[i];
            if constexpr (E8) w = pack<true>(__uint_as_float(w << 16) * factor, __uint_as_float(w & 0xffff0000u) * factor);
            qf[i >> 1][(i & 1) * 2 + r] = w;
        }
    }
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
    int top_e = -128;  // the largest exponent among the values so far
    float o[D / 8][4];
#pragma unroll
    for (int i = 0; i < D / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;

    for (int it = 0; it < n_tiles; ++it) {
        const int s = it % S::STAGES, round = it / S::STAGES;
        if (!mbar_wait(&full[s], round & 1, failed)) {
            *failed = 1;
            atomicOr(a.status, HB_STATUS_WAIT_EXPIRED | HB_STATUS_IN_ATTENTION_STRIPS);
            break;
        }
        const unsigned char* ks = ring + (size_t)s * 2 * S::TILE;
        const unsigned char* vs = ks + S::TILE;
        const int key0 = warp * 16, pos0 = start + it * BN + key0;  // this warp's keys
        if (pos0 < key_hi && pos0 + 16 > key_lo) {
            float sc[2][4];
#pragma unroll
            for (int n = 0; n < 2; ++n) sc[n][0] = sc[n][1] = sc[n][2] = sc[n][3] = 0.f;
#pragma unroll
            for (int j = 0; j < S::CHUNKS / 4; ++j) {
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    const uint4 raw = *reinterpret_cast<const uint4*>(ks + S::at(key0 + n * 8 + g, t + 4 * j));
                    const unsigned* words = reinterpret_cast<const unsigned*>(&raw);
#pragma unroll
                    for (int w = 0; w < S::STEPS; ++w) {
                        if constexpr (E8) mma<true>(sc[n], qf[j * S::STEPS + w], halves_of(words[w]), upper_halves_of(words[w]));
                        else mma<false>(sc[n], qf[j * S::STEPS + w], words[2 * w], words[2 * w + 1]);
                    }
                }
            }
            float back[2][2];  // 2^-e of the values' exponents
            bool far_apart = false;
            float mx[2] = {-INFINITY, -INFINITY};
            int low_e = 127;
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                float key_scale[2] = {1.f, 1.f}, value_e[2] = {0.f, 0.f};
                back[n][0] = back[n][1] = 1.f;
                if constexpr (E8) {
                    const unsigned char* ex = exps + s * 128 + key0 + n * 8 + t * 2;
                    const char2 ke = *reinterpret_cast<const char2*>(ex), ve = *reinterpret_cast<const char2*>(ex + 64);
#pragma unroll
                    for (int c = 0; c < 2; ++c) {  // what was never stored is no exponent: kept in range, it meets only scores that are replaced
                        const int k = min(max((int)(c ? ke.y : ke.x), -40), 40), v = min(max((int)(c ? ve.y : ve.x), -40), 40);
                        key_scale[c] = power_of_two(k);
                        value_e[c] = (float)v;
                        back[n][c] = power_of_two(-v);
                        const int pos = pos0 + n * 8 + t * 2 + c;
                        if (pos < key_hi && pos >= key_lo) low_e = min(low_e, v), top_e = max(top_e, v);
                    }
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int pos = pos0 + n * 8 + t * 2 + (e & 1);
                    float z = -INFINITY;
                    if (pos <= hi[e >> 1] && pos >= key_lo) z = fmaf(sc[n][e] * key_scale[e & 1], row_scale[e >> 1], value_e[e & 1]);
                    sc[n][e] = z;
                    mx[e >> 1] = fmaxf(mx[e >> 1], z);
                }
            }
            if constexpr (E8) {
                top_e = __reduce_max_sync(0xffffffffu, top_e);
                far_apart = top_e - __reduce_min_sync(0xffffffffu, low_e) > FAR_APART;
            }
            float alpha[2];
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 1));
                mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 2));
                const float m_new = fmaxf(m[r], mx[r] - (E8 ? HEADROOM : 0.f));
                alpha[r] = m_new == -INFINITY ? 1.f : fast_exp2(m[r] - m_new);
                m[r] = m_new;
                mx[r] = m_new == -INFINITY ? 0.f : m_new;
            }
            float sum[2] = {0.f, 0.f};
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float p = fast_exp2(sc[n][e] - mx[e >> 1]);
                    sc[n][e] = p;
                    sum[e >> 1] = E8 ? fmaf(p, back[n][e & 1], sum[e >> 1]) : sum[e >> 1] + p;
                }
#pragma unroll
            for (int r = 0; r < 2; ++r) l[r] = fmaf(l[r], alpha[r], sum[r]);  // of this lane's keys; the quad's lanes are added up at the end
            if (__any_sync(0xffffffffu, alpha[0] != 1.f || alpha[1] != 1.f)) {
#pragma unroll
                for (int i = 0; i < D / 8; ++i) o[i][0] *= alpha[0], o[i][1] *= alpha[0], o[i][2] *= alpha[1], o[i][3] *= alpha[1];
            }
            const unsigned pf[4] = {pack<E8>(sc[0][0], sc[0][1]), pack<E8>(sc[0][2], sc[0][3]), pack<E8>(sc[1][0], sc[1][1]), pack<E8>(sc[1][2], sc[1][3])};
            unsigned pr[4];  // bfloat16: what the weights lose by rounding, as weights of their own
            if constexpr (!E8) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    pr[i] = pack<false>(sc[i >> 1][(i & 1) * 2] - __uint_as_float(pf[i] << 16), sc[i >> 1][(i & 1) * 2 + 1] - __uint_as_float(pf[i] & 0xffff0000u));
            }
            // Values beyond the range read as zeros, whatever their slots hold.  A fragment register holds keys 2 t and 2 t + 1 in its halves.
            unsigned keep[2] = {0xffffffffu, 0xffffffffu};
            const bool whole = pos0 >= key_lo && pos0 + 16 <= key_hi;
            if (!whole) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int pos = pos0 + h * 8 + t * 2;
                    keep[h] = (pos >= key_lo && pos < key_hi ? 0xffffu : 0u) | (pos + 1 >= key_lo && pos + 1 < key_hi ? 0xffff0000u : 0u);
                }
            }
            if (E8 && far_apart) {
                // Weights by size, 2^18 at a time, each lot scaled up to where float16 holds it and the products scaled back.
#pragma unroll 1
                for (int lot = 0; lot < 7; ++lot) {
                    const float up = power_of_two(18 * lot), down = power_of_two(-18 * lot), from = lot < 6 ? down * 0x1p-10f : 0.f, to = lot ? down * 256.f : INFINITY;
                    unsigned part[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float p0 = sc[i >> 1][(i & 1) * 2], p1 = sc[i >> 1][(i & 1) * 2 + 1];
                        part[i] = pack<true>(p0 <= from || p0 > to ? 0.f : p0 * up, p1 <= from || p1 > to ? 0.f : p1 * up);
                    }
                    if (!__any_sync(0xffffffffu, (part[0] | part[1] | part[2] | part[3]) != 0)) continue;
#pragma unroll
                    for (int c = 0; c < S::CHUNKS; c += 2) {
                        unsigned b[4];
                        ldmatrix_x4_trans(b, vs + S::at(key0 + (lane & 15), c + (lane >> 4)));
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const unsigned b0 = __byte_perm(b[2 * h] & keep[0], 0, 0x3120), b1 = __byte_perm(b[2 * h + 1] & keep[1], 0, 0x3120);
                            float even[4] = {0.f, 0.f, 0.f, 0.f}, odd[4] = {0.f, 0.f, 0.f, 0.f};
                            mma<true>(even, part, halves_of(b0), halves_of(b1));
                            mma<true>(odd, part, upper_halves_of(b0), upper_halves_of(b1));
                            if constexpr (E8)
#pragma unroll
                                for (int e = 0; e < 4; ++e) o[2 * (c + h)][e] = fmaf(even[e], down, o[2 * (c + h)][e]), o[2 * (c + h) + 1][e] = fmaf(odd[e], down, o[2 * (c + h) + 1][e]);
                        }
                    }
                }
            } else
#pragma unroll
            for (int c = 0; c < S::CHUNKS; c += 2) {
                unsigned b[4];
                ldmatrix_x4_trans(b, vs + S::at(key0 + (lane & 15), c + (lane >> 4)));
                if (!whole) b[0] &= keep[0], b[1] &= keep[1], b[2] &= keep[0], b[3] &= keep[1];
#pragma unroll
                for (int h = 0; h < 2; ++h) {  // chunk c + h
                    if constexpr (E8) {
                        // bytes (key 2t: entries 2g, 2g + 1; key 2t + 1: the same) -> the two keys' even entries, and their odd ones
                        const unsigned b0 = __byte_perm(b[2 * h], 0, 0x3120), b1 = __byte_perm(b[2 * h + 1], 0, 0x3120);
                        mma<true>(o[2 * (c + h)], pf, halves_of(b0), halves_of(b1));
                        mma<true>(o[2 * (c + h) + 1], pf, upper_halves_of(b0), upper_halves_of(b1));
                    } else {
                        mma<false>(o[c + h], pf, b[2 * h], b[2 * h + 1]);
                        mma<false>(o[c + h], pr, b[2 * h], b[2 * h + 1]);
                    }
                }
            }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[s]);
    }
    // The warps' results meet in the ring, which no copy targets any more once all of them have passed the last stage.
    asm volatile("bar.sync 1, %0;" ::"n"(32 * WARPS) : "memory");
    float* wo = reinterpret_cast<float*>(ring);  // [WARPS][ROWS][D]
    float* wm = wo + WARPS * ROWS * D;           // [WARPS][ROWS]
    float* wl = wm + WARPS * ROWS;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        const int row = g + r * 8;
        l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
        l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
        if (t == 0) wm[warp * ROWS + row] = m[r], wl[warp * ROWS + row] = l[r];
        float* dst = wo + ((size_t)warp * ROWS + row) * D;
        if constexpr (E8) {
#pragma unroll
            for (int c = 0; c < D / 16; ++c)
                *reinterpret_cast<float4*>(dst + 16 * c + 4 * t) = make_float4(o[2 * c][2 * r], o[2 * c + 1][2 * r], o[2 * c][2 * r + 1], o[2 * c + 1][2 * r + 1]);
        } else {
#pragma unroll
            for (int n = 0; n < D / 8; ++n) *reinterpret_cast<float2*>(dst + 8 * n + 2 * t) = make_float2(o[n][2 * r], o[n][2 * r + 1]);
        }
    }
    asm volatile("bar.sync 1, %0;" ::"n"(32 * WARPS) : "memory");
    if (*failed) return;
    for (int e = tid; e < ROWS * (D / 4); e += 32 * WARPS) {
        const int row = e / (D / 4), c = (e - row * (D / 4)) * 4, tok = row / a.gc, hh = row - tok * a.gc;
        if (tok >= ntok || hh >= heads_here) continue;
        float top = -INFINITY, total = 0.f, value[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < WARPS; ++w) top = fmaxf(top, wm[w * ROWS + row]);
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            const float mw = wm[w * ROWS + row], f = mw == -INFINITY ? 0.f : fast_exp2(mw - top);
            total = fmaf(f, wl[w * ROWS + row], total);
            float part[4];
            load4(wo + ((size_t)w * ROWS + row) * D + c, part);
#pragma unroll
            for (int i = 0; i < 4; ++i) value[i] = fmaf(f, part[i], value[i]);
        }
        const int token = tok0 + tok, head = first_head + hh;
        if (a.pieces) {
            const size_t slot = (size_t)(a.piece_start[token] + piece) * a.heads + head;
            store4(a.pieces + slot * D + c, value);
            if (c == 0) a.sums[slot] = make_float2(top, total);
        } else {
            const float inv = total > 0.f ? 1.f / total : (total == 0.f ? 0.f : total);  // a row that sees nothing is zeros; a NaN stays one
#pragma unroll
            for (int i = 0; i < 4; ++i) value[i] *= inv;
            store4(a.out + (size_t)token * a.out_stride + (size_t)head * D + c, value);
        }
    }
}

__device__ __forceinline__ void load_floats(const float* p, float (&v)[4]) { load4(p, v); }
__device__ __forceinline__ void load_floats(const float* p, float (&v)[2]) {
    const float2 x = *reinterpret_cast<const float2*>(p);
    v[0] = x.x, v[1] = x.y;
}

// A warp puts a (token, head)'s pieces together.
constexpr int MERGE_WARPS = 4;
__global__ void __launch_bounds__(32 * MERGE_WARPS) attention_pieces_kernel(const float* __restrict__ pieces, const float2* __restrict__ sums, const int* __restrict__ piece_start,
                                                                            bf16* __restrict__ out, int out_stride, int heads) {
    constexpr int PER = D / 32, AHEAD = 8;
    let_next_kernel_start();
    wait_for_previous_kernels();
    const int token = blockIdx.x, head = blockIdx.y * MERGE_WARPS + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (head >= heads) return;
    const int first = piece_start[token], n = piece_start[token + 1] - first;
    float top = -INFINITY, total = 0.f, value[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) value[i] = 0.f;
    for (int p = lane; p < n; p += 32) top = fmaxf(top, sums[(size_t)(first + p) * heads + head].x);
    top = warp_max(top);
    for (int p0 = 0; p0 < n; p0 += AHEAD) {  // AHEAD pieces are on their way together
        float part[AHEAD][PER];
        float2 ml[AHEAD];
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
            if (p0 + k >= n) break;
            const size_t slot = (size_t)(first + p0 + k) * heads + head;
            ml[k] = sums[slot];
            const float* src = pieces + slot * D + lane * PER;
            load_floats(src, part[k]);
        }
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
            if (p0 + k >= n) break;
            const float f = ml[k].x == -INFINITY ? 0.f : fast_exp2(ml[k].x - top);
            total = fmaf(f, ml[k].y, total);
#pragma unroll
            for (int i = 0; i < PER; ++i) value[i] = fmaf(f, part[k][i], value[i]);
        }
    }
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
template <bool E8>
int cache_map(CUtensorMap* map, const void* cache, int pages, int kv_heads, int page_size) {
    EncodeTiled encode = encode_tiled();
    if (!encode) return HB_BAD_ARGUMENT;
    const cuuint64_t dims[2] = {(cuuint64_t)D, (cuuint64_t)pages * 2 * kv_heads * page_size};
    const cuuint64_t strides[1] = {(cuuint64_t)D * Shape<E8>::BYTES};
    const cuuint32_t box[2] = {(cuuint32_t)(Shape<E8>::PANEL_BYTES / Shape<E8>::BYTES), (cuuint32_t)page_size};
    const cuuint32_t elem[2] = {1, 1};
    const CUresult r = encode(map, E8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(cache), dims, strides, box, elem,
                              CU_TENSOR_MAP_INTERLEAVE_NONE, Shape<E8>::PANEL_BYTES == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B,
                              CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? 0 : HB_BAD_ARGUMENT;
}

template <bool E8>
int launch_strips(const Args& a, const void* cache, int n_items, cudaStream_t stream) {
    CUtensorMap map;
    if (int code = cache_map<E8>(&map, cache, a.pages, a.kv_heads, a.page_size)) return code;
    static const cudaError_t configured = cudaFuncSetAttribute(attention_strip_kernel<E8>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Shape<E8>::SMEM);
    if (configured != cudaSuccess) return (int)configured;
    return launch_after_previous(attention_strip_kernel<E8>, dim3(n_items, a.kv_heads * a.chunks), dim3(THREADS), Shape<E8>::SMEM, stream, map, a);
}
}  // namespace

// cache: [pages, 2, kv_heads, page_size, D] in bfloat16 (exponents null) or e4m3 codes with exponents [pages, 2, kv_heads, page_size].
// strips [n_strips, 6]: see ITEM_WORDS; a strip has at most 16 / min(heads / kv_heads, 16) tokens.  pieces, sums null: one piece a row.
HB_EXPORT int hb_attention_strips(const void* q, int q_stride, void* out, int out_stride, const void* cache, const void* exponents, const int* block_table, int table_width,
                                  const int* strips, int n_strips, const int* last, const int* piece_start, float* pieces, float* sums, int heads, int kv_heads,
                                  int page_size, int pages, float scale, int* status, cudaStream_t stream) {
    if (n_strips <= 0) return 0;
    if (!q || !out || !cache || !block_table || !strips || !last || !piece_start || !status || (!pieces != !sums)) return HB_BAD_ARGUMENT;
    if (kv_heads <= 0 || heads <= 0 || heads % kv_heads || pages <= 0 || table_width <= 0 || q_stride % 8 || out_stride % 4) return HB_BAD_ARGUMENT;
    if (page_size < 8 || page_size > 64 || (page_size & (page_size - 1))) return HB_UNSUPPORTED_SIZE;
    if ((((uintptr_t)q | (uintptr_t)cache | (uintptr_t)pieces) & 15) || ((uintptr_t)exponents & 3) || ((uintptr_t)out & 7)) return HB_BAD_ARGUMENT;
    if ((long long)pages * 2 * kv_heads * page_size > 0x7fffffffLL) return HB_UNSUPPORTED_SIZE;  // a row's number in the cache's tensor map
    const int group = heads / kv_heads, gc = group < ROWS ? group : ROWS, chunks = (group + gc - 1) / gc;
    if ((long long)kv_heads * chunks > 65535) return HB_UNSUPPORTED_SIZE;
    const Args a{(const bf16*)q, q_stride, (bf16*)out, out_stride, (const signed char*)exponents, block_table, table_width, strips, last, piece_start, pieces, (float2*)sums,
                 heads, kv_heads, page_size, pages, gc, chunks, scale * 1.4426950408889634f, status};
    return exponents ? launch_strips<true>(a, cache, n_strips, stream) : launch_strips<false>(a, cache, n_strips, stream);
}

// Puts the pieces [piece_start[tokens], heads, D] of every token together.  A token without a piece is zeros.
HB_EXPORT int hb_attention_pieces(const float* pieces, const float* sums, const int* piece_start, void* out, int out_stride, int tokens, int heads, cudaStream_t stream) {
    if (tokens <= 0) return 0;
    if (!pieces || !sums || !piece_start || !out || heads <= 0 || out_stride % 2 || ((uintptr_t)pieces & 15) || ((uintptr_t)out & 3)) return HB_BAD_ARGUMENT;
    const int rows = (heads + MERGE_WARPS - 1) / MERGE_WARPS;
    if (rows > 65535) return HB_UNSUPPORTED_SIZE;
    return launch_after_previous(attention_pieces_kernel, dim3(tokens, rows), dim3(32 * MERGE_WARPS), 0, stream, pieces, (const float2*)sums, piece_start, (bf16*)out, out_stride, heads);
}
