// A paged cache whose keys and values are held in 8 bits: records (a key or a value of one head and position) are quantised as they are
// written, and read back.
//
//   e = the smallest integer in [-40, 40] with max|x| <= 448 * 2^e          (-40 for a record of zeros)
//   code_i = x_i * 2^-e rounded to e4m3 (nearest, ties to even), beyond 448 to +-448; a NaN stays one and takes no part in the maximum
//   value_i = code_i * 2^e
//
// The scale is a power of two: e4m3 is itself a floating format, so a finer scale would not make the typical entry's relative error (at most
// 2^-4) any smaller, and with powers of two both directions are exact but for the one rounding: the codes are the same bits whoever computes
// them, and a value fits bfloat16 without another rounding.  The bounds of e keep products of two scales inside float's range.
//
// codes [pages, 2, kv_heads, page, d] bytes, exponents [pages, 2, kv_heads, page] signed bytes.  Both kernels are bound by memory: a thread
// holds eight entries (16 bytes in bfloat16, 8 in codes), the threads of a record stand side by side, and a thread serves PER tokens at once
// so that their loads are on their way together.
#include "common.cuh"

namespace {
typedef __nv_bfloat16 bf16;
constexpr int THREADS = 256;
constexpr int LOW_EXPONENT = -40, HIGH_EXPONENT = 40;

// The exponent of a record from its largest magnitude's bits: 448 = 1.75 * 2^8.
__device__ __forceinline__ int record_exponent(float largest) {
    const unsigned bits = __float_as_uint(largest);
    const int e = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
    return min(max(e, LOW_EXPONENT), HIGH_EXPONENT);
}
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float((unsigned)(127 + e) << 23); }
__device__ __forceinline__ unsigned short codes_of(float lo, float hi) {
    unsigned short c;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(c) : "f"(hi), "f"(lo));
    return c;
}
__device__ __forceinline__ void values_of(unsigned short codes, float scale, float& lo, float& hi) {
    unsigned halves;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(halves) : "h"(codes));
    float a, b;
    asm("{.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.f32.f16 %0, l;\n\tcvt.f32.f16 %1, h;\n\t}" : "=f"(a), "=f"(b) : "r"(halves));
    lo = a * scale, hi = b * scale;
}

struct Places {
    const int* block_table; int table_width;
    const int* token_row; const int* positions;
    int tokens, kv_heads, head_dim, page_size, pages;
    int lanes_log;  // threads of a record, as a power of two
    int* status;
};

// A thread's place: the record (`which`: 0 key, 1 value) and the first of its eight entries; its tokens are first_token .. + PER - 1.
struct Unit {
    int token, which, head, d;
    bool active;
};
__device__ __forceinline__ Unit unit_of(const Places& p, int per) {
    const int records = 2 * p.kv_heads, units = records << p.lanes_log;
    const unsigned i = blockIdx.x * THREADS + threadIdx.x;
    const int group = i / units, u = i - group * units, record = u >> p.lanes_log;
    Unit x;
    x.token = group * per;
    x.which = record >= p.kv_heads ? 1 : 0;
    x.head = record - x.which * p.kv_heads;
    x.d = (u & ((1 << p.lanes_log) - 1)) * 8;
    x.active = x.d < p.head_dim;
    return x;
}
// Where a token's record of this unit starts, counted in records; -1 for a token beyond the batch, or without a page (which is reported).
__device__ __forceinline__ long long record_of(const Places& p, const Unit& u, int token) {
    if (token >= p.tokens) return -1;
    const int pos = p.positions[token], block = pos / p.page_size;
    const int page = pos >= 0 && block < p.table_width ? p.block_table[(size_t)p.token_row[token] * p.table_width + block] : -1;
    if (page < 0 || page >= p.pages) {
        if (u.which == 0 && u.head == 0 && u.d == 0) atomicOr(p.status, HB_STATUS_BAD_PAGE);
        return -1;
    }
    return (((long long)page * 2 + u.which) * p.kv_heads + u.head) * p.page_size + (pos - block * p.page_size);
}

template <typename T, bool WIDE>
__device__ __forceinline__ void load_entries(const T* p, float (&v)[8]) {
    if constexpr (WIDE) {
        load8(p, v);
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = to_float(p[k]);
    }
}

// WIDE: rows and columns of the source stand on 16-byte boundaries.
template <typename T, int PER, bool WIDE>
__global__ void __launch_bounds__(THREADS) cache8_store_kernel(const T* __restrict__ src, int stride, int k_offset, int v_offset, const Places p,
                                                               uint2* __restrict__ codes, signed char* __restrict__ exponents) {
    let_next_kernel_start();
    wait_for_previous_kernels();
    const Unit u = unit_of(p, PER);
    long long record[PER];
    float x[PER][8];
#pragma unroll
    for (int k = 0; k < PER; ++k) {
        const int token = u.token + k;
        if (token < p.tokens && u.active) {
            load_entries<T, WIDE>(src + (size_t)token * stride + (u.which ? v_offset : k_offset) + u.head * p.head_dim + u.d, x[k]);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) x[k][e] = 0.f;
        }
        record[k] = record_of(p, u, token);
    }
#pragma unroll
    for (int k = 0; k < PER; ++k) {
        float largest = 0.f;  // fmaxf passes over a NaN
#pragma unroll
        for (int e = 0; e < 8; ++e) largest = fmaxf(largest, fabsf(x[k][e]));
        for (int offset = 1 << p.lanes_log >> 1; offset > 0; offset >>= 1) largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, offset));
        const int e = record_exponent(largest);
        const float scale = power_of_two(-e);
        if (record[k] < 0 || !u.active) continue;
        uint2 packed;
        unsigned short* pairs = reinterpret_cast<unsigned short*>(&packed);
#pragma unroll
        for (int i = 0; i < 4; ++i) pairs[i] = codes_of(x[k][2 * i] * scale, x[k][2 * i + 1] * scale);
        codes[(record[k] * p.head_dim + u.d) >> 3] = packed;
        if (u.d == 0) exponents[record[k]] = (signed char)e;
    }
}

// out [tokens, 2, kv_heads, d]; a token without a page reads as zeros.
template <typename T, int PER>
__global__ void __launch_bounds__(THREADS) cache8_load_kernel(const uint2* __restrict__ codes, const signed char* __restrict__ exponents, const Places p,
                                                              T* __restrict__ out) {
    let_next_kernel_start();
    wait_for_previous_kernels();
    const Unit u = unit_of(p, PER);
    if (!u.active) return;
    uint2 packed[PER];
    int e[PER];
#pragma unroll
    for (int k = 0; k < PER; ++k) {
        const long long record = record_of(p, u, u.token + k);
        packed[k] = record < 0 ? make_uint2(0, 0) : codes[(record * p.head_dim + u.d) >> 3];
        e[k] = record < 0 ? 0 : exponents[record];
    }
#pragma unroll
    for (int k = 0; k < PER; ++k) {
        const int token = u.token + k;
        if (token >= p.tokens) break;
        const unsigned short* pairs = reinterpret_cast<const unsigned short*>(&packed[k]);
        const float scale = power_of_two(e[k]);
        float v[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) values_of(pairs[i], scale, v[2 * i], v[2 * i + 1]);
        store8(out + (((size_t)token * 2 + u.which) * p.kv_heads + u.head) * p.head_dim + u.d, v);
    }
}

int places(Places& p, const int* block_table, int table_width, const int* token_row, const int* positions, int tokens, int kv_heads, int head_dim, int page_size,
           int pages, int* status) {
    if (!block_table || !token_row || !positions || !status || table_width <= 0 || kv_heads <= 0 || page_size <= 0 || pages <= 0) return HB_BAD_ARGUMENT;
    if (head_dim <= 0 || head_dim % 8 || head_dim > 256) return HB_UNSUPPORTED_SIZE;
    int lanes_log = 0;
    while ((8 << lanes_log) < head_dim) ++lanes_log;
    if ((long long)tokens * ((2LL * kv_heads) << lanes_log) > 0x7fffffffLL - THREADS) return HB_UNSUPPORTED_SIZE;
    p = Places{block_table, table_width, token_row, positions, tokens, kv_heads, head_dim, page_size, pages, lanes_log, status};
    return 0;
}
unsigned blocks_for(const Places& p, int per) {
    const long long groups = (p.tokens + per - 1) / per;
    return (unsigned)((groups * ((2LL * p.kv_heads) << p.lanes_log) + THREADS - 1) / THREADS);
}
constexpr int PER = 4;
// Four tokens a thread once their threads alone fill the device (148 SMs of 2,048 threads); below that one, for the shorter way of a thread.
bool takes_several(const Places& p) { return (long long)p.tokens * ((2LL * p.kv_heads) << p.lanes_log) >= (long long)PER * 148 * 2048; }
}  // namespace

HB_EXPORT int hb_cache8_store(const void* src, int is_bf16, int stride, int k_offset, int v_offset, void* codes, void* exponents, const int* block_table,
                              int table_width, const int* token_row, const int* positions, int tokens, int kv_heads, int head_dim, int page_size, int pages,
                              int* status, cudaStream_t stream) {
    if (tokens <= 0) return 0;
    if (!src || !codes || !exponents || k_offset < 0 || v_offset < 0 || ((uintptr_t)codes & 7)) return HB_BAD_ARGUMENT;
    Places p;
    if (int code = places(p, block_table, table_width, token_row, positions, tokens, kv_heads, head_dim, page_size, pages, status)) return code;
    const int per16 = is_bf16 ? 8 : 4;
    const bool wide = !((uintptr_t)src & 15) && stride % per16 == 0 && k_offset % per16 == 0 && v_offset % per16 == 0;
    const bool several = takes_several(p);
#define HB_STORE(T, N, W) \
    return launch_after_previous(cache8_store_kernel<T, N, W>, dim3(blocks_for(p, N)), dim3(THREADS), 0, stream, (const T*)src, stride, k_offset, v_offset, p, (uint2*)codes, (signed char*)exponents)
    if (is_bf16) {
        if (!wide) HB_STORE(bf16, 1, false);
        if (several) HB_STORE(bf16, PER, true);
        HB_STORE(bf16, 1, true);
    }
    if (!wide) HB_STORE(float, 1, false);
    if (several) HB_STORE(float, PER, true);
    HB_STORE(float, 1, true);
#undef HB_STORE
}

HB_EXPORT int hb_cache8_load(const void* codes, const void* exponents, const int* block_table, int table_width, const int* token_row, const int* positions,
                             void* out, int is_bf16, int tokens, int kv_heads, int head_dim, int page_size, int pages, int* status, cudaStream_t stream) {
    if (tokens <= 0) return 0;
    if (!codes || !exponents || !out || ((uintptr_t)codes & 7) || ((uintptr_t)out & 15)) return HB_BAD_ARGUMENT;
    Places p;
    if (int code = places(p, block_table, table_width, token_row, positions, tokens, kv_heads, head_dim, page_size, pages, status)) return code;
    const bool several = takes_several(p);
#define HB_LOAD(T, N) \
    return launch_after_previous(cache8_load_kernel<T, N>, dim3(blocks_for(p, N)), dim3(THREADS), 0, stream, (const uint2*)codes, (const signed char*)exponents, p, (T*)out)
    if (is_bf16) {
        if (several) HB_LOAD(bf16, PER);
        HB_LOAD(bf16, 1);
    }
    if (several) HB_LOAD(float, PER);
    HB_LOAD(float, 1);
#undef HB_LOAD
}
