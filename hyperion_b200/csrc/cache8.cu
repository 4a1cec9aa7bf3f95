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
// codes [pages, 2, kv_heads, page, d] bytes, exponents [pages, 2, kv_heads, page] signed bytes.  Both kernels are bound by memory: the threads of a record stand side by
// side with WIDTH entries each, and a thread serves PER tokens whose places are all looked up, and whose entries are all fetched, before the first is used.  To and
// from bfloat16, heads of 128: 8,191 tokens of 8 heads are written in 12.1 us (50 MB, 4.2 TB/s: one turn of the device, a start and two dependent trips to memory),
// 131,072 of 4 heads read in 76 us (404 MB, 5.3 TB/s, 0.82 of a plain copy's rate).
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
    int lanes_log;   // threads of a record, as a power of two
    int page_shift;  // of a page size that is a power of two, or -1
    int* status;
};

// A thread's place: the record (`which`: 0 key, 1 value) and the first of its entries; its tokens are token .. token + PER - 1.
struct Unit {
    int token, which, head, d;
    bool active;
};
template <int WIDTH, int PER>
__device__ __forceinline__ Unit unit_of(const Places& p) {
    const unsigned units = (unsigned)(2 * p.kv_heads) << p.lanes_log, i = blockIdx.x * THREADS + threadIdx.x;
    const unsigned group = i / units, u = i - group * units, record = u >> p.lanes_log;
    Unit x;
    x.token = (int)group * PER;
    x.which = record >= (unsigned)p.kv_heads ? 1 : 0;
    x.head = (int)record - x.which * p.kv_heads;
    x.d = (int)(u & ((1u << p.lanes_log) - 1)) * WIDTH;
    x.active = x.d < p.head_dim;
    return x;
}
// Where the records of this unit's tokens start, counted in records; -1 for a token beyond the batch, or without a page (which is reported).  No branch stands between
// the look-ups, so that they are on their way together.
template <int PER>
__device__ __forceinline__ void records_of(const Places& p, const Unit& u, long long (&record)[PER]) {
    int pos[PER], row[PER], page[PER];
#pragma unroll
    for (int k = 0; k < PER; ++k) {
        const int token = min(u.token + k, p.tokens - 1);
        pos[k] = p.positions[token];
        row[k] = p.token_row[token];
    }
    bool missing = false;
#pragma unroll
    for (int k = 0; k < PER; ++k) {
        const int block = p.page_shift >= 0 ? pos[k] >> p.page_shift : pos[k] / p.page_size;
        const bool inside = pos[k] >= 0 && block < p.table_width;
        page[k] = p.block_table[inside ? (size_t)row[k] * p.table_width + block : 0];
        if (!inside) page[k] = -1;
    }
#pragma unroll
    for (int k = 0; k < PER; ++k) {
        const bool there = page[k] >= 0 && page[k] < p.pages, wanted = u.token + k < p.tokens;
        const int slot = p.page_shift >= 0 ? pos[k] & (p.page_size - 1) : pos[k] % p.page_size;
        record[k] = wanted && there ? (((long long)page[k] * 2 + u.which) * p.kv_heads + u.head) * p.page_size + slot : -1;
        missing |= wanted && !there;
    }
    if (missing && u.which == 0 && u.head == 0 && u.d == 0) atomicOr(p.status, HB_STATUS_BAD_PAGE);
}

// WIDTH entries of a row as they stand in memory.  ALIGNED: their first is on a boundary of their size (32 bytes at most).
template <typename T, int WIDTH>
struct Entries {
    static constexpr int WORDS = WIDTH * (int)sizeof(T) / 4;
    unsigned words[WORDS];
    __device__ __forceinline__ float operator[](int i) const {
        if constexpr (sizeof(T) == 4) return __uint_as_float(words[i]);
        else return __uint_as_float(i & 1 ? words[i >> 1] & 0xffff0000u : words[i >> 1] << 16);
    }
};
__device__ __forceinline__ void fetch32(const void* p, unsigned* w) {
    asm volatile("ld.global.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7]) : "l"(p));
}
__device__ __forceinline__ void put32(void* p, const unsigned* w) {
    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7]) : "memory");
}
template <typename T, int WIDTH, bool ALIGNED>
__device__ __forceinline__ void fetch(const T* p, Entries<T, WIDTH>& x) {
    constexpr int WORDS = Entries<T, WIDTH>::WORDS;
    if constexpr (!ALIGNED) {
#pragma unroll
        for (int i = 0; i < WORDS; ++i) {
            if constexpr (sizeof(T) == 4) x.words[i] = __float_as_uint(p[i]);
            else x.words[i] = (unsigned)__bfloat16_as_ushort(p[2 * i]) | (unsigned)__bfloat16_as_ushort(p[2 * i + 1]) << 16;
        }
    } else if constexpr (WORDS % 8 == 0) {
#pragma unroll
        for (int i = 0; i < WORDS; i += 8) fetch32(reinterpret_cast<const unsigned*>(p) + i, x.words + i);
    } else {
        const uint4 w = *reinterpret_cast<const uint4*>(p);
        x.words[0] = w.x, x.words[1] = w.y, x.words[2] = w.z, x.words[3] = w.w;
    }
}
template <int WIDTH>
__device__ __forceinline__ void put_codes(unsigned char* p, const unsigned (&w)[WIDTH / 4]) {
    if constexpr (WIDTH == 16) *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    else *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
}
template <int WIDTH>
__device__ __forceinline__ void fetch_codes(const unsigned char* p, unsigned (&w)[WIDTH / 4]) {
    if constexpr (WIDTH == 16) {
        const uint4 x = *reinterpret_cast<const uint4*>(p);
        w[0] = x.x, w[1] = x.y, w[2] = x.z, w[3] = x.w;
    } else {
        const uint2 x = *reinterpret_cast<const uint2*>(p);
        w[0] = x.x, w[1] = x.y;
    }
}

template <typename T, int WIDTH, int PER, bool ALIGNED>
__global__ void __launch_bounds__(THREADS) cache8_store_kernel(const T* __restrict__ src, int stride, int k_offset, int v_offset, const Places p,
                                                               unsigned char* __restrict__ codes, signed char* __restrict__ exponents) {
    let_next_kernel_start();
    wait_for_previous_kernels();
    const Unit u = unit_of<WIDTH, PER>(p);
    Entries<T, WIDTH> x[PER];
#pragma unroll
    for (int k = 0; k < PER; ++k)  // a thread beyond the record's entries reads its first ones, and brings nothing
        fetch<T, WIDTH, ALIGNED>(src + (size_t)min(u.token + k, p.tokens - 1) * stride + (u.which ? v_offset : k_offset) + u.head * p.head_dim + (u.active ? u.d : 0), x[k]);
    long long record[PER];
    records_of<PER>(p, u, record);
#pragma unroll
    for (int k = 0; k < PER; ++k) {
        float largest = 0.f;  // fmaxf passes over a NaN
#pragma unroll
        for (int e = 0; e < WIDTH; ++e) largest = fmaxf(largest, fabsf(x[k][e]));
        for (int offset = 1 << p.lanes_log >> 1; offset > 0; offset >>= 1) largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, offset));
        const int e = record_exponent(largest);
        const float scale = power_of_two(-e);
        unsigned packed[WIDTH / 4];
#pragma unroll
        for (int i = 0; i < WIDTH / 4; ++i)
            packed[i] = (unsigned)codes_of(x[k][4 * i] * scale, x[k][4 * i + 1] * scale) | (unsigned)codes_of(x[k][4 * i + 2] * scale, x[k][4 * i + 3] * scale) << 16;
        if (record[k] < 0 || !u.active) continue;
        put_codes<WIDTH>(codes + record[k] * p.head_dim + u.d, packed);
        if (u.d == 0) exponents[record[k]] = (signed char)e;
    }
}

// out [tokens, 2, kv_heads, d]; a token without a page reads as zeros.
template <typename T, int WIDTH, int PER>
__global__ void __launch_bounds__(THREADS) cache8_load_kernel(const unsigned char* __restrict__ codes, const signed char* __restrict__ exponents, const Places p,
                                                              T* __restrict__ out) {
    let_next_kernel_start();
    wait_for_previous_kernels();
    const Unit u = unit_of<WIDTH, PER>(p);
    if (!u.active) return;
    long long record[PER];
    records_of<PER>(p, u, record);
    unsigned packed[PER][WIDTH / 4];
    int e[PER];
#pragma unroll
    for (int k = 0; k < PER; ++k) {
        const long long from = max(record[k], 0ll);
        fetch_codes<WIDTH>(codes + from * p.head_dim + u.d, packed[k]);
        e[k] = exponents[from];
    }
#pragma unroll
    for (int k = 0; k < PER; ++k) {
        const int token = u.token + k;
        if (token >= p.tokens) break;
        const float scale = power_of_two(e[k]);
        constexpr int WORDS = WIDTH * (int)sizeof(T) / 4;
        unsigned words[WORDS];
#pragma unroll
        for (int i = 0; i < WIDTH / 2; ++i) {
            float lo, hi;
            values_of((unsigned short)(packed[k][i >> 1] >> (i & 1) * 16), scale, lo, hi);
            if (record[k] < 0) lo = hi = 0.f;
            if constexpr (sizeof(T) == 4) {
                words[2 * i] = __float_as_uint(lo), words[2 * i + 1] = __float_as_uint(hi);
            } else {
                const __nv_bfloat162 both = __floats2bfloat162_rn(lo, hi);
                words[i] = *reinterpret_cast<const unsigned*>(&both);
            }
        }
        T* dst = out + (((size_t)token * 2 + u.which) * p.kv_heads + u.head) * p.head_dim + u.d;
        if constexpr (WORDS % 8 == 0) {
#pragma unroll
            for (int i = 0; i < WORDS; i += 8) put32(reinterpret_cast<unsigned*>(dst) + i, words + i);
        } else {
            *reinterpret_cast<uint4*>(dst) = make_uint4(words[0], words[1], words[2], words[3]);
        }
    }
}

int places(Places& p, const int* block_table, int table_width, const int* token_row, const int* positions, int tokens, int kv_heads, int head_dim, int page_size,
           int pages, int* status) {
    if (!block_table || !token_row || !positions || !status || table_width <= 0 || kv_heads <= 0 || page_size <= 0 || pages <= 0) return HB_BAD_ARGUMENT;
    if (head_dim <= 0 || head_dim % 8 || head_dim > 256) return HB_UNSUPPORTED_SIZE;
    if ((long long)tokens * (2LL * kv_heads) * 32 > 0x7fffffffLL - THREADS) return HB_UNSUPPORTED_SIZE;
    int shift = 0;
    while ((1 << shift) < page_size) ++shift;
    p = Places{block_table, table_width, token_row, positions, tokens, kv_heads, head_dim, page_size, pages, 0, (1 << shift) == page_size ? shift : -1, status};
    return 0;
}
// Threads of a record, and how many blocks there are.
unsigned set_width(Places& p, int width, int per) {
    p.lanes_log = 0;
    while ((width << p.lanes_log) < p.head_dim) ++p.lanes_log;
    const long long groups = (p.tokens + per - 1) / per;
    return (unsigned)((groups * ((2LL * p.kv_heads) << p.lanes_log) + THREADS - 1) / THREADS);
}
constexpr int PER = 4;
// Four tokens and sixteen entries a thread once their threads alone fill the device (multiprocessors of 1,024 such threads); below that one token and eight entries, for the
// shorter way of a thread: 700 tokens of 4 heads of 128 read back in 2.6 us.
bool takes_several(const Places& p, int sms) { return p.head_dim % 16 == 0 && (long long)p.tokens * 2 * p.kv_heads * p.head_dim >= (long long)PER * 16 * 1024 * sms; }
}  // namespace

HB_EXPORT int hb_cache8_store(const void* src, int is_bf16, long long stride, long long k_offset, long long v_offset, void* codes, void* exponents, const int* block_table,
                              int table_width, const int* token_row, const int* positions, int tokens, int kv_heads, int head_dim, int page_size, int pages,
                              int sms, int* status, cudaStream_t stream) {
    if (tokens <= 0) return 0;
    if (!src || !codes || !exponents || k_offset < 0 || v_offset < 0 || ((uintptr_t)codes & 15)) return HB_BAD_ARGUMENT;
    Places p;
    if (int code = places(p, block_table, table_width, token_row, positions, tokens, kv_heads, head_dim, page_size, pages, status)) return code;
    if (stride > 0x7fffffffLL || k_offset > 0x7fffffffLL || v_offset > 0x7fffffffLL) return HB_UNSUPPORTED_SIZE;
    const unsigned element = is_bf16 ? 2 : 4;
    const auto on = [&](unsigned bytes) {  // every record starts on such a boundary
        return !(((uintptr_t)src | (uintptr_t)stride * element | (uintptr_t)k_offset * element | (uintptr_t)v_offset * element | (uintptr_t)head_dim * element) & (bytes - 1));
    };
#define HB_STORE(T, WIDTH, N, ALIGNED)                                                                                                                     \
    do {                                                                                                                                                   \
        const unsigned blocks = set_width(p, WIDTH, N);                                                                                                    \
        return launch_after_previous(cache8_store_kernel<T, WIDTH, N, ALIGNED>, dim3(blocks), dim3(THREADS), 0, stream, (const T*)src, (int)stride, (int)k_offset, \
                                     (int)v_offset, p, (unsigned char*)codes, (signed char*)exponents);                                                         \
    } while (0)
    if (is_bf16) {
        if (on(32) && takes_several(p, sms)) HB_STORE(bf16, 16, PER, true);
        if (on(16)) HB_STORE(bf16, 8, 1, true);
        HB_STORE(bf16, 8, 1, false);
    }
    if (on(32)) HB_STORE(float, 8, 1, true);
    HB_STORE(float, 8, 1, false);
#undef HB_STORE
}

HB_EXPORT int hb_cache8_load(const void* codes, const void* exponents, const int* block_table, int table_width, const int* token_row, const int* positions,
                             void* out, int is_bf16, int tokens, int kv_heads, int head_dim, int page_size, int pages, int sms, int* status, cudaStream_t stream) {
    if (tokens <= 0) return 0;
    if (!codes || !exponents || !out || ((uintptr_t)codes & 15) || ((uintptr_t)out & 31)) return HB_BAD_ARGUMENT;
    Places p;
    if (int code = places(p, block_table, table_width, token_row, positions, tokens, kv_heads, head_dim, page_size, pages, status)) return code;
    const bool several = takes_several(p, sms);
#define HB_LOAD(T, WIDTH, N)                                                                                                                               \
    do {                                                                                                                                                   \
        const unsigned blocks = set_width(p, WIDTH, N);                                                                                                    \
        return launch_after_previous(cache8_load_kernel<T, WIDTH, N>, dim3(blocks), dim3(THREADS), 0, stream, (const unsigned char*)codes,                 \
                                     (const signed char*)exponents, p, (T*)out);                                                                           \
    } while (0)
    if (is_bf16) {
        if (several) HB_LOAD(bf16, 16, PER);
        HB_LOAD(bf16, 8, 1);
    }
    if (several) HB_LOAD(float, 16, 2);
    HB_LOAD(float, 8, 1);
#undef HB_LOAD
}
