// Drafted tokens against the target model's logits, from given random numbers (speculative sampling).
//
// A request brings n drafted tokens and n + 1 rows of logits.  With p_i = softmax(row i / temperature) and q_i the drafter's probabilities
// (a token that stands for itself where there are none: q_i = 1 there), draft x_i stands when u_i q_i(x_i) < p_i(x_i).  The first one that
// does not is replaced by a draw from max(p_i - q_i, 0), normalised; when all stand, one more token is drawn from p_n.  A draw from weights w
// is argmax_v w_v / noise_v with exponential noise: exponential clocks ring in the order of their rates, so v wins with w_v / sum(w), no
// running sum over the vocabulary is needed, and the answer does not hang on the order of one.  With temperature 0 a draft stands when it is
// its row's largest logit (the lowest index of equal ones), and that token follows.
//
// Both kernels are bound by memory.  The first reads every row once, in pieces of CHUNK entries a block, and leaves each piece's maximum and
// sum (or its argmax); a request's end is known only when all its rows' sums are.  The second takes, per request, the one row at which the
// request ends, the drafter's and the noise: each of its blocks first works out the request's end from the pieces (a few kilobytes out of L2),
// then looks through its chunk, and the block that comes last writes the request's answer.  A NaN counts as -infinity, +infinity as the
// largest number; a row without any finite logit has p = 0 everywhere, and its token is the lowest index.
#include <float.h>

#include "common.cuh"

namespace {
typedef __nv_bfloat16 bf16;
typedef unsigned long long Key;  // (value's bits, ~index): the largest value, of equal ones the lowest index
constexpr int THREADS = 256, STEPS = 4;
constexpr int CHUNK = THREADS * STEPS * 4;

__device__ __forceinline__ float cleaned(float v) { return v != v ? -INFINITY : fminf(v, FLT_MAX); }
__device__ __forceinline__ float rate_of(float temperature) { return fminf(1.4426950408889634f / temperature, FLT_MAX); }
// exp((v - m) / temperature): the difference first, which is exact where it matters
__device__ __forceinline__ float weight_of(float v, float m, float rate) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"((v - m) * rate));
    return y;
}
// Order-preserving for all floats but NaN.
__device__ __forceinline__ unsigned ordered(float v) {
    const unsigned b = __float_as_uint(v);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ Key key_of(float v, int index) { return ((Key)ordered(v) << 32) | (unsigned)~index; }
__device__ __forceinline__ int index_of(Key k) { return (int)~(unsigned)k; }

__device__ __forceinline__ Key warp_max_key(Key k) {
#pragma unroll
    for (int offset = 16; offset > 0; offset >>= 1) {
        const Key other = __shfl_xor_sync(0xffffffffu, k, offset);
        k = other > k ? other : k;
    }
    return k;
}
__device__ __forceinline__ Key block_max_key(Key k, Key* scratch) {  // the result stands in thread 0
    k = warp_max_key(k);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = k;
    __syncthreads();
    if (threadIdx.x == 0)
        for (int w = 1; w < THREADS / 32; ++w) k = scratch[w] > k ? scratch[w] : k;
    return k;
}

// Four entries of a row from `at` on, `fill` beyond its end.
template <typename T, bool WIDE>
__device__ __forceinline__ void entries(const T* row, int at, int vocab, float fill, float (&v)[4]) {
    if (WIDE && at + 4 <= vocab) {
        load4(row + at, v);
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = at + e < vocab ? to_float(row[at + e]) : fill;
    }
}

struct Args {
    const void* logits; long long stride;
    const int* row_start; int requests; int rows; int vocab;
    const int* drafts;
    const float* probabilities; long long q_stride;
    const float* uniform;
    const float* noise; long long noise_stride;
    const float* temperature;
    int chunks;
    float2* pieces;        // [rows, chunks]: (maximum, sum), or with temperature 0 (maximum, its index's bits)
    Key* best;             // [requests, 2]: of what is left beside the drafter's, and of the target's own
    int* arrived;          // [requests]
    int* accepted;         // [requests]
    int* tokens; int most; // [requests, most]
    int* status;
};

// The request that owns `row`: the last one whose rows start at or before it (requests without rows are passed over).
__device__ __forceinline__ int request_of(const Args& a, int row) {
    int low = 0, high = a.requests - 1;
    while (low < high) {
        const int middle = (low + high + 1) >> 1;
        if (a.row_start[middle] <= row) low = middle; else high = middle - 1;
    }
    return low;
}

template <typename T, bool WIDE>
__global__ void __launch_bounds__(THREADS) verify_rows_kernel(const Args a) {
    __shared__ Key keys[THREADS / 32];
    __shared__ __align__(16) float scratch[32];
    let_next_kernel_start();
    wait_for_previous_kernels();
    const int row = blockIdx.y, chunk = blockIdx.x;
    if (row == 0 && chunk == 0)
        for (int r = threadIdx.x; r < a.requests; r += THREADS) a.best[2 * r] = a.best[2 * r + 1] = 0, a.arrived[r] = 0;
    const T* logits = (const T*)a.logits + (size_t)row * a.stride;
    const int first = chunk * CHUNK + threadIdx.x * 4;
    float v[STEPS][4];
#pragma unroll
    for (int s = 0; s < STEPS; ++s) entries<T, WIDE>(logits, first + s * THREADS * 4, a.vocab, -INFINITY, v[s]);
    const float temperature = a.temperature[request_of(a, row)];
    float2* piece = a.pieces + (size_t)row * a.chunks + chunk;
    if (!(temperature > 0.f)) {
        Key k = 0;
#pragma unroll
        for (int s = 0; s < STEPS; ++s)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int at = first + s * THREADS * 4 + e;
                if (at >= a.vocab) continue;
                const Key mine = key_of(cleaned(v[s][e]), at);
                k = mine > k ? mine : k;
            }
        k = block_max_key(k, keys);
        if (threadIdx.x == 0) {
            const unsigned o = (unsigned)(k >> 32);
            *piece = make_float2(__uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o), __int_as_float(index_of(k)));
        }
        return;
    }
    const float rate = rate_of(temperature);
    float m = -INFINITY;
#pragma unroll
    for (int s = 0; s < STEPS; ++s)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            v[s][e] = cleaned(v[s][e]);
            m = fmaxf(m, v[s][e]);
        }
    m = block_max(m, scratch);
    float sum = 0.f;
    if (m > -INFINITY) {
#pragma unroll
        for (int s = 0; s < STEPS; ++s)
#pragma unroll
            for (int e = 0; e < 4; ++e) sum += weight_of(v[s][e], m, rate);
    }
    sum = block_sum(sum, scratch);
    if (threadIdx.x == 0) *piece = make_float2(m, sum);
}

template <typename T, bool WIDE>
__global__ void __launch_bounds__(THREADS) verify_requests_kernel(const Args a) {
    __shared__ Key keys[THREADS / 32];
    __shared__ int refused_at;            // the first draft that does not stand, counted in the request's rows
    __shared__ float end_max, end_total;  // of the row at which the request ends; with temperature 0 its largest logit's index
    __shared__ int last_block;
    let_next_kernel_start();
    const int r = blockIdx.y, chunk = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    wait_for_previous_kernels();
    const int row0 = min(max(a.row_start[r], 0), a.rows), row1 = min(max(a.row_start[r + 1], row0), a.rows), drafted = row1 - row0 - 1;
    if (drafted < 0) {  // a request without rows
        if (chunk == 0) {
            if (threadIdx.x == 0) a.accepted[r] = 0;
            for (int j = threadIdx.x; j < a.most; j += THREADS) a.tokens[(size_t)r * a.most + j] = -1;
        }
        return;
    }
    const float temperature = a.temperature[r];
    const bool greedy = !(temperature > 0.f);
    const float rate = greedy ? 0.f : rate_of(temperature);
    if (threadIdx.x == 0) refused_at = drafted;
    __syncthreads();
    // A warp takes a row: its maximum and sum from its pieces, in the order of the lanes.
    auto row_of_pieces = [&](int row, float& m, float& total) {
        const float2* pieces = a.pieces + (size_t)row * a.chunks;
        m = -INFINITY, total = 0.f;
        if (greedy) {
            Key k = 0;
            for (int c = lane; c < a.chunks; c += 32) {
                const Key mine = key_of(pieces[c].x, __float_as_int(pieces[c].y));
                k = mine > k ? mine : k;
            }
            total = __int_as_float(index_of(warp_max_key(k)));
            return;
        }
        for (int c = lane; c < a.chunks; c += 32) m = fmaxf(m, pieces[c].x);
        m = warp_max(m);
        if (m > -INFINITY)
            for (int c = lane; c < a.chunks; c += 32) total = fmaf(weight_of(pieces[c].x, m, rate), pieces[c].y, total);
        total = warp_sum(total);
    };
    for (int j = warp; j < drafted; j += THREADS / 32) {
        const int row = row0 + j, draft = a.drafts[row];
        float m, total;
        row_of_pieces(row, m, total);
        if (lane == 0) {
            bool stands = false;
            if (draft < 0 || draft >= a.vocab) {
                atomicOr(a.status, HB_STATUS_BAD_TOKEN);
            } else if (greedy) {
                stands = draft == __float_as_int(total);
            } else {
                const float p = total > 0.f ? weight_of(cleaned(to_float(((const T*)a.logits)[(size_t)row * a.stride + draft])), m, rate) / total : 0.f;
                const float q = a.probabilities ? a.probabilities[(size_t)row * a.q_stride + draft] : 1.f;
                stands = a.uniform[row] * q < p;
            }
            if (!stands) atomicMin(&refused_at, j);
        }
    }
    __syncthreads();
    const int accepted = refused_at, end = row0 + accepted;
    if (warp == 0) {
        float m, total;
        row_of_pieces(end, m, total);
        if (lane == 0) end_max = m, end_total = total;
    }
    __syncthreads();
    auto write_answer = [&](int token) {  // the whole block
        if (threadIdx.x == 0) a.accepted[r] = accepted;
        for (int j = threadIdx.x; j < a.most; j += THREADS) a.tokens[(size_t)r * a.most + j] = j < accepted ? a.drafts[row0 + j] : (j == accepted ? token : -1);
    };
    if (greedy) {
        if (chunk == 0) write_answer(__float_as_int(end_total));
        return;
    }
    const bool refused = accepted < drafted;
    const int banned = refused && !a.probabilities ? a.drafts[end] : -1;  // a draft that stood for itself takes all of its place
    const bool beside = refused && a.probabilities;
    const T* logits = (const T*)a.logits + (size_t)end * a.stride;
    const float* q = a.probabilities + (size_t)end * a.q_stride;
    const float* noise = a.noise + (size_t)r * a.noise_stride;
    const float m = end_max, share = end_total > 0.f ? 1.f / end_total : 0.f;
    const int first = chunk * CHUNK + threadIdx.x * 4;
    float v[STEPS][4], n[STEPS][4], d[STEPS][4];
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
        const int at = first + s * THREADS * 4;
        entries<T, WIDE>(logits, at, a.vocab, -INFINITY, v[s]);
        entries<float, WIDE>(noise, at, a.vocab, 1.f, n[s]);
        if (beside) entries<float, WIDE>(q, at, a.vocab, 0.f, d[s]);
        else d[s][0] = d[s][1] = d[s][2] = d[s][3] = 0.f;
    }
    Key rest = 0, left = 0;
#pragma unroll
    for (int s = 0; s < STEPS; ++s)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int at = first + s * THREADS * 4 + e;
            if (at >= a.vocab) continue;
            const float p = share > 0.f ? weight_of(cleaned(v[s][e]), m, rate) * share : 0.f, clock = 1.f / fmaxf(n[s][e], FLT_MIN);
            const Key own = key_of(p * clock, at);
            left = own > left ? own : left;
            const Key more = key_of(at == banned ? 0.f : fmaxf(p - d[s][e], 0.f) * clock, at);
            rest = more > rest ? more : rest;
        }
    rest = block_max_key(rest, keys);
    left = block_max_key(left, keys);
    if (threadIdx.x == 0) {
        atomicMax(&a.best[2 * r], rest);
        atomicMax(&a.best[2 * r + 1], left);
        __threadfence();
        last_block = atomicAdd(&a.arrived[r], 1) == (int)gridDim.x - 1;
    }
    __syncthreads();
    if (!last_block) return;
    __threadfence();
    const volatile Key* best = a.best + 2 * r;
    // where the drafter's probabilities leave nothing (rounding alone can do that), the target's own stand
    const Key winner = refused && (unsigned)(best[0] >> 32) > ordered(0.f) ? best[0] : best[1];
    write_answer(index_of(winner));
}
}  // namespace

// workspace: rows * ceil(vocab / CHUNK) + 3 * requests words of 8 bytes.
HB_EXPORT int hb_verify_drafts(const void* logits, int is_bf16, long long stride, const int* row_start, int requests, int rows, int vocab, const int* drafts,
                               const float* probabilities, long long q_stride, const float* uniform, const float* noise, long long noise_stride,
                               const float* temperature, void* workspace, int* accepted, int* tokens, int most, int* status, cudaStream_t stream) {
    if (requests <= 0) return 0;
    if (rows < 0 || vocab <= 0 || most <= 0 || !row_start || !temperature || !workspace || !accepted || !tokens || !status || ((uintptr_t)workspace & 7)) return HB_BAD_ARGUMENT;
    if (rows > 0 && (!logits || !drafts || !uniform || !noise)) return HB_BAD_ARGUMENT;
    const int chunks = (int)(((long long)vocab + CHUNK - 1) / CHUNK);
    if (rows > 65535 || requests > 65535 || vocab > 0x7fffffff - 2 * CHUNK) return HB_UNSUPPORTED_SIZE;
    float2* pieces = (float2*)workspace;
    Key* best = (Key*)(pieces + (size_t)rows * chunks);
    const Args a{logits, stride, row_start, requests, rows, vocab, drafts, probabilities, q_stride, uniform, noise, noise_stride, temperature, chunks, pieces, best,
                 (int*)(best + 2 * (size_t)requests), accepted, tokens, most, status};
    const int element = is_bf16 ? 2 : 4;
    const bool wide = !(((uintptr_t)logits | (uintptr_t)(stride * element)) & (4 * element - 1)) && !(((uintptr_t)noise | (uintptr_t)(noise_stride * 4)) & 15) &&
                      !(((uintptr_t)probabilities | (uintptr_t)(probabilities ? q_stride * 4 : 0)) & 15);
#define HB_VERIFY(T, W)                                                                                                                     \
    do {                                                                                                                                    \
        if (rows > 0)                                                                                                                       \
            if (int code = launch_after_previous(verify_rows_kernel<T, W>, dim3(chunks, rows), dim3(THREADS), 0, stream, a)) return code;   \
        return launch_after_previous(verify_requests_kernel<T, W>, dim3(chunks, requests), dim3(THREADS), 0, stream, a);                    \
    } while (0)
    if (is_bf16) {
        if (wide) HB_VERIFY(bf16, true);
        HB_VERIFY(bf16, false);
    }
    if (wide) HB_VERIFY(float, true);
    HB_VERIFY(float, false);
#undef HB_VERIFY
}
