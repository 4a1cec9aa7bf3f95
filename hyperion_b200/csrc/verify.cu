// Drafted tokens against the target model's logits, from given random numbers (speculative sampling).
//
// A request brings n drafted tokens and n + 1 rows of logits.  With p_i = softmax(row i / temperature) and q_i the drafter's probabilities
// (a token that stands for itself where there are none: q_i = 1 there), draft x_i stands when u_i q_i(x_i) < p_i(x_i).  The first one that
// does not is replaced by a draw from max(p_i - q_i, 0), normalised; when all stand, one more token is drawn from p_n.  A draw from weights w
// is argmax_v w_v / noise_v with exponential noise: exponential clocks ring in the order of their rates, so v wins with w_v / sum(w), no
// running sum over the vocabulary is needed, and the answer does not hang on the order of one.  With temperature 0 a draft stands when it is
// its row's largest logit (the lowest index of equal ones), and that token follows.
//
// The first kernel reads every row once, a block a piece of it, and leaves each piece's maximum and sum (or its argmax); a request's end is
// known only when all its rows' sums are.  The second takes, per request, the one row at which the request ends, the drafter's and the noise: each of its blocks first works
// out the request's end from the pieces (a few kilobytes out of L2, with the noise on its way meanwhile), then looks through its part, and the block that comes last
// writes the request's answer.  Pieces are as many as the device holds blocks at once: a block's start (which request is this, what is its temperature; where does it
// end) costs as much as some 20,000 entries.  Both keep the batches to come on their way while they look at the one at hand, some 64 KB an SM.  64 requests of up to six
// bfloat16 rows of 152,064 logits, with the drafter's probabilities: 41 us for 165 MB, 4.0 TB/s (one batch of 8 KB ahead in the first kernel and none in the second: 47 us).  Alone the two run at 3.2 and 3.1 TB/s
// with issue slots at 45 and 28 %: neither memory nor instructions bound them, but the trips of the batches on their way, and the starts.  One
// request of five float rows: 9.4 us, two kernels' starts and a few trips to memory.  Exponentials and reciprocals are the hardware's (2^-22 of a weight), sums float.  A NaN counts as -infinity, +infinity as the largest number; a row without any finite logit has p = 0 everywhere, and its
// token is the lowest index.
#include <float.h>

#include "common.cuh"

namespace {
typedef __nv_bfloat16 bf16;
typedef unsigned long long Key;  // (value's bits, ~index): the largest value, of equal ones the lowest index
constexpr int THREADS = 256, STEPS = 4;
constexpr int CHUNK = THREADS * STEPS * 4;  // entries a block holds at a time
constexpr int ROWS_PER_SM = 4, REQUESTS_PER_SM = 2;  // blocks, by registers
template <typename T>
constexpr int AHEAD = sizeof(T) == 2 ? 2 : 1;  // batches of a row on their way beside the one at hand: some 64 KB an SM
constexpr int KEPT = 64;                    // rows of a request whose sums a block keeps

__device__ __forceinline__ float cleaned(float v) { return v != v ? -INFINITY : fminf(v, FLT_MAX); }
// Above 0, too, so that a logit of -infinity has weight 0 at an infinite temperature.
__device__ __forceinline__ float rate_of(float temperature) { return fminf(fmaxf(1.4426950408889634f / temperature, FLT_MIN), FLT_MAX); }
__device__ __forceinline__ float fast_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float fast_reciprocal(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// exp((v - m) / temperature)
__device__ __forceinline__ float weight_of(float v, float m, float rate) { return fast_exp2((v - m) * rate); }
// The same for the many entries of a batch, in one multiplication and addition each: 2^(v * rate + offset) * rest with offset = -m * rate.  The offset's rounding is an absolute error of the
// exponent, which grows with |m| / temperature; what it has been rounded by is itself a float, which one fused multiplication and addition gives, and 2^ that is the rest.
// `exact`: the rest is between 2^-0.5 and 2^0.5; where it is not (or not finite), entries take weight_of.
struct Offset {
    float offset, rest;
    bool exact;
    __device__ __forceinline__ Offset(float m, float rate) : offset(-m * rate), rest(fast_exp2(-fmaf(m, rate, offset))), exact(fabsf(offset) < 0x1p24f) {}
};
__device__ __forceinline__ float max3(float a, float b, float c) {  // passes over a NaN, as fmaxf does
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
// Order-preserving for all floats but NaN; both zeros are the same.
__device__ __forceinline__ unsigned ordered(float v) {
    const unsigned b = __float_as_uint(v + 0.f);
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

// Four entries of a row as they stand in memory: nothing waits for them before they are used.
template <typename T>
struct Four;
template <>
struct Four<float> {
    float4 raw;
    __device__ __forceinline__ float operator[](int e) const { return e == 0 ? raw.x : e == 1 ? raw.y : e == 2 ? raw.z : raw.w; }
    __device__ __forceinline__ void set(int e, float v) { (e == 0 ? raw.x : e == 1 ? raw.y : e == 2 ? raw.z : raw.w) = v; }
};
template <>
struct Four<bf16> {
    uint2 raw;
    __device__ __forceinline__ float operator[](int e) const {
        const unsigned w = e < 2 ? raw.x : raw.y;
        return __uint_as_float(e & 1 ? w & 0xffff0000u : w << 16);
    }
    __device__ __forceinline__ void set(int e, bf16 v) {
        unsigned& w = e < 2 ? raw.x : raw.y;
        w = e & 1 ? (w & 0xffffu) | (unsigned)__bfloat16_as_ushort(v) << 16 : (w & 0xffff0000u) | __bfloat16_as_ushort(v);
    }
};
// A thread's part of CHUNK entries of a row, its first at `first`; what lies at `end` and beyond is not read, and is not to be looked at.
template <typename T, bool WIDE>
__device__ __forceinline__ void batch(const T* row, int first, int end, Four<T> (&v)[STEPS]) {
    if (WIDE && first - (int)threadIdx.x * 4 + CHUNK <= end) {  // for the whole block
#pragma unroll
        for (int s = 0; s < STEPS; ++s) v[s].raw = *reinterpret_cast<const decltype(v[s].raw)*>(row + first + s * THREADS * 4);
    } else {
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            const int at = first + s * THREADS * 4;
            v[s] = {};
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (at + e < end) v[s].set(e, row[at + e]);
        }
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
    int pieces_per_row, row_span, request_span;  // a block of the first kernel, and of the second, has so many entries of its row (a multiple of CHUNK)
    float2* pieces;        // [rows, pieces_per_row]: (maximum, sum), or with temperature 0 (maximum, its index's bits)
    Key* best;             // [requests]
    int* arrived;          // [requests]
    int* accepted;         // [requests]
    int* tokens; int most; // [requests, most]
    int* status;
};

template <typename T, bool WIDE>
__global__ void __launch_bounds__(THREADS, ROWS_PER_SM) verify_rows_kernel(const Args a) {
    __shared__ Key keys[THREADS / 32];
    __shared__ float2 parts[THREADS / 32];
    __shared__ int owner;
    wait_for_previous_kernels();
    let_next_kernel_start();  // only now: the kernel behind takes its start as the sign that all that came before this one has finished
    const int row = blockIdx.y, piece = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (row == 0 && piece == 0)
        for (int r = threadIdx.x; r < a.requests; r += THREADS) a.best[r] = 0, a.arrived[r] = 0;
    const T* logits = (const T*)a.logits + (size_t)row * a.stride;
    const int end = min(a.vocab, (piece + 1) * a.row_span);
    int first = piece * a.row_span + threadIdx.x * 4;
    constexpr int BUFFERS = AHEAD<T> + 1;
    Four<T> buffer[BUFFERS][STEPS];
#pragma unroll
    for (int d = 0; d < AHEAD<T>; ++d) batch<T, WIDE>(logits, first + d * CHUNK, end, buffer[d]);
    // The row's batches one after the other, each buffer filled again as soon as it has been looked at.
    auto walk = [&](auto&& look) {
        while (true) {
#pragma unroll
            for (int k = 0; k < BUFFERS; ++k) {
                const int at = first - (int)threadIdx.x * 4;  // the block's
                if (at + AHEAD<T> * CHUNK < end) batch<T, WIDE>(logits, first + AHEAD<T> * CHUNK, end, buffer[(k + AHEAD<T>) % BUFFERS]);
                look(buffer[k]);
                if (at + CHUNK >= end) return;
                first += CHUNK;
            }
        }
    };
    // The request that owns the row; a row that is no one's is treated as greedy, and never looked at.
    if (threadIdx.x == 0) owner = -1;
    __syncthreads();
    for (int r = threadIdx.x; r < a.requests; r += THREADS)
        if (a.row_start[r] <= row && row < a.row_start[r + 1]) owner = r;
    __syncthreads();
    const float temperature = owner < 0 ? 0.f : a.temperature[owner];
    float2* out = a.pieces + (size_t)row * a.pieces_per_row + piece;
    if (!(temperature > 0.f)) {
        Key k = 0;
        walk([&](const Four<T>(&v)[STEPS]) {
#pragma unroll
            for (int s = 0; s < STEPS; ++s)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int at = first + s * THREADS * 4 + e;
                    if (at >= end) continue;
                    const Key mine = key_of(cleaned(v[s][e]), at);
                    k = mine > k ? mine : k;
                }
        });
        k = block_max_key(k, keys);
        if (threadIdx.x == 0) {
            const unsigned o = (unsigned)(k >> 32);
            *out = make_float2(__uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o), __int_as_float(index_of(k)));
        }
        return;
    }
    const float rate = rate_of(temperature);
    float m = -INFINITY, sum = 0.f;
    walk([&](const Four<T>(&v)[STEPS]) {
        float z[STEPS][4], top = m;
#pragma unroll
        for (int s = 0; s < STEPS; ++s)
#pragma unroll
            for (int e = 0; e < 4; ++e) z[s][e] = v[s][e];
        if (first - (int)threadIdx.x * 4 + CHUNK > end) {
#pragma unroll
            for (int s = 0; s < STEPS; ++s)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (first + s * THREADS * 4 + e >= end) z[s][e] = -INFINITY;
        }
#pragma unroll
        for (int s = 0; s < STEPS; ++s) top = max3(max3(top, z[s][0], z[s][1]), z[s][2], z[s][3]);
        top = fminf(top, FLT_MAX);
        if (top > -INFINITY) {
            // A sum that a NaN or an infinity has got into is made again with those put right.
            const Offset from(top, rate);
            float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int s = 0; s < STEPS; ++s)
#pragma unroll
                for (int e = 0; e < 4; ++e) part[e] += fast_exp2(fmaf(z[s][e], rate, from.offset));
            float more_sum = ((part[0] + part[1]) + (part[2] + part[3])) * from.rest;
            if (!(from.exact && more_sum < INFINITY)) {
                more_sum = 0.f;
#pragma unroll
                for (int s = 0; s < STEPS; ++s)
#pragma unroll
                    for (int e = 0; e < 4; ++e) more_sum += weight_of(cleaned(z[s][e]), top, rate);
            }
            sum = fmaf(sum, m == -INFINITY ? 0.f : weight_of(m, top, rate), more_sum);
            m = top;
        }
    });
    float top = warp_max(m);
    sum = warp_sum(m == -INFINITY ? 0.f : sum * weight_of(m, top, rate));
    if (lane == 0) parts[warp] = make_float2(top, sum);
    __syncthreads();
    if (warp == 0) {
        const float2 part = lane < THREADS / 32 ? parts[lane] : make_float2(-INFINITY, 0.f);
        top = warp_max(part.x);
        sum = warp_sum(part.x == -INFINITY ? 0.f : part.y * weight_of(part.x, top, rate));
        if (lane == 0) *out = make_float2(top, sum);
    }
}

template <typename T, bool WIDE>
__global__ void __launch_bounds__(THREADS, REQUESTS_PER_SM) verify_requests_kernel(const Args a) {
    __shared__ Key keys[THREADS / 32];
    __shared__ float2 sums[KEPT];         // a row's maximum and sum; with temperature 0 the index of its largest logit in the latter's place
    __shared__ int refused_at;            // the first draft that does not stand, counted in the request's rows
    __shared__ int last_block;
    let_next_kernel_start();
    const int r = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (!a.rows) wait_for_previous_kernels();  // else the kernel above is the one before, which lets this one start when all but itself has finished: the inputs may be read
    const int end_at = min(a.vocab, ((int)blockIdx.x + 1) * a.request_span);
    int first = blockIdx.x * a.request_span + threadIdx.x * 4;
    const float* noise = a.noise + (size_t)r * a.noise_stride;
    struct Batch { Four<T> v[STEPS]; Four<float> d[STEPS], n[STEPS]; } buffer[2];
    batch<float, WIDE>(noise, first, end_at, buffer[0].n);
    if (a.rows) wait_for_previous_kernels();
    const int row0 = min(max(a.row_start[r], 0), a.rows), row1 = min(max(a.row_start[r + 1], row0), a.rows), drafted = row1 - row0 - 1;
    const float temperature = a.temperature[r];
    if (drafted < 0) {  // a request without rows
        if (blockIdx.x == 0) {
            if (threadIdx.x == 0) a.accepted[r] = 0;
            for (int j = threadIdx.x; j < a.most; j += THREADS) a.tokens[(size_t)r * a.most + j] = -1;
        }
        return;
    }
    const bool greedy = !(temperature > 0.f);
    const float rate = greedy ? 0.f : rate_of(temperature);
    if (threadIdx.x == 0) refused_at = drafted;
    __syncthreads();
    // A warp takes a row: its maximum and sum from its pieces, in the order of the lanes.
    auto row_of_pieces = [&](int row) {
        const float2* pieces = a.pieces + (size_t)row * a.pieces_per_row;
        if (greedy) {
            Key k = 0;
            for (int c = lane; c < a.pieces_per_row; c += 32) {
                const float2 piece = pieces[c];
                const Key mine = key_of(piece.x, __float_as_int(piece.y));
                k = mine > k ? mine : k;
            }
            return make_float2(0.f, __int_as_float(index_of(warp_max_key(k))));
        }
        float m = -INFINITY, total = 0.f;
        for (int c = lane; c < a.pieces_per_row; c += 32) m = fmaxf(m, pieces[c].x);
        m = warp_max(m);
        if (m > -INFINITY)
            for (int c = lane; c < a.pieces_per_row; c += 32) total = fmaf(weight_of(pieces[c].x, m, rate), pieces[c].y, total);
        return make_float2(m, warp_sum(total));
    };
    for (int j = warp; j <= drafted; j += THREADS / 32) {
        const int row = row0 + j, draft = j < drafted ? a.drafts[row] : 0;
        const bool known = draft >= 0 && draft < a.vocab;
        float logit = 0.f, q = 1.f, u = 0.f;
        if (lane == 0 && j < drafted && known && !greedy) {
            logit = to_float(((const T*)a.logits)[(size_t)row * a.stride + draft]);
            if (a.probabilities) q = a.probabilities[(size_t)row * a.q_stride + draft];
            u = a.uniform[row];
        }
        const float2 sum = row_of_pieces(row);
        if (lane == 0) {
            if (j < KEPT) sums[j] = sum;
            if (j < drafted) {
                bool stands;
                if (!known) {
                    atomicOr(a.status, HB_STATUS_BAD_TOKEN);
                    stands = false;
                } else if (greedy) {
                    stands = draft == __float_as_int(sum.y);
                } else {
                    const float p = sum.y > 0.f ? weight_of(cleaned(logit), sum.x, rate) / sum.y : 0.f;
                    stands = u * q < p;
                }
                if (!stands) atomicMin(&refused_at, j);
            }
        }
    }
    __syncthreads();
    const int accepted = refused_at, end = row0 + accepted;
    if (accepted >= KEPT) {
        if (warp == 0) {
            const float2 sum = row_of_pieces(end);
            if (lane == 0) sums[0] = sum;
        }
        __syncthreads();
    }
    const float2 sum = sums[accepted < KEPT ? accepted : 0];
    auto write_answer = [&](int token) {  // the whole block
        if (threadIdx.x == 0) a.accepted[r] = accepted;
        for (int j = threadIdx.x; j < a.most; j += THREADS) a.tokens[(size_t)r * a.most + j] = j < accepted ? a.drafts[row0 + j] : (j == accepted ? token : -1);
    };
    if (greedy) {
        if (blockIdx.x == 0) write_answer(__float_as_int(sum.y));
        return;
    }
    const bool refused = accepted < drafted;
    const int banned = refused && !a.probabilities ? a.drafts[end] : -1;  // a draft that stood for itself takes all of its place
    const bool beside = refused && a.probabilities;
    const T* logits = (const T*)a.logits + (size_t)end * a.stride;
    const float* probabilities = a.probabilities + (size_t)end * a.q_stride;
    const float m = sum.x, share = sum.y > 0.f ? 1.f / sum.y : 0.f;
    // Looks through entries from `first` on to `end_at`, `step` apart: the best of the target's probabilities (`own`), or of what is left of them beside the drafter's.
    auto look = [&](int first, int end_at, int step, bool own) {
        Key best_key = 0;
        float best = -1.f;
        const Offset from(m, rate);
        const float scaled_share = share * from.rest;
        const bool clean = share > 0.f && m < FLT_MAX && from.exact;
        const auto fetch = [&](Batch& b, int at) {  // all but the noise
            batch<T, WIDE>(logits, at, end_at, b.v);
            if (beside && !own) {
                batch<float, WIDE>(probabilities, at, end_at, b.d);
            } else {
#pragma unroll
                for (int s = 0; s < STEPS; ++s) b.d[s].raw = make_float4(0.f, 0.f, 0.f, 0.f);
            }
        };
        const auto weigh = [&](const Batch& b) {
            const Four<T>(&v)[STEPS] = b.v;
            const Four<float>(&d)[STEPS] = b.d, (&n)[STEPS] = b.n;
            float z[STEPS][4], top = -1.f;
            if (clean) {
#pragma unroll
                for (int s = 0; s < STEPS; ++s)
#pragma unroll
                    for (int e = 0; e < 4; ++e) z[s][e] = fast_exp2(fmaf(v[s][e], rate, from.offset)) * scaled_share;
            } else {  // the row's largest logit is infinite, or too far from zero for the temperature, or there is none
#pragma unroll
                for (int s = 0; s < STEPS; ++s)
#pragma unroll
                    for (int e = 0; e < 4; ++e) z[s][e] = share > 0.f ? weight_of(cleaned(v[s][e]), m, rate) * share : 0.f;
            }
#pragma unroll
            for (int s = 0; s < STEPS; ++s) {
#pragma unroll
                for (int e = 0; e < 4; ++e) z[s][e] = fmaxf(z[s][e] - d[s][e], 0.f) * fast_reciprocal(fmaxf(n[s][e], FLT_MIN));  // a NaN, too, comes to 0
                const int at = first + s * THREADS * 4;
                if (!own && banned >= at && banned < at + 4) {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (banned == at + e) z[s][e] = 0.f;
                }
                if (at + 4 > end_at) {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (at + e >= end_at) z[s][e] = -1.f;
                }
                top = max3(max3(top, z[s][0], z[s][1]), z[s][2], z[s][3]);
            }
            if (top > best) {  // seldom, once a few batches have been looked at: where does it stand?
                best = top;
                int at = 0;
#pragma unroll
                for (int s = STEPS - 1; s >= 0; --s)
#pragma unroll
                    for (int e = 3; e >= 0; --e)
                        if (z[s][e] == top) at = first + s * THREADS * 4 + e;
                best_key = key_of(best, at);
            }
        };
        fetch(buffer[0], first);
        for (bool more = true; more;) {
#pragma unroll
            for (int k = 0; k < 2 && more; ++k) {
                more = first - (int)threadIdx.x * 4 + step < end_at;
                if (more) batch<float, WIDE>(noise, first + step, end_at, buffer[1 - k].n), fetch(buffer[1 - k], first + step);
                weigh(buffer[k]);
                first += step;
            }
        }
        return block_max_key(best_key, keys);
    };
    const Key found = look(first, end_at, CHUNK, !refused);
    if (threadIdx.x == 0) {
        atomicMax(&a.best[r], found);
        __threadfence();
        last_block = atomicAdd(&a.arrived[r], 1) == (int)gridDim.x - 1;
    }
    __syncthreads();
    if (!last_block) return;
    __threadfence();
    Key winner = *const_cast<const volatile Key*>(a.best + r);
    if (refused && (unsigned)(winner >> 32) <= ordered(0.f)) {  // nothing is left beside the drafter's (rounding alone can do that): the target's own probabilities stand
        batch<float, WIDE>(noise, (int)threadIdx.x * 4, a.vocab, buffer[0].n);
        winner = look((int)threadIdx.x * 4, a.vocab, CHUNK, true);
        if (threadIdx.x == 0) keys[0] = winner;
        __syncthreads();
        winner = keys[0];
    }
    write_answer(index_of(winner));
}
}  // namespace

// workspace: rows * ceil(vocab / CHUNK) + 2 * requests words of 8 bytes.  sms: the device's multiprocessors.
HB_EXPORT int hb_verify_drafts(const void* logits, int is_bf16, long long stride, const int* row_start, int requests, int rows, int vocab, const int* drafts,
                               const float* probabilities, long long q_stride, const float* uniform, const float* noise, long long noise_stride,
                               const float* temperature, void* workspace, int* accepted, int* tokens, int most, int sms, int* status, cudaStream_t stream) {
    if (requests <= 0) return 0;
    if (rows < 0 || vocab <= 0 || most <= 0 || sms <= 0 || !row_start || !noise || !temperature || !workspace || !accepted || !tokens || !status || ((uintptr_t)workspace & 7)) return HB_BAD_ARGUMENT;
    if (rows > 0 && (!logits || !drafts || !uniform)) return HB_BAD_ARGUMENT;
    if (rows > 65535 || requests > 65535 || vocab > 0x7fffffff - 2 * CHUNK) return HB_UNSUPPORTED_SIZE;
    // As many blocks a row, and then a request, as the device holds at once between them, one for each CHUNK at most: a second turn of a few blocks would cost as much as
    // the first.
    const int chunks = (vocab + CHUNK - 1) / CHUNK;
    const auto span = [&](int lines, int slots) {
        const int wanted = slots / (lines > 0 ? lines : 1), blocks = wanted < 1 ? 1 : (wanted < chunks ? wanted : chunks);
        return (chunks + blocks - 1) / blocks * CHUNK;
    };
    const int row_span = span(rows, sms * ROWS_PER_SM), request_span = span(requests, sms * REQUESTS_PER_SM);
    const int row_blocks = (vocab + row_span - 1) / row_span, request_blocks = (vocab + request_span - 1) / request_span;
    float2* pieces = (float2*)workspace;
    Key* best = (Key*)(pieces + (size_t)rows * chunks);
    const Args a{logits, stride, row_start, requests, rows, vocab, drafts, probabilities, q_stride, uniform, noise, noise_stride, temperature, row_blocks, row_span, request_span,
                 pieces, best, (int*)(best + requests), accepted, tokens, most, status};
    const int element = is_bf16 ? 2 : 4;
    const bool wide = !(((uintptr_t)logits | (uintptr_t)(stride * element)) & (4 * element - 1)) && !(((uintptr_t)noise | (uintptr_t)(noise_stride * 4)) & 15) &&
                      !(((uintptr_t)probabilities | (uintptr_t)(probabilities ? q_stride * 4 : 0)) & 15);
#define HB_VERIFY(T, W)                                                                                                                     \
    do {                                                                                                                                    \
        if (rows > 0)                                                                                                                       \
            if (int code = launch_after_previous(verify_rows_kernel<T, W>, dim3(row_blocks, rows), dim3(THREADS), 0, stream, a)) return code;   \
        return launch_after_previous(verify_requests_kernel<T, W>, dim3(request_blocks, requests), dim3(THREADS), 0, stream, a);                    \
    } while (0)
    if (is_bf16) {
        if (wide) HB_VERIFY(bf16, true);
        HB_VERIFY(bf16, false);
    }
    if (wide) HB_VERIFY(float, true);
    HB_VERIFY(float, false);
#undef HB_VERIFY
}
