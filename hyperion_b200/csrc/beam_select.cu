// The best continuations of a group's beams over beams and vocabulary:
//
//     score(b, v) = score_b + z_bv - log sum_u e^(z_bu)            the `take` largest of them, of equal ones the lowest (b, v)
//
// Within a row the order is that of the logits, so a row's best are found without its sum, in the one walk that makes the sum.  The first kernel reads every row once, a block a piece of it: each thread adds
// up exponentials below its own running maximum, and entries above the `take`-th best so far go into a list in shared memory, which is cut back to `take` when it grows.  In the first batch, where
// nothing is known yet, the `take`-th largest of the threads' own maxima is a bound that at least `take` entries reach.  After it few entries do: of the n-th batch about take / n.
// The second kernel has a block per group: it brings the pieces' sums together, and finds the best of the rows' best.
//
// Scores are compared as float64: a score is score_b - lse_b, a number of the row, plus the logit, and float32 would make ties of scores that are not equal.  Sums of a thread's 16 entries are float, everything above
// them float64; exponentials are the hardware's (2^-22 of a term).  Which thread adds up what goes by the entry's index alone, not by the row's alignment, so rows that hold the same have the same sums.
//
// A NaN counts as -infinity, +infinity as the largest number.  A logit of -infinity, and everything of a beam whose score is -infinity or NaN, is no candidate.  A place without a candidate has parent -1,
// token -1 and score -infinity.
#include <float.h>

#include "common.cuh"

namespace {
typedef __nv_bfloat16 bf16;
typedef unsigned long long Key;  // (value's bits, ~index): the largest value, of equal ones the lowest index; 0: none
constexpr int THREADS = 256, PER = 16, CHUNK = THREADS * PER;
constexpr int MOST_TAKE = 64;
constexpr int ROOM = CHUNK + 4 * MOST_TAKE + 256;  // of the list: a whole batch may join it

__device__ __forceinline__ float cleaned(float v) { return v != v ? -INFINITY : fminf(v, FLT_MAX); }
__device__ __forceinline__ float fast_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// Order-preserving for all floats but NaN; both zeros are the same.
__device__ __forceinline__ unsigned ordered(float v) {
    const unsigned b = __float_as_uint(v + 0.f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(unsigned o) { return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o); }
__device__ __forceinline__ Key ordered(double v) {
    const Key b = (Key)__double_as_longlong(v + 0.0);
    return b >> 63 ? ~b : b | 1ull << 63;
}
__device__ __forceinline__ double value_of(Key o) { return __longlong_as_double((long long)(o >> 63 ? o & ~(1ull << 63) : ~o)); }

// The sum over the block, in every thread.  `words` holds a word a warp.
__device__ __forceinline__ int block_count(int n, int* words) {
    n = __reduce_add_sync(0xffffffffu, n);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) words[threadIdx.x >> 5] = n;
    __syncthreads();
    int all = 0;
    for (int w = 0; w < (int)blockDim.x / 32; ++w) all += words[w];
    return all;
}

struct Args {
    const void* logits; long long stride;
    const float* scores;
    int groups, beams, vocab, take, pieces, span;  // a block has `span` entries of its row, a multiple of CHUNK
    Key* best;        // [rows, pieces, take]
    double2* sums;    // [rows, pieces]: (maximum, sum of e^(z - maximum))
    int* parents; int* tokens; float* out_scores;  // [groups, take]
};

// The list cut back to its `take` largest keys, all of which are different; what stays has no order.
__device__ int cut_back(Key* list, int n, int take, int* words, int* fill) {
    if (n <= take) return n;
    Key last = 0;  // the largest number that `take` keys reach, from its highest digit down
    for (int bit = 63; bit >= 0; --bit) {
        const Key higher = last | 1ull << bit;
        int reach = 0;
        for (int i = threadIdx.x; i < n; i += THREADS) reach += list[i] >= higher;
        if (block_count(reach, words) >= take) last = higher;
    }
    // the places below `take` that do not reach it take those behind that do
    __syncthreads();
    if (threadIdx.x == 0) *fill = 0;
    __syncthreads();
    Key kept[ROOM / THREADS + 1];
    int mine = 0;
#pragma unroll
    for (int k = 0; k < ROOM / THREADS + 1; ++k) {
        const int i = k * THREADS + threadIdx.x;
        kept[k] = i < n && list[i] >= last ? list[i] : 0;
        mine += kept[k] != 0;
    }
    __syncthreads();
    int at = mine ? atomicAdd(fill, mine) : 0;
#pragma unroll
    for (int k = 0; k < ROOM / THREADS + 1; ++k)
        if (kept[k]) list[at++] = kept[k];
    __syncthreads();
    return take;
}

template <typename T>
__device__ __forceinline__ void batch(const T* row, int first, int end, bool wide, float (&v)[PER]) {
    constexpr int AT_ONCE = 16 / sizeof(T);
    // a thread has PER / AT_ONCE runs of AT_ONCE entries, THREADS * AT_ONCE apart
#pragma unroll
    for (int s = 0; s < PER / AT_ONCE; ++s) {
        const int at = first + (s * THREADS + threadIdx.x) * AT_ONCE;
        if (wide && at + AT_ONCE <= end) {
            if constexpr (sizeof(T) == 4) {
                const float4 x = *reinterpret_cast<const float4*>(row + at);
                v[4 * s] = x.x, v[4 * s + 1] = x.y, v[4 * s + 2] = x.z, v[4 * s + 3] = x.w;
            } else {
                const uint4 x = *reinterpret_cast<const uint4*>(row + at);
                const unsigned w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) v[8 * s + 2 * i] = __uint_as_float(w[i] << 16), v[8 * s + 2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
            }
        } else {
#pragma unroll
            for (int i = 0; i < AT_ONCE; ++i) v[AT_ONCE * s + i] = at + i < end ? to_float(row[at + i]) : -INFINITY;
        }
    }
}
template <typename T>
__device__ __forceinline__ int index_of(int first, int k) {
    constexpr int AT_ONCE = 16 / sizeof(T);
    return first + (k / AT_ONCE * THREADS + threadIdx.x) * AT_ONCE + k % AT_ONCE;
}

template <typename T>
__global__ void __launch_bounds__(THREADS) beam_rows_kernel(const Args a) {
    __shared__ Key list[ROOM];
    __shared__ int words[THREADS / 32], fill, count;
    __shared__ double2 parts[THREADS / 32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, row = blockIdx.y, piece = blockIdx.x;
    let_next_kernel_start();
    wait_for_previous_kernels();
    const T* logits = reinterpret_cast<const T*>(a.logits) + (size_t)row * a.stride;
    const bool wide = ((uintptr_t)logits & 15) == 0;
    const int from = piece * a.span, end = min(a.vocab, from + a.span);
    float m = -INFINITY;  // this thread's
    double sum = 0.0;
    Key bound = 0;        // a key below it is not among the best
    if (tid == 0) count = 0;
    int n = 0;            // of the list, as all threads know it
    for (int first = from; first < end; first += CHUNK) {
        float v[PER];
        batch(logits, first, end, wide, v);
        float top = -INFINITY;
#pragma unroll
        for (int k = 0; k < PER; ++k) v[k] = cleaned(v[k]), top = fmaxf(top, v[k]);
        if (first == from) {
            // the `take`-th largest of the threads' maxima
            const unsigned mine = top == -INFINITY ? 0u : ordered(top);
            unsigned reached = 0;
            for (int bit = 31; bit >= 0; --bit) {
                const unsigned higher = reached | 1u << bit;
                if (__syncthreads_count(mine >= higher) >= a.take) reached = higher;
            }
            bound = (Key)reached << 32;
        }
        if (top != -INFINITY && ((Key)ordered(top) << 32 | 0xffffffffu) >= bound) {
#pragma unroll
            for (int k = 0; k < PER; ++k) {
                const Key key = (Key)ordered(v[k]) << 32 | (unsigned)~index_of<T>(first, k);
                if (v[k] != -INFINITY && key >= bound) list[atomicAdd(&count, 1)] = key;
            }
        }
        if (top != -INFINITY) {
            const float above = fmaxf(m, top);
            if (above > m) sum *= m == -INFINITY ? 0.0 : (double)fast_exp2((m - above) * 1.4426950408889634f);
            m = above;
            float part = 0.f;
#pragma unroll
            for (int k = 0; k < PER; ++k) part += fast_exp2((v[k] - above) * 1.4426950408889634f);
            sum += part;
        }
        __syncthreads();
        n = count;
        __syncthreads();
        if (n > ROOM - CHUNK || (n > a.take && first + CHUNK >= end) || (first == from && n >= a.take) || n > 2 * a.take + 32) {
            n = cut_back(list, n, a.take, words, &fill);
            if (n == a.take) {  // the smallest of them is the new bound
                Key smallest = ~0ull;
                for (int i = lane; i < n; i += 32) smallest = list[i] < smallest ? list[i] : smallest;
#pragma unroll
                for (int offset = 16; offset > 0; offset >>= 1) {
                    const Key other = __shfl_xor_sync(0xffffffffu, smallest, offset);
                    smallest = other < smallest ? other : smallest;
                }
                bound = smallest;
            }
            if (tid == 0) count = n;
            __syncthreads();
        }
    }
    Key* best = a.best + ((size_t)row * a.pieces + piece) * a.take;
    for (int i = tid; i < a.take; i += THREADS) best[i] = i < n ? list[i] : 0;
    // the threads' sums, below the block's maximum, in the order of the threads
    const float above = warp_max(m);
    double part = m == -INFINITY ? 0.0 : sum * (double)fast_exp2((m - above) * 1.4426950408889634f);
#pragma unroll
    for (int offset = 16; offset > 0; offset >>= 1) part += __shfl_xor_sync(0xffffffffu, part, offset);
    if (lane == 0) parts[warp] = make_double2(above, part);
    __syncthreads();
    if (tid == 0) {
        double top = -INFINITY, all = 0.0;
        for (int w = 0; w < THREADS / 32; ++w) top = fmax(top, parts[w].x);
        for (int w = 0; w < THREADS / 32; ++w) all += parts[w].x == -INFINITY ? 0.0 : parts[w].y * exp(parts[w].x - top);
        a.sums[(size_t)row * a.pieces + piece] = make_double2(top, all);
    }
}

// The second kernel: block = group.  Shared memory: the candidates' values, and the numbers of those that reach the last of the best.
constexpr int GROUP_THREADS = 512, MOST_BEAMS = 32, MOST_CANDIDATES = 12288;
__global__ void __launch_bounds__(GROUP_THREADS) beam_group_kernel(const Args a) {
    extern __shared__ Key values[];
    int* reaching = reinterpret_cast<int*>(values + a.beams * a.pieces * a.take);
    __shared__ double offset[MOST_BEAMS];
    __shared__ int words[GROUP_THREADS / 32], count;
    const int tid = threadIdx.x, group = blockIdx.x, per_row = a.pieces * a.take, n = a.beams * per_row;
    let_next_kernel_start();
    wait_for_previous_kernels();
    const Key* best = a.best + (size_t)group * n;
    if (tid < a.beams) {
        const double2* sums = a.sums + ((size_t)group * a.beams + tid) * a.pieces;
        double top = -INFINITY, all = 0.0;
        for (int p = 0; p < a.pieces; ++p) top = fmax(top, sums[p].x);
        for (int p = 0; p < a.pieces; ++p) all += sums[p].x == -INFINITY ? 0.0 : sums[p].y * exp(sums[p].x - top);
        const float score = cleaned(a.scores[group * a.beams + tid]);
        offset[tid] = score == -INFINITY || top == -INFINITY ? -INFINITY : (double)score - (top + log(all));
    }
    if (tid == 0) count = 0;
    __syncthreads();
    int there = 0;
    for (int i = tid; i < n; i += GROUP_THREADS) {
        const Key key = best[i];
        const double off = offset[i / per_row];
        const Key value = key && off != -INFINITY ? ordered((double)value_of((unsigned)(key >> 32)) + off) : 0;
        values[i] = value;
        there += value != 0;
    }
    there = block_count(there, words);
    const int take = min(a.take, there);
    Key last = 0;  // the largest number that `take` values reach
    if (there > take) {
        for (int bit = 63; bit >= 0; --bit) {
            const Key higher = last | 1ull << bit;
            int reach = 0;
            for (int i = tid; i < n; i += GROUP_THREADS) reach += values[i] >= higher;
            if (block_count(reach, words) >= take) last = higher;
        }
    }
    __syncthreads();
    // those that reach it, and their places: the number of those before them
    for (int i = tid; i < n; i += GROUP_THREADS)
        if (values[i] != 0 && values[i] >= last) reaching[atomicAdd(&count, 1)] = i;
    __syncthreads();
    auto place_of = [&](int i) { return ((long long)(i / per_row) << 32) | (unsigned)~(unsigned)best[i]; };  // (beam, token)
    for (int k = tid; k < count; k += GROUP_THREADS) {
        const int i = reaching[k];
        const Key value = values[i];
        const long long place = place_of(i);
        int before = 0;
        for (int c = 0; c < count; ++c) {
            const int j = reaching[c];
            const Key other = values[j];
            before += other > value || (other == value && j != i && place_of(j) < place);
        }
        if (before < take) {
            const size_t at = (size_t)group * a.take + before;
            a.parents[at] = i / per_row, a.tokens[at] = (int)(unsigned)place, a.out_scores[at] = (float)value_of(value);
        }
    }
    for (int i = take + tid; i < a.take; i += GROUP_THREADS) {
        const size_t at = (size_t)group * a.take + i;
        a.parents[at] = -1, a.tokens[at] = -1, a.out_scores[at] = -INFINITY;
    }
}
}  // namespace

// Into how many pieces rows are cut: what fills the device, four blocks a multiprocessor, and no more candidates of a group than the second kernel holds.
static int pieces_for(int groups, int beams, int vocab, int take, int sms) {
    const long long chunks = (vocab + CHUNK - 1) / CHUNK, room = 4LL * sms / ((long long)groups * beams), most = MOST_CANDIDATES / ((long long)beams * take);
    long long n = room < 1 ? 1 : room;
    n = n < chunks ? n : chunks;
    n = n < most ? n : most;
    const long long span = (chunks + n - 1) / n;
    return (int)((chunks + span - 1) / span);
}
// Bytes of scratch that hb_beam_select takes.
HB_EXPORT long long hb_beam_select_scratch(int groups, int beams, int vocab, int take, int sms) {
    if (groups <= 0 || beams <= 0 || beams > MOST_BEAMS || vocab <= 0 || take <= 0 || take > MOST_TAKE || sms <= 0) return 0;
    return (long long)groups * beams * pieces_for(groups, beams, vocab, take, sms) * (16 + 8 * take);
}
// logits [groups * beams, vocab] (bfloat16 or float) with rows `stride` apart; scores [groups, beams]; parents, tokens, out_scores [groups, take].  scratch: hb_beam_select_scratch bytes on a
// 16-byte boundary.
HB_EXPORT int hb_beam_select(const void* logits, int is_bf16, long long stride, const float* scores, int groups, int beams, int vocab, int take, int* parents, int* tokens, float* out_scores, int sms,
                             void* scratch, cudaStream_t stream) {
    if (groups <= 0) return 0;
    if (!logits || !scores || !parents || !tokens || !out_scores || !scratch || beams <= 0 || vocab <= 0 || take <= 0 || sms <= 0 || stride < vocab || ((uintptr_t)scratch & 15)) return HB_BAD_ARGUMENT;
    if (beams > MOST_BEAMS || take > MOST_TAKE || (long long)groups * beams > 65535 || vocab > 0x7fffffff - 2 * CHUNK) return HB_UNSUPPORTED_SIZE;
    const int pieces = pieces_for(groups, beams, vocab, take, sms), chunks = (vocab + CHUNK - 1) / CHUNK;
    const size_t rows = (size_t)groups * beams;
    double2* sums = (double2*)scratch;
    const Args a{logits, stride, scores, groups, beams, vocab, take, pieces, (chunks + pieces - 1) / pieces * CHUNK, (Key*)(sums + rows * pieces), sums, parents, tokens, out_scores};
    if (int code = launch_after_previous(is_bf16 ? beam_rows_kernel<bf16> : beam_rows_kernel<float>, dim3(pieces, (unsigned)rows), dim3(THREADS), 0, stream, a)) return code;
    const size_t shared = (size_t)beams * pieces * take * 12;
    const cudaError_t configured = cudaFuncSetAttribute(beam_group_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, MOST_CANDIDATES * 12);
    if (configured != cudaSuccess) return (int)configured;
    return launch_after_previous(beam_group_kernel, dim3(groups), dim3(GROUP_THREADS), shared, stream, a);
}
