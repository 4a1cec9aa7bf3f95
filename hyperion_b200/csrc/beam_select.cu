// The best continuations of a group's beams over beams and vocabulary:
//
//     score(b, v) = score_b + z_bv - log sum_u e^(z_bu)            the `take` largest of them, of equal ones the lowest (b, v)
//
// The first kernel reads every row once and leaves the sum, and the maximum of every run of 256 logits.  The second has a block per group: with the rows' sums it knows every run's best score.  The runs whose best
// are the `take` best of all runs hold the `take` best continuations (of a run that is not among them, `take` others hold something better), so only those are read again: a few KB of them.  Both
// searches take a bound first and then look at what reaches it.  For the runs it is the `take`-th largest of what each 128th of the threads has found to be its best; where that lets many more through than are taken
// (a search's first step has one beam), it is found bit by bit among all threads.  That is little more than `take` in all but contrived rows, for which there is a way that goes by one continuation after the other.
//
// Measured: 32 groups of 8 beams over bfloat16 logits of 152,064 26.5 us for 78 MB: the first kernel 17 (4.6 TB/s; as long without its exponentials, and with more or fewer blocks or loads on their way), the second 9, a chain of a
// logarithm, three meetings of the block and two trips to memory.  Over 157,831, rows of every alignment, 28.9.  One group of four beams 8.3 us.  A first step, 32 beams of which one is alive, 64 taken: 23 (by one continuation after
// the other 985).
//
// Scores are compared as float64: a score is score_b - lse_b, a number of the row, plus the logit, and float32 would make ties of scores that are not equal.  Sums of a thread's 32 entries are float, everything above
// them float64; exponentials are the hardware's (2^-22 of a term), of differences rounded to float.  A row's sum is off by (2.224 D + 4 R + 31) 2^-24 of itself at most, where D, at most ln vocab, is how far below the maximum its
// terms lie on average and R how often a thread's maximum rises behind a term: scores of two beams may come in either order where they are closer than two such errors (measured 2^-20.8 for one outlier over equal logits, 2^-23 else).
// Which thread adds up what goes by the entry's index alone, not by the row's alignment, so rows of a call that hold the same have the same sums.
//
// A NaN counts as -infinity, +infinity as the largest number.  A logit of -infinity, and everything of a beam whose score is -infinity or NaN, is no candidate.  A place without a candidate has parent -1,
// token -1 and score -infinity.
#include <float.h>

#include <type_traits>

#include "common.cuh"

namespace {
typedef __nv_bfloat16 bf16;
typedef unsigned long long Key;  // a float64's bits in its order; 0: none
constexpr int THREADS = 256, WARPS = THREADS / 32, RUN = 256, PER = RUN / 32, MOST_AT_ONCE = 4;  // a warp looks at several runs at a time, PER entries a lane of each
constexpr int MOST_TAKE = 64, MOST_BEAMS = 32;
constexpr float LOG2E = 1.4426950408889634f;

__device__ __forceinline__ float cleaned(float v) { return v != v ? -INFINITY : fminf(v, FLT_MAX); }
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
__device__ __forceinline__ float warp_largest(float v) {
    float d;
    asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(d) : "f"(v));
    return d;
}
// Order-preserving for all numbers; both zeros are the same.
__device__ __forceinline__ Key ordered(double v) {
    const Key b = (Key)__double_as_longlong(v + 0.0);
    return b >> 63 ? ~b : b | 1ull << 63;
}
__device__ __forceinline__ double value_of(Key o) { return __longlong_as_double((long long)(o >> 63 ? o & ~(1ull << 63) : ~o)); }

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

struct Args {
    const void* logits; long long stride;
    const float* scores;
    int groups, beams, vocab, take, runs, pieces, piece_runs;  // runs of a row; blocks of a row, and runs of each
    float* tops;      // [rows, runs]
    double2* sums;    // [rows, pieces]: (maximum, sum of e^(z - maximum))
    int* parents; int* tokens; float* out_scores;  // [groups, take]
};

// A lane's eight entries of the run that begins at `first`: bfloat16 [8 lane, 8 lane + 8), float [4 lane, 4 lane + 4) and 128 further on.  Where rows begin K words and, ODD, half a word behind a boundary of 16 bytes, they are
// fetched by the widest loads that the boundaries allow, and the row's halves of words put together.  (256 rows of 157,831 bfloat16, us: 28.9; by 16 bytes from the boundary before, shifted, one run after the other, 40.8.)
struct Words { uint4 lo, hi; };
template <int K, int N>
__device__ __forceinline__ void load_words(const unsigned* p, unsigned (&w)[N]) {  // p is K words behind a boundary
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int at = (K + i) & 3;  // behind the boundary before
        if (i >= at && i - at + 4 <= N) {
            if (at) continue;
            const uint4 v = *reinterpret_cast<const uint4*>(p + i);
            w[i] = v.x, w[i + 1] = v.y, w[i + 2] = v.z, w[i + 3] = v.w;
        } else if (at & 1 ? i > 0 : i + 1 < N) {
            if (at & 1) continue;
            const uint2 v = *reinterpret_cast<const uint2*>(p + i);
            w[i] = v.x, w[i + 1] = v.y;
        } else {
            w[i] = p[i];
        }
    }
}
template <typename T, int AT_ONCE, int K, bool ODD>
__device__ __forceinline__ void load_runs(const T* row, const int (&first)[AT_ONCE], int lane, Words (&w)[AT_ONCE]) {
    if constexpr (sizeof(T) == 2) {
        constexpr int N = ODD ? 5 : 4;  // a row's first and last word may have a half that is not the row's: it is fetched with the other one, and shifted out
        unsigned x[AT_ONCE][N];
#pragma unroll
        for (int u = 0; u < AT_ONCE; ++u) load_words<K, N>(reinterpret_cast<const unsigned*>(row + (first[u] + 8 * lane - (ODD ? 1 : 0))), x[u]);
#pragma unroll
        for (int u = 0; u < AT_ONCE; ++u)
            w[u].lo = ODD ? make_uint4(__funnelshift_r(x[u][0], x[u][1], 16), __funnelshift_r(x[u][1], x[u][2], 16), __funnelshift_r(x[u][2], x[u][3], 16), __funnelshift_r(x[u][3], x[u][N - 1], 16))
                          : make_uint4(x[u][0], x[u][1], x[u][2], x[u][3]);
    } else if constexpr (!ODD) {
        unsigned x[AT_ONCE][2][4];
#pragma unroll
        for (int u = 0; u < AT_ONCE; ++u)
#pragma unroll
            for (int h = 0; h < 2; ++h) load_words<K, 4>(reinterpret_cast<const unsigned*>(row + (first[u] + 4 * lane + 128 * h)), x[u][h]);
#pragma unroll
        for (int u = 0; u < AT_ONCE; ++u) w[u] = {make_uint4(x[u][0][0], x[u][0][1], x[u][0][2], x[u][0][3]), make_uint4(x[u][1][0], x[u][1][1], x[u][1][2], x[u][1][3])};
    }
}
template <typename T>
__device__ __forceinline__ Words nothing() {  // eight entries of -infinity
    const unsigned x = sizeof(T) == 2 ? 0xff80ff80u : 0xff800000u;
    return {make_uint4(x, x, x, x), make_uint4(x, x, x, x)};
}
template <typename T>
__device__ __forceinline__ Words one_by_one(const T* row, int first, int end, int lane) {
    Words w;
    if constexpr (sizeof(T) == 2) {
        const int at = first + 8 * lane;
        unsigned short h[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) h[i] = at + i < end ? __bfloat16_as_ushort(reinterpret_cast<const bf16*>(row)[at + i]) : 0xff80;
        w.lo = make_uint4(h[0] | (unsigned)h[1] << 16, h[2] | (unsigned)h[3] << 16, h[4] | (unsigned)h[5] << 16, h[6] | (unsigned)h[7] << 16);
    } else {
        const int at = first + 4 * lane;
        unsigned x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int k = at + (i & 3) + (i >> 2) * 128;
            x[i] = k < end ? reinterpret_cast<const unsigned*>(row)[k] : 0xff800000u;
        }
        w.lo = make_uint4(x[0], x[1], x[2], x[3]), w.hi = make_uint4(x[4], x[5], x[6], x[7]);
    }
    return w;
}
template <typename T>
__device__ __forceinline__ void unpack(const Words& w, float (&v)[PER]) {
    const unsigned a[4] = {w.lo.x, w.lo.y, w.lo.z, w.lo.w}, b[4] = {w.hi.x, w.hi.y, w.hi.z, w.hi.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (sizeof(T) == 2) v[2 * i] = __uint_as_float(a[i] << 16), v[2 * i + 1] = __uint_as_float(a[i] & 0xffff0000u);
        else v[i] = __uint_as_float(a[i]), v[4 + i] = __uint_as_float(b[i]);
    }
}

template <typename T, bool ALIGNED>
__global__ void __launch_bounds__(THREADS, 4) beam_rows_kernel(const Args a) {
    constexpr int AT_ONCE = ALIGNED || sizeof(T) == 2 ? MOST_AT_ONCE : 2;  // what 64 registers hold
    __shared__ double2 parts[WARPS];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, row = blockIdx.y;
    let_next_kernel_start();
    wait_for_previous_kernels();
    const T* logits = reinterpret_cast<const T*>(a.logits) + (size_t)row * a.stride;
    const int end_run = min(a.runs, (int)(blockIdx.x + 1) * a.piece_runs);
    float* tops = a.tops + (size_t)row * a.runs;
    float m = -INFINITY;  // this thread's
    double sum = 0.0;
    auto look = [&](int run, int end, const Words (&w)[AT_ONCE]) {
        float v[AT_ONCE][PER], top[AT_ONCE], above = m;
        auto tops_of = [&] {
            above = m;
#pragma unroll
            for (int u = 0; u < AT_ONCE; ++u) {
                top[u] = max3(max3(v[u][0], v[u][1], v[u][2]), max3(v[u][3], v[u][4], v[u][5]), fmaxf(v[u][6], v[u][7]));
                above = fmaxf(above, top[u]);
            }
        };
#pragma unroll
        for (int u = 0; u < AT_ONCE; ++u) unpack<T>(w[u], v[u]);
        tops_of();
        // 2^(v log2 e + offset) * rest: the offset's rounding is an error of the exponent that all entries share, and what it has been rounded by is a float, too
        const float offset = -above * LOG2E, rest = fast_exp2(-fmaf(above, LOG2E, offset));
        Pair parts[4] = {};
#pragma unroll
        for (int u = 0; u < AT_ONCE; ++u)
#pragma unroll
            for (int k = 0; k < PER; k += 2) {
                const Pair y = fma2(Pair{v[u][k], v[u][k + 1]}, Pair{LOG2E, LOG2E}, Pair{offset, offset});
                parts[k / 2] = add2(parts[k / 2], Pair{fast_exp2(y.x), fast_exp2(y.y)});
            }
        const Pair half = add2(add2(parts[0], parts[1]), add2(parts[2], parts[3]));
        float part = (half.x + half.y) * rest;
        if (!(part < INFINITY) || !(fabsf(offset) < 0x1p24f)) {  // a NaN, an infinity, nothing but -infinity, or a maximum whose offset is too large to be precise
#pragma unroll
            for (int u = 0; u < AT_ONCE; ++u)
#pragma unroll
                for (int k = 0; k < PER; ++k) v[u][k] = cleaned(v[u][k]);
            tops_of();
            part = 0.f;
            if (above != -INFINITY) {
#pragma unroll
                for (int u = 0; u < AT_ONCE; ++u)
#pragma unroll
                    for (int k = 0; k < PER; ++k) part += fast_exp2((v[u][k] - above) * LOG2E);
            }
        }
        if (above > m) {
            sum *= m == -INFINITY ? 0.0 : (double)fast_exp2((m - above) * LOG2E);
            m = above;
        }
        sum += part;
#pragma unroll
        for (int u = 0; u < AT_ONCE; ++u) {
            const float largest = warp_largest(top[u]);
            if (lane == 0 && run + u * WARPS < end) tops[run + u * WARPS] = largest;
        }
    };
    // whole runs, all loads of a look on their way together; then the row's last one where it is not whole
    const int whole = min(end_run, a.vocab / RUN);
    int run = blockIdx.x * a.piece_runs + warp;
    auto looks = [&](auto full, int end) {  // FULL: all runs of a look are there
        constexpr bool FULL = decltype(full)::value;
        for (; run < end; run += WARPS * AT_ONCE) {
            Words w[AT_ONCE];
            int first[AT_ONCE];
#pragma unroll
            for (int u = 0; u < AT_ONCE; ++u) first[u] = (FULL ? run + u * WARPS : min(run + u * WARPS, whole - 1)) * RUN;
            const unsigned from = ALIGNED ? 0 : (unsigned)(uintptr_t)logits & 15;  // bytes behind a boundary
            switch (sizeof(T) == 2 ? from >> 1 : from >> 2) {
                case 0: load_runs<T, AT_ONCE, 0, false>(logits, first, lane, w); break;
                case 1: load_runs<T, AT_ONCE, sizeof(T) == 2 ? 0 : 1, sizeof(T) == 2>(logits, first, lane, w); break;
                case 2: load_runs<T, AT_ONCE, sizeof(T) == 2 ? 1 : 2, false>(logits, first, lane, w); break;
                case 3: load_runs<T, AT_ONCE, sizeof(T) == 2 ? 1 : 3, sizeof(T) == 2>(logits, first, lane, w); break;
                case 4: load_runs<T, AT_ONCE, 2, false>(logits, first, lane, w); break;
                case 5: load_runs<T, AT_ONCE, 2, true>(logits, first, lane, w); break;
                case 6: load_runs<T, AT_ONCE, 3, false>(logits, first, lane, w); break;
                default: load_runs<T, AT_ONCE, 3, true>(logits, first, lane, w);
            }
            if (!FULL) {
#pragma unroll
                for (int u = 1; u < AT_ONCE; ++u)
                    if (run + u * WARPS >= whole) w[u] = nothing<T>();
            }
            look(run, FULL ? 0x7fffffff : whole, w);
        }
    };
    if (ALIGNED) looks(std::true_type{}, whole - (AT_ONCE - 1) * WARPS);
    looks(std::false_type{}, whole);
    if (whole < end_run && warp == whole % WARPS) {
        Words w[AT_ONCE];
        w[0] = one_by_one<T>(logits, whole * RUN, a.vocab, lane);
#pragma unroll
        for (int u = 1; u < AT_ONCE; ++u) w[u] = nothing<T>();
        look(whole, end_run, w);
    }
    // the threads' sums, below the block's maximum, in the order of the threads
    const float above = warp_max(m);
    double part = m == -INFINITY ? 0.0 : sum * (double)fast_exp2((m - above) * LOG2E);
#pragma unroll
    for (int offset = 16; offset > 0; offset >>= 1) part += __shfl_xor_sync(0xffffffffu, part, offset);
    if (lane == 0) parts[warp] = make_double2(above, part);
    __syncthreads();
    if (tid == 0) {
        double top = -INFINITY, all = 0.0;
        for (int w = 0; w < WARPS; ++w) top = fmax(top, parts[w].x);
        for (int w = 0; w < WARPS; ++w) all += parts[w].x == -INFINITY ? 0.0 : parts[w].y * (double)fast_exp2((float)(parts[w].x - top) * LOG2E);
        a.sums[(size_t)row * a.pieces + blockIdx.x] = make_double2(top, all);
    }
}

// The second kernel: block = group.
constexpr int MOST_GROUP_THREADS = 1024, MOST_RUNS = 256, MOST_CANDIDATES = 1024, BESTS = 128, EARLY = 5, SPARE = 8;
static_assert(BESTS >= MOST_TAKE, "as many as are wanted");
struct Best {
    Key value;
    long long place;  // (beam, run or token): of equal values the lowest
};
__device__ __forceinline__ bool before(const Best& a, const Best& b) { return a.value > b.value || (a.value == b.value && a.place < b.place); }
// The best of the block, in every thread.
template <int GROUP_THREADS>
__device__ Best best_of_block(Best mine, Best* words) {
#pragma unroll
    for (int offset = 16; offset > 0; offset >>= 1) {
        const Best other{__shfl_xor_sync(0xffffffffu, mine.value, offset), __shfl_xor_sync(0xffffffffu, mine.place, offset)};
        if (before(other, mine)) mine = other;
    }
    __syncthreads();
    if ((threadIdx.x & 31) == 0) words[threadIdx.x >> 5] = mine;
    __syncthreads();
    Best best = words[0];
    for (int w = 1; w < GROUP_THREADS / 32; ++w)
        if (before(words[w], best)) best = words[w];
    return best;
}

template <typename T, int GROUP_THREADS>
__global__ void __launch_bounds__(GROUP_THREADS) beam_group_kernel(const Args a) {
    constexpr int WARPS = GROUP_THREADS / 32, TEAM = GROUP_THREADS / BESTS;
    __shared__ double offset[MOST_BEAMS];
    __shared__ Best words[WARPS];
    __shared__ Best candidates[MOST_CANDIDATES];
    __shared__ __align__(16) float bests[BESTS];
    __shared__ float shared_best;
    __shared__ float float_offset[MOST_BEAMS];  // -infinity: a beam that has no continuations
    __shared__ int chosen[MOST_RUNS], n_chosen, n_candidates;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, group = blockIdx.x, n = a.beams * a.runs;
    let_next_kernel_start();
    wait_for_previous_kernels();
    const float* tops = a.tops + (size_t)group * n;
    // thread t has the runs t, t + GROUP_THREADS, ... of all beams; its first ones are on their way while the sums are put together
    float early[EARLY];
#pragma unroll
    for (int k = 0; k < EARLY; ++k) early[k] = tid + k * GROUP_THREADS < n ? tops[tid + k * GROUP_THREADS] : -INFINITY;
    for (int beam = warp; beam < a.beams; beam += WARPS) {
        const double2* sums = a.sums + ((size_t)group * a.beams + beam) * a.pieces;
        const float score = cleaned(a.scores[group * a.beams + beam]);
        double top = -INFINITY, all = 0.0;
        for (int p = lane; p < a.pieces; p += 32) {
            const double2 part = sums[p];
            const double higher = fmax(top, part.x);
            if (higher != -INFINITY) all = (top == -INFINITY ? 0.0 : all * (double)fast_exp2((float)(top - higher) * LOG2E)) + (part.x == -INFINITY ? 0.0 : part.y * (double)fast_exp2((float)(part.x - higher) * LOG2E));
            top = higher;
        }
        const float above = warp_largest((float)top);  // a logit, which float holds
        all = top == -INFINITY ? 0.0 : all * (double)fast_exp2(((float)top - above) * LOG2E);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
        if (lane == 0) {
            const double off = score == -INFINITY || above == -INFINITY ? -INFINITY : (double)score - ((double)above + log(all));
            offset[beam] = off;
            float_offset[beam] = off == -INFINITY ? -INFINITY : (float)fmax(off, -(double)FLT_MAX);  // one that is no float counts as its lowest number, or as infinity
        }
    }
    if (tid == 0) n_chosen = n_candidates = 0;
    __syncthreads();
    auto score_of = [&](float logit, double off) -> Key { return logit == -INFINITY || off == -INFINITY ? 0 : ordered((double)logit + off); };
    // The runs: a bound that the best of at least `take` of them reach, if there are so many.  In float: what is added up there is off by 2^-24 of the offset and of itself, so the bound is lowered by 2^-21 of both,
    // and whatever scores as much as the `take`-th best in earnest reaches it.
    static_assert(MOST_BEAMS <= 32, "a lane a beam");
    const float largest = warp_largest(lane < a.beams && float_offset[lane] != -INFINITY ? fabsf(float_offset[lane]) : 0.f);  // offset
    const int beams_a_step = GROUP_THREADS / a.runs, runs_a_step = GROUP_THREADS - beams_a_step * a.runs, first_beam = tid / a.runs, first_run = tid - first_beam * a.runs;
    auto each = [&](auto with) {  // (run of all beams, its best logit, its beam's offset)
        int beam = first_beam, run = first_run;
        auto next = [&] {
            beam += beams_a_step, run += runs_a_step;
            if (run >= a.runs) run -= a.runs, ++beam;
        };
#pragma unroll
        for (int k = 0; k < EARLY; ++k) {
            if (tid + k * GROUP_THREADS < n) with(tid + k * GROUP_THREADS, early[k], float_offset[beam]);
            next();
        }
        for (int i = tid + EARLY * GROUP_THREADS; i < n; i += EARLY * GROUP_THREADS) {
            float more[EARLY];
#pragma unroll
            for (int k = 0; k < EARLY; ++k) more[k] = i + k * GROUP_THREADS < n ? tops[i + k * GROUP_THREADS] : -INFINITY;
#pragma unroll
            for (int k = 0; k < EARLY; ++k) {
                if (i + k * GROUP_THREADS < n) with(i + k * GROUP_THREADS, more[k], float_offset[beam]);
                next();
            }
        }
    };
    float mine = -INFINITY;
    each([&](int, float top, float off) { mine = fmaxf(mine, top + off); });
    auto lowered = [&](float best) {
        const float bound = best - 0x1p-21f * (largest + fabsf(best));
        return largest < FLT_MAX / 4 && bound > -INFINITY ? bound : -INFINITY;  // no number, or scores that float does not add up: everything reaches it
    };
    auto choose = [&](float bound) {
        each([&](int i, float top, float off) {
            if (top == -INFINITY || off == -INFINITY || !(top + off >= bound)) return;
            const int at = atomicAdd(&n_chosen, 1);
            if (at < MOST_RUNS) chosen[at] = i;
        });
    };
    // The `take`-th largest of what the threads have, found bit by bit, or a number that few more reach.
    auto reached_by_take = [&](float value) {
        const unsigned bits = __float_as_uint(value), rank = value == -INFINITY ? 0u : bits >> 31 ? ~bits : bits | 1u << 31;  // in the order of the numbers
        unsigned reached = 0;
        for (unsigned bit = 1u << 31; bit; bit >>= 1) {
            const int ranks = __syncthreads_count(rank >= (reached | bit));
            if (ranks >= a.take) {
                reached |= bit;
                if (ranks <= a.take + SPARE) break;
            }
        }
        return __uint_as_float(reached >> 31 ? reached ^ 1u << 31 : ~reached);  // no number where fewer threads have one
    };
    // First the `take`-th largest of what teams of threads have as their best.
    {
        float best = mine;
#pragma unroll
        for (int o = 1; o < TEAM; o <<= 1) best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, o));
        if (tid % TEAM == 0) bests[tid / TEAM] = best;
        __syncthreads();
        // a team counts for one of them what comes before it, equal ones by their numbers
        const int of = tid / TEAM;
        const float me = bests[of];
        int ahead = 0;
#pragma unroll
        for (int k = 0; k < BESTS / TEAM; ++k) {
            const int other = k * TEAM + tid % TEAM;
            ahead += bests[other] > me || (bests[other] == me && other < of);
        }
#pragma unroll
        for (int o = 1; o < TEAM; o <<= 1) ahead += __shfl_xor_sync(0xffffffffu, ahead, o);
        if (ahead == a.take - 1 && tid % TEAM == 0) shared_best = me;
        __syncthreads();
    }
    float bound = lowered(shared_best);
    choose(bound);
    __syncthreads();
    if (n_chosen > 2 * a.take + 32) {  // a few beams have all that is best, and so do few of the teams
        bound = lowered(reached_by_take(mine));
        if (tid == 0) n_chosen = 0;
        __syncthreads();
        choose(bound);
    }
    __syncthreads();
    int n_runs = n_chosen;
    if (n_runs > MOST_RUNS) {  // many equal ones: the `take` best, one after the other
        Best last{~0ull, -1};
        for (n_runs = 0; n_runs < a.take; ++n_runs) {
            Best best{0, 0x7fffffffffffffffll};
            for (int i = tid; i < n; i += GROUP_THREADS) {
                const Best here{score_of(tops[i], offset[i / a.runs]), i};
                if (here.value && before(last, here) && before(here, best)) best = here;
            }
            last = best_of_block<GROUP_THREADS>(best, words);
            if (!last.value) break;
            if (tid == 0) chosen[n_runs] = (int)last.place;
            __syncthreads();
        }
    }
    // their entries that reach it
    struct Entry { float logit; int beam, token; };
    auto entry = [&](int i, int k) -> Entry {  // entry k of chosen run i
        const int run = chosen[i], beam = run / a.runs, token = (run - beam * a.runs) * RUN + k;
        return {token < a.vocab ? cleaned(to_float(reinterpret_cast<const T*>(a.logits)[(size_t)(group * a.beams + beam) * a.stride + token])) : -INFINITY, beam, token};
    };
    auto exactly = [&](const Entry& e) -> Best { return {score_of(e.logit, offset[e.beam]), (long long)e.beam << 32 | e.token}; };
    float best = -INFINITY;  // of this thread's entries
    auto read_runs = [&](auto at_once) {
        constexpr int RUNS_AT_ONCE = decltype(at_once)::value;
        for (int i0 = warp; i0 < n_runs; i0 += RUNS_AT_ONCE * WARPS) {
            float v[RUNS_AT_ONCE][PER];
            int beam[RUNS_AT_ONCE], token[RUNS_AT_ONCE];
#pragma unroll
            for (int u = 0; u < RUNS_AT_ONCE; ++u) {
                const int i = i0 + u * WARPS, run = chosen[min(i, n_runs - 1)];
                beam[u] = run / a.runs, token[u] = (run - beam[u] * a.runs) * RUN + lane;
                const T* row = reinterpret_cast<const T*>(a.logits) + (size_t)(group * a.beams + beam[u]) * a.stride;
#pragma unroll
                for (int k = 0; k < PER; ++k) v[u][k] = i < n_runs && token[u] + k * 32 < a.vocab ? to_float(row[token[u] + k * 32]) : -INFINITY;
            }
#pragma unroll
            for (int u = 0; u < RUNS_AT_ONCE; ++u) {
                const float off = float_offset[beam[u]];
#pragma unroll
                for (int k = 0; k < PER; ++k) {
                    const float logit = cleaned(v[u][k]);
                    if (logit == -INFINITY || !(logit + off >= bound)) continue;
                    best = fmaxf(best, logit + off);
                    const int at = atomicAdd(&n_candidates, 1);
                    if (at < MOST_CANDIDATES) candidates[at] = exactly(Entry{logit, beam[u], token[u] + k * 32});
                }
            }
        }
    };
    if (n_runs <= WARPS) read_runs(std::integral_constant<int, 1>{});
    else if (n_runs <= 2 * WARPS) read_runs(std::integral_constant<int, 2>{});
    else read_runs(std::integral_constant<int, 3>{});
    __syncthreads();
    if (n_candidates > MOST_CANDIDATES) {  // the best stand close together in the vocabulary
        bound = fmaxf(bound, lowered(reached_by_take(best)));
        if (tid == 0) n_candidates = 0;
        __syncthreads();
        read_runs(std::integral_constant<int, 1>{});
        __syncthreads();
    }
    const int found = n_candidates;
    int written = min(a.take, found);
    auto write = [&](int place, const Best& best) {
        const size_t at = (size_t)group * a.take + place;
        a.parents[at] = (int)(best.place >> 32), a.tokens[at] = (int)best.place, a.out_scores[at] = (float)value_of(best.value);
    };
    if (found <= MOST_CANDIDATES) {
        // a team of threads, a power of two of a warp's, counts for a candidate what comes before it
        int team = 1;
        while (team < 32 && 2 * team * found <= GROUP_THREADS) team *= 2;
        for (int of0 = 0; of0 < found; of0 += GROUP_THREADS / team) {
            const int of = of0 + tid / team;
            const Best me = candidates[min(of, found - 1)];
            int ahead = 0;
            for (int i = tid & (team - 1); i < found; i += team) ahead += before(candidates[i], me);
            for (int o = 1; o < team; o <<= 1) ahead += __shfl_xor_sync(0xffffffffu, ahead, o);
            if (of < found && ahead < a.take && (tid & (team - 1)) == 0) write(ahead, me);
        }
    } else {  // one after the other
        Best last{~0ull, -1};
        for (written = 0; written < a.take; ++written) {
            Best best{0, 0x7fffffffffffffffll};
            for (int i = warp; i < n_runs; i += WARPS)
                for (int k = lane; k < RUN; k += 32) {
                    const Best here = exactly(entry(i, k));
                    if (here.value && before(last, here) && before(here, best)) best = here;
                }
            last = best_of_block<GROUP_THREADS>(best, words);
            if (!last.value) break;
            if (tid == 0) write(written, last);
        }
    }
    for (int i = written + tid; i < a.take; i += GROUP_THREADS) {
        const size_t at = (size_t)group * a.take + i;
        a.parents[at] = -1, a.tokens[at] = -1, a.out_scores[at] = -INFINITY;
    }
}
template <typename T>
int launch(const Args& a, cudaStream_t stream) {
    // rows that all begin on 16 bytes ask nothing in their loop (256 rows of float, us: 33.0 / 35.0 by the other kernel)
    const bool aligned = ((uintptr_t)a.logits & 15) == 0 && (a.groups * a.beams == 1 || a.stride * (long long)sizeof(T) % 16 == 0);
    if (int code = launch_after_previous(aligned ? beam_rows_kernel<T, true> : beam_rows_kernel<T, false>, dim3(a.pieces, a.groups * a.beams), dim3(THREADS), 0, stream, a)) return code;
    // Half the threads where there is little to look through (us on the device, 512 / 1024 threads: four beams of 152,064 8.3 / 8.9, 32 groups of them 17.8 / 18.5, 256 groups of one beam 30.1 / 31.4; but eight beams, 16 taken
    // 9.8 / 9.3, 16 beams, 32 taken 13.6 / 12.3, 32 beams 19.2 / 15.8).
    if ((long long)a.beams * a.runs <= 2560 && a.take <= 16) return launch_after_previous(beam_group_kernel<T, 512>, dim3(a.groups), dim3(512), 0, stream, a);
    return launch_after_previous(beam_group_kernel<T, MOST_GROUP_THREADS>, dim3(a.groups), dim3(MOST_GROUP_THREADS), 0, stream, a);
}
}  // namespace

// Into how many pieces rows are cut, and runs of a piece: eight blocks a multiprocessor, which holds four of them, of two looks of its warps at least.  (32 groups of 8 beams: 28.2 us; four 29.6, six 30.7, twelve 28.5.)
static int pieces_for(int rows, int vocab, int sms, int* piece_runs) {
    const long long runs = (vocab + RUN - 1) / RUN, room = 8LL * sms / rows, most = (runs + 2 * WARPS * MOST_AT_ONCE - 1) / (2 * WARPS * MOST_AT_ONCE);
    long long n = room < 1 ? 1 : room;
    n = n < most ? n : most;
    const long long each = ((runs + n - 1) / n + WARPS * MOST_AT_ONCE - 1) / (WARPS * MOST_AT_ONCE) * (WARPS * MOST_AT_ONCE);
    *piece_runs = (int)each;
    return (int)((runs + each - 1) / each);
}
// Bytes of scratch that hb_beam_select takes.
HB_EXPORT long long hb_beam_select_scratch(int groups, int beams, int vocab, int take, int sms) {
    if (groups <= 0 || beams <= 0 || beams > MOST_BEAMS || vocab <= 0 || vocab > 0x7fffffff - RUN || take <= 0 || take > MOST_TAKE || sms <= 0) return 0;
    const long long rows = (long long)groups * beams;
    if (rows > 65535) return 0;
    int piece_runs;
    return rows * pieces_for((int)rows, vocab, sms, &piece_runs) * 16 + rows * ((vocab + RUN - 1) / RUN) * 4;
}
// logits [groups * beams, vocab] (bfloat16 or float) with rows `stride` apart; scores [groups, beams]; parents, tokens, out_scores [groups, take].  scratch: hb_beam_select_scratch bytes on a
// 16-byte boundary.
HB_EXPORT int hb_beam_select(const void* logits, int is_bf16, long long stride, const float* scores, int groups, int beams, int vocab, int take, int* parents, int* tokens, float* out_scores, int sms,
                             void* scratch, cudaStream_t stream) {
    if (groups <= 0) return 0;
    if (!logits || !scores || !parents || !tokens || !out_scores || !scratch || beams <= 0 || vocab <= 0 || take <= 0 || sms <= 0 || stride < vocab || ((uintptr_t)scratch & 15)) return HB_BAD_ARGUMENT;
    if (((uintptr_t)logits & (is_bf16 ? 1 : 3))) return HB_BAD_ARGUMENT;
    const long long rows = (long long)groups * beams, runs = ((long long)vocab + RUN - 1) / RUN;
    if (beams > MOST_BEAMS || take > MOST_TAKE || rows > 65535 || vocab > 0x7fffffff - RUN || beams * runs > 0x7fffffffLL - 2 * EARLY * MOST_GROUP_THREADS) return HB_UNSUPPORTED_SIZE;
    Args a{logits, stride, scores, groups, beams, vocab, take, (int)runs};
    a.pieces = pieces_for((int)rows, vocab, sms, &a.piece_runs);
    a.sums = (double2*)scratch, a.tops = (float*)(a.sums + rows * a.pieces), a.parents = parents, a.tokens = tokens, a.out_scores = out_scores;
    return is_bf16 ? launch<bf16>(a, stream) : launch<float>(a, stream);
}
HB_EXPORT int hb_beam_select_packed(const void* arguments) { return call_packed(&hb_beam_select, arguments); }
