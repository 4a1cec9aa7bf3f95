// The best continuations of a group's beams over beams and vocabulary:
//
//     score(b, v) = score_b + z_bv - log sum_u e^(z_bu)            the `take` largest of them, of equal ones the lowest (b, v)
//
// The first kernel reads every row once and leaves the sum, and the maximum of every run of 256 logits.  The second has a block per group: with the rows' sums it knows every run's best score.  The runs whose best
// are the `take` best of all runs hold the `take` best continuations (of a run that is not among them, `take` others hold something better), so only those are read again: a few KB of them.  Both
// searches take a bound first, the `take`-th largest of what eighths of the warps have found to be their best, and then look at what reaches it: little more than `take` in all but contrived rows, for which there is a way that goes by one
// continuation after the other.
//
// Measured: 32 groups of 8 beams over bfloat16 logits of 152,064 26.3 us for 78 MB: the first kernel 17 (4.6 TB/s; as long without its exponentials, and with more or fewer blocks or loads on their way), the second 9, a chain of a
// logarithm, three meetings of the block and two trips to memory.  One group of four beams 8.6 us.
//
// Scores are compared as float64: a score is score_b - lse_b, a number of the row, plus the logit, and float32 would make ties of scores that are not equal.  Sums of a thread's 32 entries are float, everything above
// them float64; exponentials are the hardware's (2^-22 of a term).  Which thread adds up what goes by the entry's index alone, not by the row's alignment, so rows that hold the same have the same sums.
//
// A NaN counts as -infinity, +infinity as the largest number.  A logit of -infinity, and everything of a beam whose score is -infinity or NaN, is no candidate.  A place without a candidate has parent -1,
// token -1 and score -infinity.
#include <float.h>

#include <type_traits>

#include "common.cuh"

namespace {
typedef __nv_bfloat16 bf16;
typedef unsigned long long Key;  // a float64's bits in its order; 0: none
constexpr int THREADS = 256, WARPS = THREADS / 32, RUN = 256, PER = RUN / 32, AT_ONCE = 4;  // a warp looks at AT_ONCE runs at a time, PER entries a lane of each
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

// A lane's eight entries of the run that begins at `first`: bfloat16 [8 lane, 8 lane + 8), float [4 lane, 4 lane + 4) and 128 further on.  Where rows do not begin on 16 bytes the words that hold a lane's entries are
// fetched from the boundary before and shifted; at a row's ends, entry by entry.
struct Words { uint4 lo, hi; };
__device__ __forceinline__ uint4 shifted(const uint4& a, const uint4& b, int words) {  // four of the eight words, from `words` on
    uint4 r = a;
    unsigned s0 = b.x, s1 = b.y, s2 = b.z;
    if (words & 2) r = make_uint4(r.z, r.w, s0, s1), s0 = s2;
    if (words & 1) r = make_uint4(r.y, r.z, r.w, s0);
    return r;
}
template <typename T, bool PLAIN>
__device__ __forceinline__ Words fetch(const T* row, int first, int end, int off, int lane) {  // off: entries that a row begins behind a 16-byte boundary; PLAIN: none, and the run is whole
    Words w;
    if (sizeof(T) == 2) {
        const int at = first + 8 * lane;
        if (PLAIN || (off == 0 && first + RUN <= end)) {
            w.lo = *reinterpret_cast<const uint4*>(row + at);
        } else if (first >= 8 && first + RUN + 8 <= end) {
            const uint4* p = reinterpret_cast<const uint4*>(row + at - off);
            const uint4 a = p[0], b = p[1];
            const uint4 c = shifted(a, b, off >> 1);
            if (off & 1) {
                const unsigned next = (off >> 1) == 0 ? b.x : (off >> 1) == 1 ? b.y : (off >> 1) == 2 ? b.z : b.w;
                w.lo = make_uint4(__funnelshift_r(c.x, c.y, 16), __funnelshift_r(c.y, c.z, 16), __funnelshift_r(c.z, c.w, 16), __funnelshift_r(c.w, next, 16));
            } else {
                w.lo = c;
            }
        } else {
            unsigned short h[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) h[i] = at + i < end ? __bfloat16_as_ushort(reinterpret_cast<const bf16*>(row)[at + i]) : 0xff80;
            w.lo = make_uint4(h[0] | (unsigned)h[1] << 16, h[2] | (unsigned)h[3] << 16, h[4] | (unsigned)h[5] << 16, h[6] | (unsigned)h[7] << 16);
        }
    } else {
        const int at = first + 4 * lane;
        if (PLAIN || (off == 0 && first + RUN <= end)) {
            w.lo = *reinterpret_cast<const uint4*>(row + at), w.hi = *reinterpret_cast<const uint4*>(row + at + 128);
        } else if (first >= 4 && first + RUN + 4 <= end) {
            const uint4* p = reinterpret_cast<const uint4*>(row + at - off);
            const uint4 a = p[0], b = p[1], c = p[32], d = p[33];
            w.lo = shifted(a, b, off), w.hi = shifted(c, d, off);
        } else {
            unsigned x[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int k = at + (i & 3) + (i >> 2) * 128;
                x[i] = k < end ? reinterpret_cast<const unsigned*>(row)[k] : 0xff800000u;
            }
            w.lo = make_uint4(x[0], x[1], x[2], x[3]), w.hi = make_uint4(x[4], x[5], x[6], x[7]);
        }
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

template <typename T>
__global__ void __launch_bounds__(THREADS, 4) beam_rows_kernel(const Args a) {
    __shared__ double2 parts[WARPS];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, row = blockIdx.y;
    let_next_kernel_start();
    wait_for_previous_kernels();
    const T* logits = reinterpret_cast<const T*>(a.logits) + (size_t)row * a.stride;
    const int off = (int)(((uintptr_t)logits & 15) / sizeof(T)), end_run = min(a.runs, (int)(blockIdx.x + 1) * a.piece_runs);
    float* tops = a.tops + (size_t)row * a.runs;
    float m = -INFINITY;  // this thread's
    double sum = 0.0;
    auto look = [&](int run, auto plain) {
        constexpr bool PLAIN = decltype(plain)::value;
        Words w[AT_ONCE];
#pragma unroll
        for (int u = 0; u < AT_ONCE; ++u) {
            if (PLAIN || run + u * WARPS < end_run) w[u] = fetch<T, PLAIN>(logits, (run + u * WARPS) * RUN, a.vocab, off, lane);
            else w[u].lo = w[u].hi = sizeof(T) == 2 ? make_uint4(0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u) : make_uint4(0xff800000u, 0xff800000u, 0xff800000u, 0xff800000u);
        }
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
            if (lane == 0 && (PLAIN || run + u * WARPS < end_run)) tops[run + u * WARPS] = largest;
        }
    };
    // the runs that a look has whole, in a loop that asks no more questions
    const int whole = min(end_run, off ? 0 : a.vocab / RUN);
    int run = blockIdx.x * a.piece_runs + warp;
    for (; run + (AT_ONCE - 1) * WARPS < whole; run += WARPS * AT_ONCE) look(run, std::true_type{});
    for (; run < end_run; run += WARPS * AT_ONCE) look(run, std::false_type{});
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
constexpr int GROUP_THREADS = 1024, MOST_RUNS = 256, MOST_CANDIDATES = GROUP_THREADS, BESTS = GROUP_THREADS / 8, EARLY = 6;
static_assert(BESTS >= MOST_TAKE, "as many as are wanted");
struct Best {
    Key value;
    long long place;  // (beam, run or token): of equal values the lowest
};
__device__ __forceinline__ bool before(const Best& a, const Best& b) { return a.value > b.value || (a.value == b.value && a.place < b.place); }
// The best of the block, in every thread.
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

template <typename T>
__global__ void __launch_bounds__(GROUP_THREADS) beam_group_kernel(const Args a) {
    __shared__ double offset[MOST_BEAMS];
    __shared__ Best words[GROUP_THREADS / 32];
    __shared__ Best candidates[MOST_CANDIDATES];
    __shared__ __align__(16) float bests[BESTS];
    __shared__ float shared_bound;
    __shared__ int chosen[MOST_RUNS], n_chosen, n_candidates;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, group = blockIdx.x, n = a.beams * a.runs;
    let_next_kernel_start();
    wait_for_previous_kernels();
    const float* tops = a.tops + (size_t)group * n;
    // a beam's runs are a team of warps'; a thread's first ones are on their way while the sums are put together
    const int team = GROUP_THREADS / 32 / a.beams, beam_here = warp / team, runs_here = beam_here < a.beams ? a.runs : 0, first_run = (warp - beam_here * team) * 32 + lane;
    const float* row_tops = tops + (size_t)(beam_here < a.beams ? beam_here : 0) * a.runs;
    float early[EARLY];
#pragma unroll
    for (int k = 0; k < EARLY; ++k) early[k] = first_run + k * team * 32 < runs_here ? row_tops[first_run + k * team * 32] : -INFINITY;
    if (warp < a.beams) {  // a warp a beam
        const double2* sums = a.sums + ((size_t)group * a.beams + warp) * a.pieces;
        const float score = cleaned(a.scores[group * a.beams + warp]);
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
        if (lane == 0) offset[warp] = score == -INFINITY || above == -INFINITY ? -INFINITY : (double)score - ((double)above + log(all));
    }
    if (tid == 0) n_chosen = n_candidates = 0;
    __syncthreads();
    auto score_of = [&](float logit, double off) -> Key { return logit == -INFINITY || off == -INFINITY ? 0 : ordered((double)logit + off); };
    // The runs: a bound that the best of at least `take` of them reach, if there are so many: the `take`-th largest of what eight lanes together have as theirs.  In float: what is added up there is off by 2^-24 of the
    // offset and of itself, so the bound is lowered by 2^-21 of both, and whatever scores as much as the `take`-th best in earnest reaches it.
    const float off_here = beam_here < a.beams ? (float)offset[beam_here] : -INFINITY;
    float mine = -INFINITY;
#pragma unroll
    for (int k = 0; k < EARLY; ++k) mine = fmaxf(mine, early[k] + off_here);
    for (int i = first_run + EARLY * team * 32; i < runs_here; i += team * 32) mine = fmaxf(mine, row_tops[i] + off_here);
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) mine = fmaxf(mine, __shfl_xor_sync(0xffffffffu, mine, o));
    if ((lane & 7) == 0) bests[tid / 8] = mine;
    __syncthreads();
    {  // eight threads count for one of them what comes before it, equal ones by their numbers
        const int of = tid / 8;
        const float me = bests[of];
        int ahead = 0;
#pragma unroll
        for (int k = 0; k < BESTS / 8; ++k) {
            const int other = k * 8 + (lane & 7);
            ahead += bests[other] > me || (bests[other] == me && other < of);
        }
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) ahead += __shfl_xor_sync(0xffffffffu, ahead, o);
        if (ahead == a.take - 1 && (lane & 7) == 0) {
            float largest = 0.f;
            for (int b = 0; b < a.beams; ++b)
                if (offset[b] != -INFINITY) largest = fmaxf(largest, fabsf((float)offset[b]));
            const float lowered = me - 0x1p-21f * (largest + fabsf(me));
            shared_bound = lowered > -INFINITY ? lowered : -INFINITY;  // no number, either: everything reaches it
        }
    }
    __syncthreads();
    const float bound = shared_bound;
    auto choose = [&](int i, float top) {
        if (top == -INFINITY || beam_here >= a.beams || offset[beam_here] == -INFINITY || !(top + off_here >= bound)) return;  // a dead beam's run reaches a bound of -infinity, too
        const int at = atomicAdd(&n_chosen, 1);
        if (at < MOST_RUNS) chosen[at] = beam_here * a.runs + i;
    };
#pragma unroll
    for (int k = 0; k < EARLY; ++k) choose(first_run + k * team * 32, early[k]);
    for (int i = first_run + EARLY * team * 32; i < runs_here; i += team * 32) choose(i, row_tops[i]);
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
            last = best_of_block(best, words);
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
    for (int i = warp; i < n_runs; i += GROUP_THREADS / 32) {
        const int run = chosen[i], beam = run / a.runs, token = (run - beam * a.runs) * RUN + lane;
        const T* row = reinterpret_cast<const T*>(a.logits) + (size_t)(group * a.beams + beam) * a.stride;
        float v[PER];
#pragma unroll
        for (int k = 0; k < PER; ++k) v[k] = token + k * 32 < a.vocab ? to_float(row[token + k * 32]) : -INFINITY;
        const float off = (float)offset[beam];
#pragma unroll
        for (int k = 0; k < PER; ++k) {
            const float logit = cleaned(v[k]);
            if (logit == -INFINITY || !(logit + off >= bound)) continue;
            const int at = atomicAdd(&n_candidates, 1);
            if (at < MOST_CANDIDATES) candidates[at] = exactly(Entry{logit, beam, token + k * 32});
        }
    }
    __syncthreads();
    const int found = n_candidates;
    int written = min(a.take, found);
    auto write = [&](int place, const Best& best) {
        const size_t at = (size_t)group * a.take + place;
        a.parents[at] = (int)(best.place >> 32), a.tokens[at] = (int)best.place, a.out_scores[at] = (float)value_of(best.value);
    };
    if (found <= MOST_CANDIDATES) {
        if (tid < found) {
            const Best me = candidates[tid];
            int ahead = 0;
            for (int i = 0; i < found; ++i) ahead += before(candidates[i], me);
            if (ahead < a.take) write(ahead, me);
        }
    } else {  // one after the other
        Best last{~0ull, -1};
        for (written = 0; written < a.take; ++written) {
            Best best{0, 0x7fffffffffffffffll};
            for (int i = warp; i < n_runs; i += GROUP_THREADS / 32)
                for (int k = lane; k < RUN; k += 32) {
                    const Best here = exactly(entry(i, k));
                    if (here.value && before(last, here) && before(here, best)) best = here;
                }
            last = best_of_block(best, words);
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
    if (int code = launch_after_previous(beam_rows_kernel<T>, dim3(a.pieces, a.groups * a.beams), dim3(THREADS), 0, stream, a)) return code;
    return launch_after_previous(beam_group_kernel<T>, dim3(a.groups), dim3(GROUP_THREADS), 0, stream, a);
}
}  // namespace

// Into how many pieces rows are cut, and runs of a piece: eight blocks a multiprocessor, which holds four of them, of two looks of its warps at least.  (32 groups of 8 beams: 28.2 us; four 29.6, six 30.7, twelve 28.5.)
static int pieces_for(int rows, int vocab, int sms, int* piece_runs) {
    const long long runs = (vocab + RUN - 1) / RUN, room = 8LL * sms / rows, most = (runs + 2 * WARPS * AT_ONCE - 1) / (2 * WARPS * AT_ONCE);
    long long n = room < 1 ? 1 : room;
    n = n < most ? n : most;
    const long long each = ((runs + n - 1) / n + WARPS * AT_ONCE - 1) / (WARPS * AT_ONCE) * (WARPS * AT_ONCE);
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
    if (beams > MOST_BEAMS || take > MOST_TAKE || rows > 65535 || vocab > 0x7fffffff - RUN || beams * runs > 0x7fffffffLL) return HB_UNSUPPORTED_SIZE;
    Args a{logits, stride, scores, groups, beams, vocab, take, (int)runs};
    a.pieces = pieces_for((int)rows, vocab, sms, &a.piece_runs);
    a.sums = (double2*)scratch, a.tops = (float*)(a.sums + rows * a.pieces), a.parents = parents, a.tokens = tokens, a.out_scores = out_scores;
    return is_bf16 ? launch<bf16>(a, stream) : launch<float>(a, stream);
}
