// A cache is cut back to a budget: of each key/value head of a request (and layer) the `keep` slots that weigh most stay, and move into the first `keep` slots.
//
// A slot ranks by its weight, a NaN as -infinity; one whose position is below `first` or among the last `recent` ones ranks as +infinity.  Of equal ranks the lowest slots stay.  What stays in the
// first `keep` slots is not moved; the i-th of the others that stay goes into the i-th slot that is left free.  Keys were rotated when they were stored, so attention does not ask in which slot one
// stands, and the positions go along with them.  Sources stand at `keep` and beyond, targets below, so nothing is read that has been written, in whatever order the records move.
//
// A request of at most `keep` slots stays as it is.
//
// A head is a cluster of one to eight blocks, each of which has a part of the slots and holds their ranks in shared memory.  The rank of the last slot that stays is found digit by digit (11, 11 and 10 bits of the
// weight's ordered bits), by counting: after the first digit few slots are left to count, and each block adds what it has counted to all blocks' sums.  Two more walks along the ranks say how many slots move and are
// free before each warp's, and then which; where a slot stands in its list follows from the slots before it alone, so nothing depends on which block came first.  Then the cluster moves what is to move, records
// included, or leaves those to a second kernel.
//
// Measured: 24 layers of 2 heads that give up one slot of 1,025 7.9 us, a chain of some 14,000 clocks: the slots' arrival, three digits of 1,500 clocks each (counts, a sum over the bins, two meetings of the block), lists.  Four layers of 8
// heads that keep 4,096 of 32,771 slots 42 us: half of it the choice (arrival 8,000 clocks, digits 14,000 with the cluster's meetings, lists and sums 10,000), half the moves of 117 MB of records at 5.4 TB/s.
#include "common.cuh"

namespace {
constexpr int MOST_BLOCKS = 8;
constexpr int DIGIT = 11, BINS = 2 * (1 << DIGIT) + (1 << (32 - 2 * DIGIT));  // 11, 11 and 10 bits of a rank
constexpr int LOOK = 128;  // slots of a warp's look, four a lane
constexpr int MOST_HELD = 40 * 1024;  // ranks that a block holds

struct Args {
    const int* lengths; const int* newest; int requests;
    const float* weights; const int* positions;  // [layers, requests, kv_heads, capacity]
    float* to_weights; int* to_positions;        // likewise; may be the same
    int capacity, longest, keep, first, recent;
    int layers, kv_heads;
    int* left;           // [requests]: min(length, keep)
    int* moves;          // [layers * requests * kv_heads]
    int* from;           // [layers * requests * kv_heads, most]
    int* to;             // likewise
    int most;            // moves of a head: min(keep, longest - keep)
    uint4* cache;        // [layers, pages, 2, kv_heads, page, record]
    int record;          // 16-byte pieces of a record
    const int* block_table; int table_width;
    int page_shift, pages;
    int blocks;          // of a cluster
    int moves_here;      // the records are moved by the first kernel, too
    int* status;
};

// Order-preserving; both zeros are the same, a NaN is -infinity.
__device__ __forceinline__ unsigned ordered(float v) {
    if (v != v) v = -INFINITY;
    const unsigned b = __float_as_uint(v + 0.f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ unsigned rank_of(float weight, int position, int first, long long after) {
    return position < first || position > after ? ordered(INFINITY) : ordered(weight);
}
__device__ __forceinline__ int length_of(const Args& a, int request) { return min(max(a.lengths[request], 0), a.longest); }

__device__ __forceinline__ unsigned their(const void* p, int rank) {  // what another block of the cluster has at this place of its shared memory
    unsigned at;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"((unsigned)__cvta_generic_to_shared(p)), "r"(rank));
    return at;
}
__device__ __forceinline__ int4 theirs4(const int* p, int rank) {
    int4 v;
    asm volatile("ld.shared::cluster.v4.s32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(their(p, rank)) : "memory");
    return v;
}
// All threads of the cluster; what they have written before, everywhere, is there for them behind it.  One thread's fence stands for its block, which has met before it (as many fences as there are warps take a
// thousand clocks).
__device__ __forceinline__ void cluster_meet(int blocks) {
    __syncthreads();
    if (blocks == 1) return;
    if (threadIdx.x == 0) asm volatile("fence.acq_rel.cluster;" ::: "memory");
    asm volatile("barrier.cluster.arrive.relaxed;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
// Adds to what each block of the cluster has at this place.
__device__ __forceinline__ void add_to_all(int* p, int n, int blocks) {
    for (int b = 0; b < blocks; ++b) asm volatile("red.relaxed.cluster.shared::cluster.add.s32 [%0], %1;" ::"r"(their(p, b)), "r"(n) : "memory");
}
// What the blocks have at this place, all on their way together.
__device__ __forceinline__ void all_of_theirs(const int* p, int blocks, int4 (&x)[MOST_BLOCKS]) {
    if (blocks == 1) {
        x[0] = *reinterpret_cast<const int4*>(p);
        return;
    }
#pragma unroll
    for (int b = 0; b < MOST_BLOCKS; ++b)
        if (b < blocks) x[b] = theirs4(p, b);
}
__device__ __forceinline__ int warp_before(int v, int lane) {  // sum over the lanes before this one
    int end = v;
#pragma unroll
    for (int offset = 1; offset < 32; offset <<= 1) {
        const int other = __shfl_up_sync(0xffffffffu, end, offset);
        if (lane >= offset) end += other;
    }
    return end - v;
}

// The records of a head's moves: warp `first` of `step` takes every step-th CHUNK of them.  A lane finds out where one of them goes from and to; then a team of lanes a move carries 16 bytes of its key and value a lane and
// turn, AHEAD moves of a team on their way together.  Records are read past L1, where a line that also holds a slot that is filled elsewhere must not stay for the kernel behind this one.
constexpr int CHUNK = 16, AHEAD = 4;
__device__ __forceinline__ void move_records(const Args& a, const int* from, const int* to, int n_moves, const int* table, int layer, int kvh, int first, int step) {
    const int lane = threadIdx.x & 31, mask = (1 << a.page_shift) - 1;
    int team = 1;  // lanes: a power of two
    while (team < 32 && team < 2 * a.record) team *= 2;
    const int teams = 32 / team, mine = lane / team;
    uint4* layer_cache = a.cache + (((size_t)layer * a.pages * 2 * a.kv_heads) << a.page_shift) * a.record;
    const size_t values = ((size_t)a.kv_heads << a.page_shift) * a.record;  // from a key to its value
    for (int base = first * CHUNK; base < n_moves; base += step * CHUNK) {
        const int n = min(CHUNK, n_moves - base);
        long long source = -1, target = -1;  // of this lane's move
        if (lane < n) {
            const int s = from[base + lane], t = to[base + lane], page = table[s >> a.page_shift], to_page = table[t >> a.page_shift];
            if (page < 0 || page >= a.pages || to_page < 0 || to_page >= a.pages) {
                atomicOr(a.status, HB_STATUS_BAD_PAGE);
            } else {
                source = ((((long long)page * 2 * a.kv_heads + kvh) << a.page_shift) + (s & mask)) * a.record;
                target = ((((long long)to_page * 2 * a.kv_heads + kvh) << a.page_shift) + (t & mask)) * a.record;
            }
        }
        for (int k0 = 0; k0 < n; k0 += AHEAD * teams) {
            long long s[AHEAD], t[AHEAD];
#pragma unroll
            for (int k = 0; k < AHEAD; ++k) {
                const int move = k0 + k * teams + mine;
                s[k] = __shfl_sync(0xffffffffu, source, move & 31), t[k] = __shfl_sync(0xffffffffu, target, move & 31);
                if (move >= n) s[k] = -1;
            }
            for (int piece = lane & (team - 1); piece < 2 * a.record; piece += team) {
                const size_t at = piece < a.record ? piece : values + piece - a.record;
                uint4 held[AHEAD];
#pragma unroll
                for (int k = 0; k < AHEAD; ++k)
                    if (s[k] >= 0) held[k] = __ldcg(layer_cache + s[k] + at);
#pragma unroll
                for (int k = 0; k < AHEAD; ++k)
                    if (s[k] >= 0) layer_cache[t[k] + at] = held[k];
            }
        }
    }
}

// HOLDS: the block's ranks are in shared memory; else they are made anew from the weights by every walk.
template <int THREADS, bool HOLDS>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS) evict_choose_kernel(const Args a) {
    constexpr int WARPS = THREADS / 32, MINE = (1 << DIGIT) / THREADS < 4 ? 4 : (1 << DIGIT) / THREADS;  // bins of a thread
    extern __shared__ __align__(16) unsigned ranks[];
    __shared__ __align__(16) int counted[BINS];  // of each digit, in the block
    __shared__ __align__(16) int summed[BINS];   // and in the cluster
    __shared__ int warp_sums[WARPS], found[2];
    __shared__ int4 counts[WARPS];      // of each warp's slots: above the rank below `keep`, above it from `keep` on, of the rank likewise
    __shared__ __align__(16) int totals[4];  // of the block's
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int block = blockIdx.x % a.blocks, kvh = blockIdx.x / a.blocks, request = blockIdx.y, layer = blockIdx.z;
    for (int i = tid; i < BINS / 4; i += THREADS) reinterpret_cast<int4*>(counted)[i] = reinterpret_cast<int4*>(summed)[i] = make_int4(0, 0, 0, 0);
    let_next_kernel_start();
    cluster_meet(a.blocks);  // the sums are zeros everywhere
    wait_for_previous_kernels();
    const int length = length_of(a, request), head = (layer * a.requests + request) * a.kv_heads + kvh;
    if (tid == 0 && block == 0 && kvh == 0 && layer == 0) {
        a.left[request] = min(length, a.keep);
        if (a.lengths[request] > a.longest || a.lengths[request] < 0) atomicOr(a.status, HB_STATUS_BAD_POSITION);
    }
    const float* weights = a.weights + (size_t)head * a.capacity;
    const int* positions = a.positions + (size_t)head * a.capacity;
    float* to_weights = a.to_weights + (size_t)head * a.capacity;
    int* to_positions = a.to_positions + (size_t)head * a.capacity;
    const bool in_place = a.to_weights == a.weights, aligned = (((uintptr_t)weights | (uintptr_t)positions | (uintptr_t)to_weights | (uintptr_t)to_positions) & 15) == 0;
    // the block's slots, a run of looks for each warp
    const int per_warp = (length + a.blocks * WARPS * LOOK - 1) / (a.blocks * WARPS * LOOK) * LOOK, slot0 = block * WARPS * per_warp, warp0 = slot0 + warp * per_warp, warp_end = min(length, warp0 + per_warp);
    int n_moves = 0;
    if (length > a.keep) {
        const long long after = (long long)a.newest[request] - a.recent;
        // a lane's four slots; 0, which is below every rank, beyond the length
        auto fetch = [&](int slot, float (&w)[4], int (&p)[4]) {
            if (aligned && slot + 4 <= length) {
                load4(weights + slot, w);
                const int4 x = *reinterpret_cast<const int4*>(positions + slot);
                p[0] = x.x, p[1] = x.y, p[2] = x.z, p[3] = x.w;
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) w[e] = slot + e < length ? weights[slot + e] : 0.f, p[e] = slot + e < length ? positions[slot + e] : 0;
            }
        };
        auto ranked = [&](int slot, const float (&w)[4], const int (&p)[4], unsigned (&r)[4]) {
#pragma unroll
            for (int e = 0; e < 4; ++e) r[e] = slot + e < length ? rank_of(w[e], p[e], a.first, after) : 0u;
        };
        auto ranks_at = [&](int slot, unsigned (&r)[4]) {
            if (HOLDS) {
                const uint4 x = *reinterpret_cast<const uint4*>(ranks + slot - slot0);
                r[0] = x.x, r[1] = x.y, r[2] = x.z, r[3] = x.w;
            } else {
                float w[4];
                int p[4];
                fetch(slot, w, p), ranked(slot, w, p, r);
            }
        };
        constexpr int TOGETHER = 4;  // looks that are on their way together
        for (int base = warp0; base < warp_end; base += TOGETHER * LOOK) {
            float w[TOGETHER][4];
            int p[TOGETHER][4];
#pragma unroll
            for (int k = 0; k < TOGETHER; ++k)
                if (base + k * LOOK < warp_end) fetch(base + k * LOOK + 4 * lane, w[k], p[k]);
#pragma unroll
            for (int k = 0; k < TOGETHER; ++k) {
                const int slot = base + k * LOOK + 4 * lane;
                if (base + k * LOOK >= warp_end) break;
                unsigned r[4];
                ranked(slot, w[k], p[k], r);
                if (HOLDS) *reinterpret_cast<uint4*>(ranks + slot - slot0) = make_uint4(r[0], r[1], r[2], r[3]);
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (r[e]) atomicAdd(&counted[r[e] >> (32 - DIGIT)], 1);
                if (in_place || slot >= a.keep) continue;
                // what moves into a free one comes later
                if (aligned && slot + 4 <= a.keep) {
                    store4(to_weights + slot, w[k]);
                    *reinterpret_cast<int4*>(to_positions + slot) = make_int4(p[k][0], p[k][1], p[k][2], p[k][3]);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (slot + e < a.keep) to_weights[slot + e] = w[k][e], to_positions[slot + e] = p[k][e];
                }
            }
        }
        // the rank of the last that stays, and how many of that rank do
        unsigned rank = 0;
        int wanted = a.keep, digit0 = 0;
#pragma unroll 1
        for (int shift = 32 - DIGIT, bits = DIGIT;;) {
            __syncthreads();
            // a thread has MINE bins, from the highest down
            const int bins = 1 << bits, bin0 = bins - MINE - MINE * tid;
            const int* here = counted + digit0;
            if (a.blocks > 1) {
                if (bin0 >= 0) {
#pragma unroll
                    for (int k = 0; k < MINE; ++k) {
                        const int n = here[bin0 + k];
                        if (n) add_to_all(summed + digit0 + bin0 + k, n, a.blocks);
                    }
                }
                cluster_meet(a.blocks);
                here = summed + digit0;
            }
            int mine[MINE], sum = 0;
#pragma unroll
            for (int k = 0; k < MINE; k += 4) {
                const int4 x = bin0 >= 0 ? *reinterpret_cast<const int4*>(here + bin0 + k) : make_int4(0, 0, 0, 0);
                mine[k] = x.x, mine[k + 1] = x.y, mine[k + 2] = x.z, mine[k + 3] = x.w;
                sum += x.x + x.y + x.z + x.w;
            }
            const int warp_sum = __reduce_add_sync(0xffffffffu, sum);
            if (lane == 0) warp_sums[warp] = warp_sum;
            __syncthreads();
            const int those = lane < WARPS ? warp_sums[lane] : 0, before_those = warp_before(those, lane);
            const int target = __ffs(__ballot_sync(0xffffffffu, before_those + those >= wanted)) - 1;  // the warp in whose bins it is
            if (warp == target) {
                int before = __shfl_sync(0xffffffffu, before_those, target) + warp_before(sum, lane);
                if (before < wanted && before + sum >= wanted) {
#pragma unroll
                    for (int k = MINE - 1; k >= 0; --k) {
                        if (before < wanted && before + mine[k] >= wanted) found[0] = bin0 + k, found[1] = wanted - before;
                        before += mine[k];
                    }
                }
            }
            __syncthreads();
            rank |= (unsigned)found[0] << shift, wanted = found[1];
            if (shift == 0) break;
            digit0 += bins;
            bits = min(shift, DIGIT);
            const int next = shift - bits;
            for (int slot = warp0 + 4 * lane; slot < warp_end; slot += LOOK) {
                unsigned r[4];
                ranks_at(slot, r);
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (r[e] && (r[e] ^ rank) >> shift == 0) atomicAdd(&counted[digit0 + (r[e] >> next & ((1 << bits) - 1))], 1);
            }
            shift = next;
        }
        // what each warp has
        int above_low = 0, above_high = 0, equal_low = 0, equal_high = 0;
        for (int slot = warp0 + 4 * lane; slot < warp_end; slot += LOOK) {
            unsigned r[4];
            ranks_at(slot, r);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const bool low = slot + e < a.keep;
                above_low += r[e] > rank && low, above_high += r[e] > rank && !low, equal_low += r[e] == rank && low, equal_high += r[e] == rank && !low;
            }
        }
        above_low = __reduce_add_sync(0xffffffffu, above_low), above_high = __reduce_add_sync(0xffffffffu, above_high);
        equal_low = __reduce_add_sync(0xffffffffu, equal_low), equal_high = __reduce_add_sync(0xffffffffu, equal_high);
        if (lane == 0) counts[warp] = make_int4(above_low, above_high, equal_low, equal_high);
        __syncthreads();
        // What is before this warp, in the block and in the blocks before, and what there is in all.
        const int4 c = lane < WARPS ? counts[lane] : make_int4(0, 0, 0, 0);
        int4 mine{warp_before(c.x, lane), warp_before(c.y, lane), warp_before(c.z, lane), warp_before(c.w, lane)};
        if (warp == 0 && lane == 31) totals[0] = mine.x + c.x, totals[1] = mine.y + c.y, totals[2] = mine.z + c.z, totals[3] = mine.w + c.w;
        mine = make_int4(__shfl_sync(0xffffffffu, mine.x, warp), __shfl_sync(0xffffffffu, mine.y, warp), __shfl_sync(0xffffffffu, mine.z, warp), __shfl_sync(0xffffffffu, mine.w, warp));
        cluster_meet(a.blocks);
        int4 all = make_int4(0, 0, 0, 0);
        int4 x[MOST_BLOCKS];
        all_of_theirs(totals, a.blocks, x);
#pragma unroll
        for (int b = 0; b < MOST_BLOCKS; ++b) {
            if (b >= a.blocks) break;
            const int4 t = x[b];
            if (b < block) mine.x += t.x, mine.y += t.y, mine.z += t.z, mine.w += t.w;
            all.x += t.x, all.y += t.y, all.z += t.z, all.w += t.w;
        }
        // Of the slots of the rank the first `wanted` stay, and those below `keep` are the first of all.
        const int stay_low = min(all.z, wanted);
        auto stay_high = [&](int equals) { return max(0, min(all.z + equals, wanted) - stay_low); };  // of the first so many from `keep` on
        int holes = min(warp0, a.keep) - mine.x - min(mine.z, wanted), movers = mine.y + stay_high(mine.w);
        n_moves = all.y + stay_high(all.w);
        int* from = a.from + (size_t)head * a.most;
        int* to = a.to + (size_t)head * a.most;
        for (int base = warp0; base < warp_end; base += LOOK) {
            const int slot = base + 4 * lane;
            unsigned r[4];
            ranks_at(slot, r);
            bool equal = false;
#pragma unroll
            for (int e = 0; e < 4; ++e) equal |= r[e] == rank;
            int low_place = 0, high_place = 0;  // of this lane's first slot of the rank
            if (__any_sync(0xffffffffu, equal)) {
                int low_here = 0, high_here = 0;
#pragma unroll
                for (int e = 0; e < 4; ++e) low_here += r[e] == rank && slot + e < a.keep, high_here += r[e] == rank && slot + e >= a.keep;
                const int both = low_here | high_here << 16, before = warp_before(both, lane);
                low_place = mine.z + (before & 0xffff), high_place = all.z + mine.w + (before >> 16);
                const int sums = __reduce_add_sync(0xffffffffu, both);
                mine.z += sums & 0xffff, mine.w += sums >> 16;
            }
            unsigned moving = 0, empty = 0;  // of the four
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const bool low = slot + e < a.keep;
                bool stays = r[e] > rank;
                if (r[e] == rank) stays = (low ? low_place++ : high_place++) < wanted;
                moving |= (stays && !low ? 1u : 0u) << e, empty |= (low && !stays ? 1u : 0u) << e;
            }
            const int both = __popc(moving) | __popc(empty) << 16, before = warp_before(both, lane), sums = __reduce_add_sync(0xffffffffu, both);
            int at_from = movers + (before & 0xffff), at_to = holes + (before >> 16);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (moving >> e & 1) from[at_from++] = slot + e;
                if (empty >> e & 1) to[at_to++] = slot + e;
            }
            movers += sums & 0xffff, holes += sums >> 16;
        }
        cluster_meet(a.blocks);
        for (int i = block * THREADS + tid; i < n_moves; i += a.blocks * THREADS) {
            const int source = from[i], target = to[i];
            to_weights[target] = weights[source], to_positions[target] = positions[source];
        }
        if (in_place) cluster_meet(a.blocks);  // what moves has been read
    } else if (!in_place) {
        for (int slot = block * THREADS + tid; slot < length; slot += a.blocks * THREADS) to_weights[slot] = weights[slot], to_positions[slot] = positions[slot];
    }
    // what has been given up; a tally in a place of its own is written to its end
    const int left = min(length, a.keep), end = in_place ? length : a.capacity;
    for (int slot = (left & ~3) + 4 * (block * THREADS + tid); slot < end; slot += 4 * a.blocks * THREADS) {
        if (aligned && slot >= left && slot + 4 <= end) {
            *reinterpret_cast<float4*>(to_weights + slot) = make_float4(0.f, 0.f, 0.f, 0.f);
            *reinterpret_cast<int4*>(to_positions + slot) = make_int4(-1, -1, -1, -1);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (slot + e >= left && slot + e < end) to_weights[slot + e] = 0.f, to_positions[slot + e] = -1;
        }
    }
    if (a.moves_here) move_records(a, a.from + (size_t)head * a.most, a.to + (size_t)head * a.most, n_moves, a.block_table + (size_t)request * a.table_width, layer, kvh, block * WARPS + warp, a.blocks * WARPS);
    else if (tid == 0 && block == 0) a.moves[head] = n_moves;
}

// The records, where the first kernel leaves them: block (part, key/value head and request, layer).
constexpr int MOVE_THREADS = 256, PER_BLOCK = CHUNK * MOVE_THREADS / 32;
__global__ void __launch_bounds__(MOVE_THREADS) evict_move_kernel(const Args a) {
    let_next_kernel_start();
    wait_for_previous_kernels();
    const int kvh = blockIdx.y % a.kv_heads, request = blockIdx.y / a.kv_heads, layer = blockIdx.z, head = (layer * a.requests + request) * a.kv_heads + kvh;
    move_records(a, a.from + (size_t)head * a.most, a.to + (size_t)head * a.most, a.moves[head], a.block_table + (size_t)request * a.table_width, layer, kvh,
                 blockIdx.x * (MOVE_THREADS / 32) + (threadIdx.x >> 5), gridDim.x * (MOVE_THREADS / 32));
}

template <int THREADS, bool HOLDS>
int launch_choose(const Args& a, size_t shared_bytes, cudaStream_t stream) {
    const auto kernel = evict_choose_kernel<THREADS, HOLDS>;
    static std::atomic<unsigned long long> allowed{0};
    if (const cudaError_t error = allow_shared((const void*)kernel, MOST_HELD * 4, allowed)) return (int)error;
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(a.blocks * a.kv_heads, a.requests, a.layers), config.blockDim = dim3(THREADS), config.dynamicSmemBytes = shared_bytes, config.stream = stream;
    cudaLaunchAttribute attributes[2];
    attributes[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attributes[0].val.programmaticStreamSerializationAllowed = overlap_launches() ? 1 : 0;
    attributes[1].id = cudaLaunchAttributeClusterDimension;
    attributes[1].val.clusterDim = {(unsigned)a.blocks, 1, 1};
    config.attrs = attributes, config.numAttrs = 2;
    return (int)cudaLaunchKernelEx(&config, kernel, a);
}
}  // namespace

// Bytes of scratch that hb_evict takes.
HB_EXPORT long long hb_evict_scratch(int layers, int requests, int kv_heads, int longest, int keep) {
    const long long heads = (long long)layers * requests * kv_heads, most = longest - keep < keep ? longest - keep : keep;
    return heads <= 0 ? 0 : (heads * 4 + 15) / 16 * 16 + heads * 8 * (most > 0 ? most : 0);
}
// cache [layers, pages, 2, kv_heads, page_size, record_bytes]; weights, positions and to_... [layers, requests, kv_heads, capacity]; lengths, newest, left [requests], lengths at most `longest`, which
// table and capacity hold.  scratch: hb_evict_scratch bytes on a 16-byte boundary.
HB_EXPORT int hb_evict(void* cache, int layers, int pages, int kv_heads, int page_size, int record_bytes, const int* block_table, int table_width, const int* lengths, const int* newest, int requests,
                       int longest, const float* weights, const int* positions, float* to_weights, int* to_positions, int capacity, int keep, int first, int recent, int* left, void* scratch, int* status,
                       int sms, cudaStream_t stream) {
    if (requests <= 0 || layers <= 0) return 0;
    if (!cache || !block_table || !lengths || !newest || !weights || !positions || !to_weights || !to_positions || !left || !scratch || !status) return HB_BAD_ARGUMENT;
    if (pages <= 0 || kv_heads <= 0 || page_size <= 0 || (page_size & (page_size - 1)) || record_bytes <= 0 || record_bytes % 16 || table_width <= 0 || longest <= 0 || capacity < longest || keep < 1 || recent < 0 || sms <= 0)
        return HB_BAD_ARGUMENT;
    if (((uintptr_t)cache | (uintptr_t)scratch) & 15 || (long long)table_width * page_size < longest) return HB_BAD_ARGUMENT;
    const long long heads = (long long)layers * requests * kv_heads;
    if (requests > 65535 || layers > 65535 || (long long)requests * kv_heads > 65535 || heads > 0x7fffffffLL || record_bytes > 65536) return HB_UNSUPPORTED_SIZE;
    if (longest > 0x7fffffff - MOST_BLOCKS * 32 * LOOK || capacity > 0x7fffffff - 4 * MOST_BLOCKS * 1024 || (long long)kv_heads * MOST_BLOCKS > 0x7fffffffLL) return HB_UNSUPPORTED_SIZE;
    const int most = longest - keep < keep ? (longest > keep ? longest - keep : 0) : keep;
    // Clusters where heads are few and long or give up much, of four blocks while there is an SM for each, else two; eight only for a few heads, because clusters of eight SMs leave others empty.  (us, one / two / four / eight
    // blocks, 16 heads, one slot given up of 8,192 12.0 / 13.1 / 13.4 / 26.8, of 16,384 16.8 / 15.5 / 13.4 / 26.9, a quarter of 8,192 22.5 / 19.9 / 17.2 / 32.5; four heads, a quarter of 16,384 39.2 / 27.8 / 21.3 / 19.3; 64
    // heads, a quarter of 16,384 46.7 / 39.4 / 50.5.)  Blocks of 256 threads where heads are short, or more than there are SMs, which hold three to five of those (us, 256 / 1,024 threads, one slot given up of 1,000: 16 heads
    // 6.9 / 8.3, 256 heads 9.7 / 16.3, of 4,097: 256 heads 15.8 / 19.8, 16 heads 11.5 / 10.0; a quarter of 1,000: 128 heads 12.5 / 9.4, 512 heads 16.2 / 28.3, of 8,192: 512 heads 101 / 80).
    const long long size = longest + 2LL * most;
    const int blocks = size < 10240 ? 1 : size >= 24576 && heads * 16 <= sms ? 8 : heads * 4 <= sms ? 4 : heads * 2 <= sms ? 2 : 1;
    const bool few = heads * 2 <= sms, many = heads > sms;
    const int threads = longest <= (many ? 6144 : few ? 2048 : 512) && blocks == 1 ? 256 : 1024, looks = threads / 32 * LOOK;
    const size_t held = (size_t)((longest + blocks * looks - 1) / (blocks * looks)) * looks;
    int* moves = (int*)scratch;
    int* lists = (int*)((char*)scratch + (heads * 4 + 15) / 16 * 16);
    // A head's records are moved by its own blocks up to a megabyte each: 1 slot of 1,025 8.1 us against 9.7 with a second kernel, 4,096 of 32,771 by four blocks 46.2 against 48.5.
    const bool moves_here = (long long)most * 2 * record_bytes <= (long long)blocks << 20;
    const Args a{lengths, newest, requests, weights, positions, to_weights, to_positions, capacity, longest, keep, first, recent, layers, kv_heads, left, moves, lists, lists + heads * most, most,
                 (uint4*)cache, record_bytes / 16, block_table, table_width, __builtin_ctz(page_size), pages, blocks, moves_here ? 1 : 0, status};
    if (int code = threads == 256 ? launch_choose<256, true>(a, held * 4, stream) : held <= MOST_HELD ? launch_choose<1024, true>(a, held * 4, stream) : launch_choose<1024, false>(a, 0, stream)) return code;
    if (!most || moves_here) return 0;
    return launch_after_previous(evict_move_kernel, dim3((most + PER_BLOCK - 1) / PER_BLOCK, kv_heads * requests, layers), dim3(MOVE_THREADS), 0, stream, a);
}
HB_EXPORT int hb_evict_packed(const void* arguments) { return call_packed(&hb_evict, arguments); }
