// A cache is cut back to a budget: of each key/value head of a request (and layer) the `keep` slots that weigh most stay, and move into the first `keep` slots.
//
// A slot ranks by its weight, a NaN as -infinity; one whose position is below `first` or among the last `recent` ones ranks as +infinity.  Of equal ranks the lowest slots stay.  What stays in the
// first `keep` slots is not moved; the i-th of the others that stay goes into the i-th slot that is left free.  Keys were rotated when they were stored, so attention does not ask in which slot one
// stands, and the positions go along with them.  Sources stand at `keep` and beyond, targets below, so nothing is read that has been written, in whatever order the records move.
//
// A request of at most `keep` slots stays as it is.
//
// The first kernel has a block per head: the rank of the last slot that stays is found digit by digit (8 bits of the weight's ordered bits at a time, by counting), then one walk along the slots lists
// what moves and what is free and writes the slots' new weights and positions.  The second moves the records.
#include "common.cuh"

namespace {
constexpr int THREADS = 1024, WARPS = THREADS / 32;

struct Args {
    const int* lengths; const int* newest; int requests;
    const float* weights; const int* positions;  // [layers, requests, kv_heads, capacity]
    float* to_weights; int* to_positions;        // likewise; may be the same
    int capacity, longest, keep, first, recent;
    int layers, kv_heads;
    int* left;           // [requests]: min(length, keep)
    int* moves;          // [layers * requests * kv_heads]
    int2* lists;         // [layers * requests * kv_heads, most]: (from, to)
    int most;            // moves of a head: min(keep, longest - keep)
    uint4* cache;        // [layers, pages, 2, kv_heads, page, record]
    int record;          // 16-byte pieces of a record
    const int* block_table; int table_width;
    int page_shift, pages;
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

// How many of the threads before this one say yes, and how many do in all.  Every thread calls it; `counts` holds WARPS + 1 words.
__device__ __forceinline__ int before_me(bool yes, int& all, int* counts) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const unsigned said = __ballot_sync(0xffffffffu, yes);
    __syncthreads();
    if (lane == 0) counts[warp] = __popc(said);
    __syncthreads();
    const int mine = counts[lane];
    int end = mine;
#pragma unroll
    for (int offset = 1; offset < 32; offset <<= 1) {
        const int other = __shfl_up_sync(0xffffffffu, end, offset);
        if (lane >= offset) end += other;
    }
    all = __shfl_sync(0xffffffffu, end, 31);
    return __shfl_sync(0xffffffffu, end - mine, warp) + __popc(said & ((1u << lane) - 1));
}

__global__ void __launch_bounds__(THREADS) evict_choose_kernel(const Args a) {
    __shared__ int histogram[256], counts[WARPS + 1], found[2];
    const int tid = threadIdx.x, kvh = blockIdx.x, request = blockIdx.y, layer = blockIdx.z;
    let_next_kernel_start();
    wait_for_previous_kernels();
    const int length = length_of(a, request), head = (layer * a.requests + request) * a.kv_heads + kvh;
    if (tid == 0 && kvh == 0 && layer == 0) {
        a.left[request] = min(length, a.keep);
        if (a.lengths[request] > a.longest || a.lengths[request] < 0) atomicOr(a.status, HB_STATUS_BAD_POSITION);
    }
    const float* weights = a.weights + (size_t)head * a.capacity;
    const int* positions = a.positions + (size_t)head * a.capacity;
    float* to_weights = a.to_weights + (size_t)head * a.capacity;
    int* to_positions = a.to_positions + (size_t)head * a.capacity;
    const bool in_place = a.to_weights == a.weights;
    const long long after = (long long)a.newest[request] - a.recent;
    int n_moves = 0;
    if (length > a.keep) {
        // the rank of the last that stays, and how many of that rank do
        unsigned rank = 0;
        int wanted = a.keep;
        for (int shift = 24; shift >= 0; shift -= 8) {
            for (int i = tid; i < 256; i += THREADS) histogram[i] = 0;
            __syncthreads();
            const unsigned above = shift == 24 ? 0u : 0xffffffffu << (shift + 8);
            for (int slot = tid; slot < length; slot += THREADS) {
                const unsigned r = rank_of(weights[slot], positions[slot], a.first, after);
                if ((r & above) == rank) atomicAdd(&histogram[(r >> shift) & 255], 1);
            }
            __syncthreads();
            if (tid == 0) {
                int digit = 255, left = wanted;
                while (digit > 0 && histogram[digit] < left) left -= histogram[digit--];
                found[0] = digit, found[1] = left;
            }
            __syncthreads();
            rank |= (unsigned)found[0] << shift, wanted = found[1];
        }
        int2* list = a.lists + (size_t)head * a.most;
        int equals = 0, holes = 0;
        for (int base = 0; base < length; base += THREADS) {
            const int slot = base + tid;
            const unsigned r = slot < length ? rank_of(weights[slot], positions[slot], a.first, after) : 0u;
            int all;
            const int mine = before_me(slot < length && r == rank, all, counts);
            const bool stays = slot < length && (r > rank || (r == rank && equals + mine < wanted));
            equals += all;
            const bool moves = stays && slot >= a.keep, hole = slot < a.keep && !stays;
            int at = before_me(moves, all, counts);
            if (moves) list[n_moves + at].x = slot;
            n_moves += all;
            at = before_me(hole, all, counts);
            if (hole) list[holes + at].y = slot;
            holes += all;
        }
        __syncthreads();
        for (int i = tid; i < n_moves; i += THREADS) {
            const int2 move = list[i];
            to_weights[move.y] = weights[move.x], to_positions[move.y] = positions[move.x];
        }
        if (!in_place) {
            // those that stay where they are: all of the first slots that are no target
            int equals = 0;
            for (int base = 0; base < a.keep; base += THREADS) {
                const int slot = base + tid;
                const unsigned r = slot < a.keep ? rank_of(weights[slot], positions[slot], a.first, after) : 0u;
                int all;
                const int mine = before_me(slot < a.keep && r == rank, all, counts);
                if (slot < a.keep && (r > rank || (r == rank && equals + mine < wanted))) to_weights[slot] = weights[slot], to_positions[slot] = positions[slot];
                equals += all;
            }
        }
    } else if (!in_place) {
        for (int slot = tid; slot < length; slot += THREADS) to_weights[slot] = weights[slot], to_positions[slot] = positions[slot];
    }
    __syncthreads();
    for (int slot = min(length, a.keep) + tid; slot < a.capacity; slot += THREADS) to_weights[slot] = 0.f, to_positions[slot] = -1;
    if (tid == 0) a.moves[head] = n_moves;
}

// A key's and a value's record a group of lanes; block x takes the moves from x * PER_BLOCK on.
constexpr int MOVE_THREADS = 256, PER_BLOCK = 64;
__global__ void __launch_bounds__(MOVE_THREADS) evict_move_kernel(const Args a) {
    let_next_kernel_start();
    wait_for_previous_kernels();
    const int kvh = blockIdx.y % a.kv_heads, request = blockIdx.y / a.kv_heads, layer = blockIdx.z, head = (layer * a.requests + request) * a.kv_heads + kvh;
    const int first = blockIdx.x * PER_BLOCK, n = min(a.moves[head] - first, PER_BLOCK);
    const int2* list = a.lists + (size_t)head * a.most + first;
    const int* table = a.block_table + (size_t)request * a.table_width;
    const int mask = (1 << a.page_shift) - 1;
    for (int at = threadIdx.x; at < n * 2 * a.record; at += MOVE_THREADS) {
        const int move = at / (2 * a.record), piece = at - move * 2 * a.record, which = piece >= a.record;
        const int2 slots = list[move];
        const int from = table[slots.x >> a.page_shift], to = table[slots.y >> a.page_shift];
        if (from < 0 || from >= a.pages || to < 0 || to >= a.pages) {
            atomicOr(a.status, HB_STATUS_BAD_PAGE);
            continue;
        }
        auto place = [&](int page, int slot) { return ((((size_t)layer * a.pages + page) * 2 + which) * a.kv_heads + kvh << a.page_shift) + (slot & mask); };
        a.cache[place(to, slots.y) * a.record + piece - which * a.record] = a.cache[place(from, slots.x) * a.record + piece - which * a.record];
    }
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
                       cudaStream_t stream) {
    if (requests <= 0 || layers <= 0) return 0;
    if (!cache || !block_table || !lengths || !newest || !weights || !positions || !to_weights || !to_positions || !left || !scratch || !status) return HB_BAD_ARGUMENT;
    if (pages <= 0 || kv_heads <= 0 || page_size <= 0 || (page_size & (page_size - 1)) || record_bytes <= 0 || record_bytes % 16 || table_width <= 0 || longest <= 0 || capacity < longest || keep < 1 || recent < 0)
        return HB_BAD_ARGUMENT;
    if (((uintptr_t)cache | (uintptr_t)scratch) & 15 || (long long)table_width * page_size < longest) return HB_BAD_ARGUMENT;
    const long long heads = (long long)layers * requests * kv_heads;
    if (requests > 65535 || layers > 65535 || (long long)requests * kv_heads > 65535 || heads > 0x7fffffffLL || longest > 0x7fffffff - THREADS || record_bytes > 65536) return HB_UNSUPPORTED_SIZE;
    const int most = longest - keep < keep ? (longest > keep ? longest - keep : 0) : keep;
    int* moves = (int*)scratch;
    const Args a{lengths, newest, requests, weights, positions, to_weights, to_positions, capacity, longest, keep, first, recent, layers, kv_heads, left, moves,
                 (int2*)((char*)scratch + (heads * 4 + 15) / 16 * 16), most, (uint4*)cache, record_bytes / 16, block_table, table_width, __builtin_ctz(page_size), pages, status};
    if (int code = launch_after_previous(evict_choose_kernel, dim3(kv_heads, requests, layers), dim3(THREADS), 0, stream, a)) return code;
    if (!most) return 0;
    return launch_after_previous(evict_move_kernel, dim3((most + PER_BLOCK - 1) / PER_BLOCK, kv_heads * requests, layers), dim3(MOVE_THREADS), 0, stream, a);
}
