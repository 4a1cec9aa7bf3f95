// Beams take over what their parents hold: beam j of a group goes on from its beam parent[j].
//
// Pages that are full are never written again, so a beam's table row points to its parent's from then on.  The page that is not full yet is each beam's own: the records that stand in the parent's are
// copied into it.  State records are copied whole.  All of a group's beams change at once, in place, and one parent may have many children: a thread owns the same 16 bytes of all beams of a group,
// reads what all of them are to have and writes it only then, so no thread reads what another writes and nothing is kept elsewhere in between.  A parent that several beams have is read from memory
// once (they follow one another), and a beam that is its own parent is neither read nor written.
//
// Bound by memory: 16 groups of 8 beams, 28 layers of part-filled pages and 4 of states, 84.9 us for the 502 MB that distinct parents and changed beams come to (5.9 TB/s, 0.90 of a copy's rate).  One group of four beams 2.6 us.
#include "common.cuh"

namespace {
constexpr int THREADS = 256, MOST_JOBS = 24, MOST_BEAMS = 32;

struct Job {
    char* base;
    long long layer, page, outer;  // bytes from a layer to the next, from a page (a row) to the next, from an outer index to the next
    int outers;
    int slot;        // bytes of a record; of state records all of them
    int states;      // 0: pages
    int width;       // bytes a thread moves at a time
    int chunks;      // blocks that an outer index of a layer takes
    int first_block; // of this job's layers * outers * chunks
};
struct Args {
    const int* parents;      // [groups, beams]
    const int* lengths;      // [groups]
    int* block_table; int table_width;
    const int* slots;        // [groups * beams]: the row of a beam's state records; null: its own number
    int slots_rows;          // rows of state records
    int beams, page_size, pages, n_jobs, table_blocks;
    Job jobs[MOST_JOBS];
    int* status;
};

// What is written in place is read past L1 (ld.global.cg): the next kernel may be on the multiprocessor by now, and a line that another one writes after it was read here would be what that kernel finds in L1, if its loads are not
// coherent ones, as those of block tables are in places.
template <typename T, int B>
__device__ __forceinline__ void move(char* const* rows, const int* parent, int beams, long long byte) {
    T value[B];
#pragma unroll
    for (int j = 0; j < B; ++j)
        if (j < beams && parent[j] != j) value[j] = __ldcg(reinterpret_cast<const T*>(rows[parent[j]] + byte));
#pragma unroll
    for (int j = 0; j < B; ++j)
        if (j < beams && parent[j] != j) *reinterpret_cast<T*>(rows[j] + byte) = value[j];
}

template <int B>
__global__ void __launch_bounds__(THREADS) beam_reorder_kernel(const __grid_constant__ Args a) {
    __shared__ int parent[MOST_BEAMS];
    __shared__ char* rows[MOST_BEAMS];
    const int tid = threadIdx.x, group = blockIdx.y, beams = a.beams;
    let_next_kernel_start();
    wait_for_previous_kernels();
    const int length = max(a.lengths ? a.lengths[group] : 0, 0), full = a.page_size ? length / a.page_size : 0, filled = a.page_size ? length - full * a.page_size : 0;
    if (tid < beams) {
        int p = a.parents[group * beams + tid];
        if (p >= beams) {
            if (blockIdx.x == 0) atomicOr(a.status, HB_STATUS_BAD_POSITION);
            p = -1;
        }
        parent[tid] = p < 0 ? tid : p;
    }
    if ((int)blockIdx.x < a.table_blocks) {
        if (tid == 0 && blockIdx.x == 0 && (full > a.table_width || (filled && full >= a.table_width))) atomicOr(a.status, HB_STATUS_BAD_POSITION);
        if (tid < beams) rows[tid] = reinterpret_cast<char*>(a.block_table + (size_t)(group * beams + tid) * a.table_width);
        __syncthreads();
        const int column = blockIdx.x * THREADS + tid;
        if (column < min(full, a.table_width)) move<int, B>(rows, parent, beams, column * 4LL);
        return;
    }
    const int block = blockIdx.x - a.table_blocks;
    int which = 0;
    while (which + 1 < a.n_jobs && block >= a.jobs[which + 1].first_block) ++which;
    const Job& job = a.jobs[which];
    const int at = block - job.first_block, chunk = at % job.chunks, outer = at / job.chunks % job.outers, layer = at / job.chunks / job.outers;
    const long long bytes = job.states ? job.slot : (long long)filled * job.slot, byte = ((long long)chunk * THREADS + tid) * job.width;
    if ((long long)chunk * THREADS * job.width >= bytes) return;
    if (tid < beams) {
        const int beam = group * beams + tid;
        int place;
        if (job.states) {
            place = a.slots ? a.slots[beam] : beam;
            if (place < 0 || place >= a.slots_rows) atomicOr(a.status, HB_STATUS_BAD_POSITION), place = -1;
        } else {
            place = full < a.table_width ? __ldcg(a.block_table + (size_t)beam * a.table_width + full) : -1;
            if (place < 0 || place >= a.pages) atomicOr(a.status, HB_STATUS_BAD_PAGE), place = -1;
        }
        rows[tid] = place < 0 ? nullptr : job.base + layer * job.layer + place * job.page + outer * job.outer;
    }
    __syncthreads();
    if (tid < 32) {  // a beam without a place, or whose parent has none, stays as it is
        const bool lost = tid < beams && (!rows[tid] || !rows[parent[tid]]);
        __syncwarp();
        if (lost) parent[tid] = tid;
    }
    __syncthreads();
    if (byte >= bytes) return;
    switch (job.width) {
        case 16: move<uint4, B>(rows, parent, beams, byte); break;
        case 4: move<unsigned, B>(rows, parent, beams, byte); break;
        default: move<unsigned char, B>(rows, parent, beams, byte);
    }
}
}  // namespace

// One tensor of pages or of state records, as hb_beam_reorder takes it: `base`, and [layers, pages or rows, outers, slots of a page (1 of a state), bytes of a slot], dense.
struct BeamTensor {
    void* base;
    long long layers, places, outers, slots, bytes, states;
};
// parents [groups, beams]; lengths [groups]; block_table [groups * beams, table_width], or null without pages; rows: [groups * beams] rows of the state records, or null.
HB_EXPORT int hb_beam_reorder(const int* parents, const int* lengths, int groups, int beams, int* block_table, int table_width, int page_size, const BeamTensor* tensors, int n_tensors, const int* slots,
                              int* status, cudaStream_t stream) {
    if (groups <= 0 || beams <= 0) return 0;
    if (!parents || !status || (block_table && (!lengths || table_width <= 0 || page_size <= 0)) || (n_tensors && !tensors)) return HB_BAD_ARGUMENT;
    if (beams > MOST_BEAMS || n_tensors > MOST_JOBS || groups > 65535) return HB_UNSUPPORTED_SIZE;
    Args a = {};
    a.parents = parents, a.lengths = lengths, a.block_table = block_table, a.table_width = table_width, a.slots = slots, a.beams = beams, a.page_size = block_table ? page_size : 0, a.status = status;
    a.table_blocks = block_table ? (table_width + THREADS - 1) / THREADS : 0;
    long long blocks = 0;
    for (int i = 0; i < n_tensors && beams > 1; ++i) {  // a beam alone has no other parent: there is nothing to move
        const BeamTensor& t = tensors[i];
        if (t.layers <= 0 || t.outers <= 0 || t.bytes <= 0) continue;
        if (!t.base || t.places <= 0 || t.slots <= 0 || (!t.states && (!block_table || t.slots != page_size))) return HB_BAD_ARGUMENT;
        if (t.places > 0x7fffffffLL || t.bytes > 0x7fffffffLL || t.outers > 0x7fffffffLL) return HB_UNSUPPORTED_SIZE;
        Job& job = a.jobs[a.n_jobs];
        job.outer = t.slots * t.bytes, job.page = t.outers * job.outer, job.layer = t.places * job.page;
        job.base = (char*)t.base, job.outers = (int)t.outers, job.slot = (int)t.bytes, job.states = (int)t.states;
        const unsigned long long bits = (uintptr_t)t.base | (unsigned long long)t.bytes;
        job.width = bits % 16 == 0 ? 16 : bits % 4 == 0 ? 4 : 1;
        const long long chunks = (job.outer + THREADS * job.width - 1) / (THREADS * job.width);
        job.chunks = (int)chunks, job.first_block = (int)blocks;
        blocks += t.layers * t.outers * chunks;
        if (blocks > 0x7fffffffLL - a.table_blocks) return HB_UNSUPPORTED_SIZE;
        if (job.states) {
            if (a.slots_rows && a.slots_rows != t.places) return HB_BAD_ARGUMENT;
            a.slots_rows = (int)t.places;
        } else {
            if (a.pages && a.pages != t.places) return HB_BAD_ARGUMENT;
            a.pages = (int)t.places;
        }
        ++a.n_jobs;
    }
    if (blocks + a.table_blocks == 0) a.table_blocks = 1;  // parents are looked at in any case
    const auto kernel = beams <= 4 ? beam_reorder_kernel<4> : beams <= 8 ? beam_reorder_kernel<8> : beams <= 16 ? beam_reorder_kernel<16> : beam_reorder_kernel<32>;
    return launch_after_previous(kernel, dim3((unsigned)(blocks + a.table_blocks), groups), dim3(THREADS), 0, stream, a);
}
HB_EXPORT int hb_beam_reorder_packed(const void* arguments) { return call_packed(&hb_beam_reorder, arguments); }
