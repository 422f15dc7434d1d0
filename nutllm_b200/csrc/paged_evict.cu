/* Eviction from the paged KV cache by accumulated attention weight
 * (nut_paged_evict).
 *
 * Of n slots the m = min(n, budget) with the greatest key stay, the key
 * being the weight, or infinity for protected positions (which an infinite
 * weight therefore ties with).  Slots below m
 * that lose their token (holes) and slots from m on that keep it (sources)
 * are equally many; the i-th source moves into the i-th hole.  So only the
 * tokens that must move do: at most min(m, n - m) of them, where packing the
 * kept ones in order would move nearly all m.
 * The first kernel finds the threshold, lists the pairs and moves the weights
 * and positions: 23 us for 512 (sequence, head)s of up to 5,000 slots, bound
 * by the barriers between its passes.  move_kernel moves keys and values: 48
 * us for their 207 MB of 256-byte rows, 4.3 TB/s out of and into DRAM.
 */
#include <algorithm>
#include <cstdint>
#include <cuda_runtime.h>

#include "paged.cuh"
#include "paged_choose.cuh"

namespace nut {
namespace {

struct SlotKeys {
    const float *weights;
    const int32_t *positions;
    int sinks;
    int64_t recent_from;
    template <int N> __device__ __forceinline__ void own(int i, int there, uint32_t (&k)[N]) const {
        float w[N];
        int32_t at[N];
        load_own(weights + i, there, w);
        if (positions)
            load_own(positions + i, there, at);
#pragma unroll
        for (int e = 0; e < N; e++) {
            k[e] = w[e] != w[e] ? 0u : ordered_bits(w[e]);
            if (positions && (at[e] < sinks || at[e] >= recent_from))
                k[e] = ordered_bits(INFINITY);
            if (e >= there)
                k[e] = 0u;
        }
    }
};

/* What both forms of the choice know of an item. */
struct SlotItem {
    int length, m;      /* slots now, slots to keep */
    bool bad;           /* the length is not one the table can hold */
    int64_t item, at;   /* its number, its first slot in the arrays */
    int32_t *holes, *sources;
    SlotKeys key;
    __device__ SlotItem(const PagedEvict &a, int s, int head) {
        const PagedPool &p = a.p;
        length = checked_length(p, p.lengths[s]);
        bad = length != p.lengths[s];
        m = min(length, a.budget);
        item = int64_t(s) * p.kv_heads + head;
        at = item * p.capacity;
        holes = a.pairs + at;
        sources = holes + p.capacity / 2;
        key = SlotKeys{a.weights + at, a.positions ? a.positions + at : nullptr, a.sinks,
                       a.recent ? int64_t(a.seen[s]) - a.recent : INT64_MAX};
    }
};

/* What forbids to trim a sequence: a bad length, or, where tokens will move, a
 * page outside the pool.  Such a sequence is left as it is (counts of 0 and
 * -1).  `me` of `threads` threads has its first page on the way from the
 * start (0.5 us of a choice among few). */
struct Pages {
    int s, me, threads, end, first;
    __device__ __forceinline__ Pages(const PagedPool &p, const SlotItem &x, int s_, int me_, int threads_)
        : s(s_), me(me_), threads(threads_), end(x.m < x.length ? (x.length - 1) / p.page_size + 1 : 0), first(0) {
        if (me < end)
            first = p.table[int64_t(s) * p.max_pages + me];
    }
    __device__ __forceinline__ bool forbid(const PagedPool &p, const SlotItem &x) const {
        bool bad = unsigned(first) >= unsigned(p.n_pages);
        for (int j = me + threads; j < end; j += threads)
            bad |= lookup(p, s, j) < 0;
        if (bad)
            paged_fail(p, kPagedBadPage);
        return bad || x.bad;
    }
};
__device__ __forceinline__ void leave(const PagedEvict &a, const SlotItem &x) {
    a.counts[x.item * 2] = 0;
    a.counts[x.item * 2 + 1] = -1;
}

/* The slots i0 .. i0 + there - 1 as holes (to be filled) and sources. */
__device__ __forceinline__ void holes_and_sources(uint32_t kept, int i0, int there, int m, uint32_t &hole,
                                                  uint32_t &source) {
    const uint32_t low = (1u << max(0, min(there, m - i0))) - 1u; /* those below m */
    hole = low & ~kept;
    source = kept & ~low;
}

__device__ __forceinline__ void list_slots(uint32_t mask, int i0, int32_t *to) {
    for (; mask; mask &= mask - 1)
        *to++ = i0 + __ffs(mask) - 1;
}

/* Weights and positions of slots i, or an empty slot's. */
__device__ __forceinline__ void keep_slot(const PagedEvict &a, int64_t to, int64_t from) {
    a.weights_out[to] = a.weights[from];
    if (a.positions)
        a.positions_out[to] = a.positions[from];
}
__device__ __forceinline__ void clear_slot(const PagedEvict &a, int64_t at) {
    a.weights_out[at] = 0.0f;
    if (a.positions)
        a.positions_out[at] = -1;
}

/* Up to N * kChooseThreads slots: a block for each sequence and kv head,
 * all keys in registers. */
template <int N>
__global__ void __launch_bounds__(kChooseThreads)
    choose_few_slots_kernel(const __grid_constant__ PagedEvict a) {
    __shared__ ChooseScratch scratch;
    begin_kernel();
    const SlotItem x(a, blockIdx.y, blockIdx.x);
    const int tid = threadIdx.x, i0 = tid * N, there = max(0, min(N, x.length - i0));
    uint32_t k[N], threshold;
    const Pages pages(a.p, x, blockIdx.y, tid, kChooseThreads);
    x.key.own(i0, there, k);
    int quota, total;
    choose_largest<1>(x.key, x.length, x.length, x.m, k, scratch, threshold, quota);
    /* counted with the ties, below 2^14 of them */
    int ties = int(pages.forbid(a.p, x)) << 16;
#pragma unroll
    for (int e = 0; e < N; e++)
        ties += e < there && k[e] == threshold;
    int rank = block_before(ties, scratch, 0, total) & 0xffff;
    if (total >> 16) {
        if (tid == 0)
            leave(a, x);
        return;
    }
    uint32_t kept = 0, hole, source;
#pragma unroll
    for (int e = 0; e < N; e++)
        if (e < there && (k[e] > threshold || (k[e] == threshold && rank++ < quota)))
            kept |= 1u << e;
    holes_and_sources(kept, i0, there, x.m, hole, source);
    /* holes and sources in one scan: below 2^15 of each */
    const int before = block_before(__popc(hole) | (__popc(source) << 16), scratch, 1, total);
    list_slots(hole, i0, x.holes + (before & 0xffff));
    list_slots(source, i0, x.sources + (before >> 16));
    const int pairs = total & 0xffff;
    if (tid == 0) {
        a.counts[x.item * 2] = pairs;
        a.counts[x.item * 2 + 1] = x.m;
    }
    /* kept slots first: a hole's own entry is overwritten after */
    if (a.weights_out != a.weights || a.positions_out != a.positions)
        for (int i = tid; i < x.m; i += kChooseThreads)
            keep_slot(a, x.at + i, x.at + i);
    __syncthreads();
    for (int i = tid; i < pairs; i += kChooseThreads)
        keep_slot(a, x.at + x.holes[i], x.at + x.sources[i]);
    __syncthreads();
    for (int i = x.m + tid; i < x.length; i += kChooseThreads)
        clear_slot(a, x.at + i);
}

/* Any number of slots: a cluster of kBlocks blocks for each sequence and kv
 * head, each with a run of the slots, whose keys are read and made anew in
 * each of six passes.  For tables that the other form's registers do not hold:
 * 64 sequences of up to 8,300 slots, 8 heads, take 328 us where the other form
 * takes 33 for 8,192; 16 of up to 40,000 take 117. */
constexpr int kBlocks = 8;

__global__ void __launch_bounds__(kChooseThreads)
    choose_slots_kernel(const __grid_constant__ PagedEvict a) {
    __shared__ ChooseScratch scratch;
    begin_kernel();
    const int rank = int(blockIdx.x) % kBlocks, tid = threadIdx.x;
    const SlotItem x(a, blockIdx.y, int(blockIdx.x) / kBlocks);
    const Pages pages(a.p, x, blockIdx.y, rank * kChooseThreads + tid, kBlocks * kChooseThreads);
    if (tid == 0)
        scratch.shared[3] = 0;
    const int run = (x.length + kBlocks * kOwn - 1) / (kBlocks * kOwn) * kOwn; /* whole groups of kOwn */
    const int from = min(rank * run, x.length), n = min(run, x.length - from);
    SlotKeys key = x.key;
    key.weights += from;
    key.positions += key.positions ? from : 0;
    uint32_t first[kOwn], threshold;
    int quota, total, all;
    own_keys(key, 0, n, first);
    choose_largest<kBlocks>(key, n, x.length, x.m, first, scratch, threshold, quota);

    auto ties_in = [&](int base, const uint32_t(&k)[kOwn]) {
        int ties = 0;
#pragma unroll
        for (int e = 0; e < kOwn; e++)
            ties += base + tid * kOwn + e < n && k[e] == threshold;
        return ties;
    };
    /* walks this block's slots: each(holes, sources, first slot) */
    int ties_before = 0;
    auto walk = [&](auto each) {
        int ties = ties_before;
        for (int base = 0; base < n; base += kChooseChunk) {
            uint32_t k[kOwn], kept = 0, hole, source;
            own_keys(key, base, n, k);
            int tie_rank = ties + block_before(ties_in(base, k), scratch, 0, total);
            ties += total;
            const int i0 = base + tid * kOwn, there = max(0, min(kOwn, n - i0));
#pragma unroll
            for (int e = 0; e < kOwn; e++)
                if (e < there && (k[e] > threshold || (k[e] == threshold && tie_rank++ < quota)))
                    kept |= 1u << e;
            holes_and_sources(kept, from + i0, there, x.m, hole, source);
            each(hole, source, from + i0);
            __syncthreads(); /* the scan's scratch is free again */
        }
    };
    /* ties, holes and sources in the blocks before this one */
    int mine = 0, holes_n, sources_n, pairs;
    for (int base = 0; base < n; base += kChooseChunk) {
        uint32_t k[kOwn];
        own_keys(key, base, n, k);
        mine += ties_in(base, k);
    }
    block_before(mine, scratch, 0, total);
    if (pages.forbid(a.p, x))
        scratch.shared[3] = 1;
    cluster_before<kBlocks>(total, scratch, 0, ties_before, all);
    /* read behind the same barrier of the cluster */
    int forbidden = 0;
#pragma unroll
    for (int b = 0; b < kBlocks; b++)
        forbidden |= *cooperative_groups::this_cluster().map_shared_rank(&scratch.shared[3], b);
    if (forbidden) {
        if (rank == 0 && tid == 0)
            leave(a, x);
        cooperative_groups::this_cluster().sync(); /* shared memory done with */
        return;
    }
    int holes_here = 0, sources_here = 0;
    walk([&](uint32_t hole, uint32_t source, int) {
        holes_here += __popc(hole);
        sources_here += __popc(source);
    });
    block_before(holes_here, scratch, 1, total);
    cluster_before<kBlocks>(total, scratch, 1, holes_n, pairs);
    __syncthreads();
    block_before(sources_here, scratch, 1, total);
    cluster_before<kBlocks>(total, scratch, 2, sources_n, all);
    __syncthreads();
    walk([&](uint32_t hole, uint32_t source, int i0) {
        const int before = block_before(__popc(hole) | (__popc(source) << 16), scratch, 1, total);
        list_slots(hole, i0, x.holes + holes_n + (before & 0xffff));
        list_slots(source, i0, x.sources + sources_n + (before >> 16));
        holes_n += total & 0xffff;
        sources_n += total >> 16;
    });
    if (rank == 0 && tid == 0) {
        a.counts[x.item * 2] = pairs;
        a.counts[x.item * 2 + 1] = x.m;
    }
    /* kept slots first: a hole's own entry is overwritten after */
    const int whole = kBlocks * kChooseThreads, me = rank * kChooseThreads + tid;
    if (a.weights_out != a.weights || a.positions_out != a.positions)
        for (int i = me; i < x.m; i += whole)
            keep_slot(a, x.at + i, x.at + i);
    __threadfence();
    cooperative_groups::this_cluster().sync();
    for (int i = me; i < pairs; i += whole)
        keep_slot(a, x.at + x.holes[i], x.at + x.sources[i]);
    cooperative_groups::this_cluster().sync(); /* sources read, and shared memory done with */
    for (int i = x.m + me; i < x.length; i += whole)
        clear_slot(a, x.at + i);
}

/* Keys and values of the pairs: a group of row16 threads moves a row of
 * row16 16-byte pieces.  One pair at a time: with 2, 4 and 8 in flight in a
 * thread the rows in flight on the chip lie further apart, and the batch took
 * 53, 59 and 85 us where this took 51 (48 by now). */
constexpr int kMoveThreads = 256;

__global__ void __launch_bounds__(kMoveThreads) move_kernel(const __grid_constant__ PagedEvict a, int row16) {
    const PagedPool &p = a.p;
    const int head = blockIdx.y, s = blockIdx.z;
    const int64_t item = int64_t(s) * p.kv_heads + head;
    begin_kernel();
    const int n = a.counts[item * 2];
    const int left = a.counts[item * 2 + 1];
    if (blockIdx.x == 0 && head == 0 && threadIdx.x == 0 && left >= 0)
        a.new_lengths[s] = left;
    const int32_t *holes = a.pairs + item * p.capacity, *sources = holes + p.capacity / 2;
    const int groups = kMoveThreads / row16, group = threadIdx.x / row16, piece = threadIdx.x % row16;
    if (group >= groups)
        return;
    const int ps = p.page_size;
    const int64_t unit = p.type == 0 ? 4 : 2;
    char *keys = static_cast<char *>(p.keys) + int64_t(head) * p.head_stride * unit + piece * 16;
    char *values = static_cast<char *>(p.values) + int64_t(head) * p.head_stride * unit + piece * 16;
    for (int i = blockIdx.x * groups + group; i < n; i += gridDim.x * groups) {
        const int to = holes[i], from = sources[i];
        const int page_to = checked_page(p, s, to / ps), page_from = checked_page(p, s, from / ps);
        if (page_to < 0 || page_from < 0)
            continue;
        const int64_t src = (page_from * p.page_stride + from % ps * p.slot_stride) * unit;
        const int64_t dst = (page_to * p.page_stride + to % ps * p.slot_stride) * unit;
        const uint4 k = *reinterpret_cast<const uint4 *>(keys + src);
        const uint4 v = *reinterpret_cast<const uint4 *>(values + src);
        *reinterpret_cast<uint4 *>(keys + dst) = k;
        *reinterpret_cast<uint4 *>(values + dst) = v;
    }
}

} // namespace

cudaError_t paged_evict(const PagedEvict &a, cudaStream_t s) {
    const PagedPool &p = a.p;
    /* keys a thread holds: no more than the table needs (12 instead of 16 for
     * 5,000 slots leaves room for another block on the SM: 23 against 26 us;
     * beyond 6,144 slots 16 are needed: 29 us for 6,200, 33 for 8,192) */
    const dim3 all(p.kv_heads, p.sequences);
    const int each = (p.capacity + kChooseThreads - 1) / kChooseThreads;
    const cudaError_t e =
        each <= 4    ? launch_kernel(choose_few_slots_kernel<4>, all, kChooseThreads, 0, s, 1, a)
        : each <= 8  ? launch_kernel(choose_few_slots_kernel<8>, all, kChooseThreads, 0, s, 1, a)
        : each <= 12 ? launch_kernel(choose_few_slots_kernel<12>, all, kChooseThreads, 0, s, 1, a)
        : each <= 16 ? launch_kernel(choose_few_slots_kernel<16>, all, kChooseThreads, 0, s, 1, a)
                     : launch_kernel(choose_slots_kernel, dim3(kBlocks * p.kv_heads, p.sequences), kChooseThreads,
                                     0, s, kBlocks, a);
    if (e != cudaSuccess)
        return e;
    const int row16 = p.head_dim * (p.type == 0 ? 4 : 2) / 16;
    /* blocks of an item: enough for all SMs together, no more than its pairs can feed */
    const int items = p.kv_heads * p.sequences, groups = kMoveThreads / row16;
    const int most = (p.capacity / 2 + groups - 1) / groups;
    const int blocks = std::max(1, std::min(most, std::max(8, 2048 / items)));
    return launch_kernel(move_kernel, dim3(blocks, p.kv_heads, p.sequences), kMoveThreads, 0, s, 1, a, row16);
}

} // namespace nut
