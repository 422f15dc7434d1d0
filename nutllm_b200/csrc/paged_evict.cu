/* Eviction from the paged KV cache by accumulated attention weight
 * (nut_paged_evict).
 *
 * Of n slots the m = min(n, budget) with the greatest key stay, the key
 * being the weight, or infinity for protected positions.  Slots below m
 * that lose their token (holes) and slots from m on that keep it (sources)
 * are equally many; the i-th source moves into the i-th hole.  So only the
 * tokens that must move do: at most min(m, n - m) of them, where packing the
 * kept ones in order would move nearly all m.
 * choose_slots_kernel finds the threshold, lists the pairs and moves the
 * weights and positions; move_kernel moves keys and values.
 */
#include <algorithm>
#include <cstdint>
#include <cuda_runtime.h>

#include "kernels.h"
#include "paged.cuh"
#include "paged_choose.cuh"

namespace nut {
namespace {

struct SlotKeys {
    const float *weights;
    const int32_t *positions;
    int sinks;
    int64_t recent_from;
    __device__ __forceinline__ void own(int i, int there, uint32_t (&k)[kOwn]) const {
        float w[kOwn];
        int32_t at[kOwn];
        load_own(weights + i, there, w);
        if (positions)
            load_own(positions + i, there, at);
#pragma unroll
        for (int e = 0; e < kOwn; e++) {
            k[e] = w[e] != w[e] ? 0u : ordered_bits(w[e]);
            if (positions && (at[e] < sinks || at[e] >= recent_from))
                k[e] = ordered_bits(INFINITY);
            if (e >= there)
                k[e] = 0u;
        }
    }
};

/* kBlocks blocks (a cluster) for each sequence and kv head, each with a run
 * of the slots. */
template <int kBlocks>
__global__ void __launch_bounds__(kChooseThreads)
    choose_slots_kernel(const __grid_constant__ PagedEvict a) {
    __shared__ ChooseScratch scratch;
    const PagedPool &p = a.p;
    const int rank = int(blockIdx.x) % kBlocks, head = int(blockIdx.x) / kBlocks, s = blockIdx.y;
    const int tid = threadIdx.x;
    const int length = checked_length(p, p.lengths[s]), m = min(length, a.budget);
    /* runs of whole groups of kOwn slots */
    const int run = (length + kBlocks * kOwn - 1) / (kBlocks * kOwn) * kOwn;
    const int from = min(rank * run, length), n = min(run, length - from);
    const int64_t item = int64_t(s) * p.kv_heads + head, at = item * p.capacity;
    const float *w = a.weights + at + from;
    const int32_t *pos = a.positions ? a.positions + at + from : nullptr;
    const int64_t recent_from = a.recent ? int64_t(a.seen[s]) - a.recent : INT64_MAX;
    const SlotKeys key{w, pos, a.sinks, recent_from};
    uint32_t first[kOwn], threshold;
    int quota;
    own_keys(key, 0, n, first);
    choose_largest<kBlocks>(key, n, length, m, first, scratch, threshold, quota);

    /* ties, holes and sources of the blocks before this one */
    int ties = 0, holes_n = 0, sources_n = 0;
    int32_t *holes = a.pairs + at, *sources = holes + p.capacity / 2;
    if constexpr (kBlocks > 1) {
        int mine = 0, total, all;
        for (int base = 0; base < n; base += kChooseChunk) {
            uint32_t k[kOwn];
            own_keys(key, base, n, k);
#pragma unroll
            for (int e = 0; e < kOwn; e++)
                mine += base + tid * kOwn + e < n && k[e] == threshold;
        }
        block_before(mine, scratch, 0, total);
        cluster_before<kBlocks>(total, scratch, 0, ties, all);
        /* kept slots below m and from m on, up to this block's run, follow
         * from the counts of kept ones */
    }
    auto flags = [&](int base, int rank0, const uint32_t (&k)[kOwn], uint32_t &kept) {
        const int i0 = base + tid * kOwn;
        kept = 0;
#pragma unroll
        for (int e = 0; e < kOwn; e++)
            if (i0 + e < n && (k[e] > threshold || (k[e] == threshold && rank0++ < quota)))
                kept |= 1u << e;
    };
    auto own_mask = [&](int base) { /* this thread's slots of the chunk, and those of them below m */
        const int i0 = base + tid * kOwn;
        const int there = max(0, min(kOwn, n - i0)), low = max(0, min(there, m - from - i0));
        return make_uint2((1u << there) - 1u, (1u << low) - 1u);
    };
    if constexpr (kBlocks > 1) {
        int h = 0, q = 0, t0 = ties, total, all;
        for (int base = 0; base < n; base += kChooseChunk) {
            uint32_t k[kOwn], kept;
            own_keys(key, base, n, k);
            int mine = 0;
#pragma unroll
            for (int e = 0; e < kOwn; e++)
                mine += base + tid * kOwn + e < n && k[e] == threshold;
            const int rank0 = t0 + block_before(mine, scratch, 0, total);
            t0 += total;
            flags(base, rank0, k, kept);
            const uint2 own = own_mask(base);
            h += __popc(own.y & ~kept);
            q += __popc(kept & ~own.y);
            __syncthreads(); /* before the scan's scratch is used again */
        }
        block_before(h, scratch, 1, total);
        cluster_before<kBlocks>(total, scratch, 1, holes_n, all);
        __syncthreads();
        block_before(q, scratch, 1, total);
        cluster_before<kBlocks>(total, scratch, 2, sources_n, all);
        __syncthreads();
    }
    int ties_seen = ties;
    for (int base = 0; base < n; base += kChooseChunk) {
        uint32_t k[kOwn], kept;
        if (base == 0) {
#pragma unroll
            for (int e = 0; e < kOwn; e++)
                k[e] = first[e];
        } else {
            own_keys(key, base, n, k);
        }
        int mine = 0, total;
#pragma unroll
        for (int e = 0; e < kOwn; e++)
            mine += base + tid * kOwn + e < n && k[e] == threshold;
        const int rank0 = ties_seen + block_before(mine, scratch, 0, total);
        ties_seen += total;
        flags(base, rank0, k, kept);
        const uint2 own = own_mask(base);
        uint32_t hole = own.y & ~kept, source = kept & ~own.y;
        /* both counts in one scan */
        const int both = __popc(hole) | (__popc(source) << 16);
        const int before = block_before(both, scratch, 1, total);
        int to = holes_n + (before & 0xffff), of = sources_n + (before >> 16);
        holes_n += total & 0xffff;
        sources_n += total >> 16;
        const int i0 = from + base + tid * kOwn;
        for (; hole; hole &= hole - 1)
            holes[to++] = i0 + __ffs(hole) - 1;
        for (; source; source &= source - 1)
            sources[of++] = i0 + __ffs(source) - 1;
    }
    /* the last block of the run has seen them all */
    if (rank == kBlocks - 1 && tid == 0) {
        a.counts[item * 2] = holes_n;
        a.counts[item * 2 + 1] = m;
        scratch.shared[3] = holes_n;
    }
    const float *w0 = a.weights + at;
    const int32_t *pos0 = a.positions ? a.positions + at : nullptr;
    /* kept slots first: a hole's own entry is overwritten after */
    const int low = max(0, min(n, m - from));
    if (a.weights_out != a.weights)
        for (int i = tid; i < low; i += kChooseThreads)
            a.weights_out[at + from + i] = w[i];
    if (pos && a.positions_out != a.positions)
        for (int i = tid; i < low; i += kChooseThreads)
            a.positions_out[at + from + i] = pos[i];
    int pairs;
    if constexpr (kBlocks > 1) {
        auto cluster = cooperative_groups::this_cluster();
        __threadfence();
        cluster.sync();
        pairs = *cluster.map_shared_rank(&scratch.shared[3], kBlocks - 1);
    } else {
        __syncthreads();
        pairs = holes_n;
    }
    for (int i = rank * kChooseThreads + tid; i < pairs; i += kBlocks * kChooseThreads) {
        const int to = holes[i], of = sources[i];
        a.weights_out[at + to] = w0[of];
        if (pos)
            a.positions_out[at + to] = pos0[of];
    }
    if constexpr (kBlocks > 1)
        cooperative_groups::this_cluster().sync(); /* sources read, and shared memory done with */
    else
        __syncthreads();
    for (int i = low + tid; i < n; i += kChooseThreads) {
        a.weights_out[at + from + i] = 0.0f;
        if (pos)
            a.positions_out[at + from + i] = -1;
    }
}

/* Keys and values of the pairs: a group of row16 threads moves a row of
 * row16 16-byte pieces.  One pair at a time: 51 us for 242 MB in 256-byte
 * rows; with 2, 4 and 8 in flight in a thread the rows in flight on the chip
 * lie further apart and it took 53, 59 and 85. */
constexpr int kMoveThreads = 256;

__global__ void __launch_bounds__(kMoveThreads) move_kernel(const __grid_constant__ PagedEvict a, int row16) {
    const PagedPool &p = a.p;
    const int head = blockIdx.y, s = blockIdx.z;
    const int64_t item = int64_t(s) * p.kv_heads + head;
    const int n = a.counts[item * 2];
    if (blockIdx.x == 0 && head == 0 && threadIdx.x == 0)
        a.new_lengths[s] = a.counts[item * 2 + 1];
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
    cudaError_t e;
    if (p.capacity <= 2 * kChooseChunk) {
        choose_slots_kernel<1><<<dim3(p.kv_heads, p.sequences), kChooseThreads, 0, s>>>(a);
        e = cudaGetLastError();
    } else {
        cudaLaunchConfig_t config{};
        config.gridDim = dim3(8 * p.kv_heads, p.sequences);
        config.blockDim = dim3(kChooseThreads);
        config.stream = s;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = 8;
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        config.attrs = attr;
        config.numAttrs = 1;
        e = cudaLaunchKernelEx(&config, choose_slots_kernel<8>, a);
    }
    if (e != cudaSuccess)
        return e;
    const int row16 = p.head_dim * (p.type == 0 ? 4 : 2) / 16;
    /* blocks of an item: enough for all SMs together, no more than its pairs can feed */
    const int items = p.kv_heads * p.sequences, groups = kMoveThreads / row16;
    const int most = (p.capacity / 2 + groups - 1) / groups;
    const int blocks = std::max(1, std::min(most, std::max(8, 2048 / items)));
    move_kernel<<<dim3(blocks, p.kv_heads, p.sequences), kMoveThreads, 0, s>>>(a, row16);
    count_launches(2);
    return cudaGetLastError();
}

} // namespace nut
