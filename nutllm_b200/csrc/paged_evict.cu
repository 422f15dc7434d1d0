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
#include <cstdint>
#include <cuda_runtime.h>

#include "kernels.h"
#include "paged.cuh"

namespace nut {
namespace {

__global__ void __launch_bounds__(kChooseThreads)
    choose_slots_kernel(const __grid_constant__ PagedEvict a) {
    __shared__ ChooseScratch scratch;
    const PagedPool &p = a.p;
    const int head = blockIdx.x, s = blockIdx.y;
    const int n = checked_length(p, p.lengths[s]), m = min(n, a.budget);
    const int64_t item = int64_t(s) * p.kv_heads + head, at = item * p.capacity;
    const float *w = a.weights + at;
    const int32_t *pos = a.positions ? a.positions + at : nullptr;
    const int64_t recent_from = a.recent ? int64_t(a.seen[s]) - a.recent : INT64_MAX;
    const int sinks = a.sinks;
    auto key = [=](int i) -> uint32_t {
        if (pos && (pos[i] < sinks || pos[i] >= recent_from))
            return ordered_bits(INFINITY);
        const float v = w[i];
        return v != v ? 0u : ordered_bits(v);
    };
    uint32_t threshold;
    int quota;
    choose_largest(key, n, m, scratch, threshold, quota);
    int32_t *holes = a.pairs + at, *sources = holes + p.capacity / 2;
    int ties = 0, hole_n = 0, source_n = 0;
    for (int i0 = 0; i0 < n; i0 += blockDim.x) {
        const int i = i0 + threadIdx.x;
        const uint32_t k = i < n ? key(i) : 0u;
        const bool tie = i < n && k == threshold;
        int total;
        const int rank = ties + block_rank(tie, scratch.warp[0], total);
        ties += total;
        const bool kept = i < n && (k > threshold || (tie && rank < quota));
        const bool hole = i < m && !kept, source = i >= m && kept;
        const int to = hole_n + block_rank(hole, scratch.warp[1], total);
        hole_n += total;
        if (hole)
            holes[to] = i;
        const int from = source_n + block_rank(source, scratch.warp[2], total);
        source_n += total;
        if (source)
            sources[from] = i;
    }
    if (threadIdx.x == 0) {
        a.counts[item * 2] = hole_n;
        a.counts[item * 2 + 1] = m;
    }
    __syncthreads();
    /* kept slots first: a hole's own entry is overwritten after */
    if (a.weights_out != a.weights)
        for (int i = threadIdx.x; i < m; i += blockDim.x)
            a.weights_out[at + i] = w[i];
    if (pos && a.positions_out != a.positions)
        for (int i = threadIdx.x; i < m; i += blockDim.x)
            a.positions_out[at + i] = pos[i];
    __syncthreads();
    for (int i = threadIdx.x; i < hole_n; i += blockDim.x) {
        a.weights_out[at + holes[i]] = w[sources[i]];
        if (pos)
            a.positions_out[at + holes[i]] = pos[sources[i]];
    }
    __syncthreads();
    for (int i = m + threadIdx.x; i < n; i += blockDim.x) {
        a.weights_out[at + i] = 0.0f;
        if (pos)
            a.positions_out[at + i] = -1;
    }
}

__global__ void __launch_bounds__(256) move_kernel(const __grid_constant__ PagedEvict a, int row16) {
    const PagedPool &p = a.p;
    const int head = blockIdx.y, s = blockIdx.z;
    const int64_t item = int64_t(s) * p.kv_heads + head;
    const int n = a.counts[item * 2];
    if (blockIdx.x == 0 && head == 0 && threadIdx.x == 0)
        a.new_lengths[s] = a.counts[item * 2 + 1];
    const int32_t *holes = a.pairs + item * p.capacity, *sources = holes + p.capacity / 2;
    const int size = p.type == 0 ? 4 : 2, ps = p.page_size;
    for (int64_t e = int64_t(blockIdx.x) * blockDim.x + threadIdx.x; e < int64_t(n) * row16;
         e += int64_t(gridDim.x) * blockDim.x) {
        const int i = int(e / row16), c = int(e % row16);
        const int to = holes[i], from = sources[i];
        const int pt = checked_page(p, s, to / ps), pf = checked_page(p, s, from / ps);
        if (pt < 0 || pf < 0)
            continue;
        const int64_t dst = (int64_t(pt) * p.page_stride + int64_t(head) * p.head_stride +
                             int64_t(to % ps) * p.slot_stride) * size + c * 16;
        const int64_t src = (int64_t(pf) * p.page_stride + int64_t(head) * p.head_stride +
                             int64_t(from % ps) * p.slot_stride) * size + c * 16;
        char *k = static_cast<char *>(p.keys), *v = static_cast<char *>(p.values);
        *reinterpret_cast<uint4 *>(k + dst) = *reinterpret_cast<const uint4 *>(k + src);
        *reinterpret_cast<uint4 *>(v + dst) = *reinterpret_cast<const uint4 *>(v + src);
    }
}

} // namespace

cudaError_t paged_evict(const PagedEvict &a, cudaStream_t s) {
    const PagedPool &p = a.p;
    choose_slots_kernel<<<dim3(p.kv_heads, p.sequences), kChooseThreads, 0, s>>>(a);
    const int row16 = p.head_dim * (p.type == 0 ? 4 : 2) / 16;
    move_kernel<<<dim3(8, p.kv_heads, p.sequences), 256, 0, s>>>(a, row16);
    count_launches(2);
    return cudaGetLastError();
}

} // namespace nut
