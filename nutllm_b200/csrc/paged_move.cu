/* Moving keys and values within a paged cache: pages of forked sequences
 * (nut_paged_copy), and the accepted ones of drafted tokens
 * (nut_paged_compact).
 *
 * Both read and write each byte once.  A block takes one kv head of one page
 * or sequence; its threads hold 16-byte pieces, kDepth loads in flight each,
 * so that a page of 16 slots of 128 16-bit elements, keys and values, is one
 * round trip.
 *
 * Latency bounds both at the sizes of a step: up to 9 accepted of 64 tokens of
 * 64 sequences, 8 kv heads of 128 (4.2 MB) 5.2 us a pass.
 */
#include <cstdint>
#include <cuda_runtime.h>

#include "paged.cuh"

namespace nut {
namespace {

constexpr int kMoveThreads = 128;
constexpr int kDepth = 4;
constexpr int kPieces = kMoveThreads * kDepth; /* of a round */

/* 16-byte pieces of a row, and where one lies. */
__device__ __forceinline__ int row_pieces(const PagedPool &p) { return p.head_dim / (p.type == 0 ? 4 : 8); }
__device__ __forceinline__ int4 *piece_at(const PagedPool &p, void *pool, int page, int head, int place, int piece) {
    const int64_t element = int64_t(page) * p.page_stride + int64_t(head) * p.head_stride + int64_t(place) * p.slot_stride;
    return reinterpret_cast<int4 *>(pool) + element / (p.type == 0 ? 4 : 8) + piece;
}

__global__ void __launch_bounds__(kMoveThreads) copy_kernel(const __grid_constant__ PagedCopy a) {
    begin_kernel();
    const PagedPool &p = a.p;
    const int i = blockIdx.x, head = blockIdx.y, tid = threadIdx.x;
    const int from = a.source[i], to = a.target[i], slots = a.slots ? a.slots[i] : p.page_size;
    if (from == -1 && to == -1)
        return;
    if (unsigned(from) >= unsigned(p.n_pages) || unsigned(to) >= unsigned(p.n_pages)) {
        paged_fail(p, kPagedBadPage);
        return;
    }
    if (slots < 0 || slots > p.page_size) {
        paged_fail(p, kPagedBadLength);
        return;
    }
    const int width = row_pieces(p);
    const int64_t all = int64_t(slots) * width * 2;
    for (int64_t e0 = 0; e0 < all; e0 += kPieces) {
        int4 v[kDepth];
#pragma unroll
        for (int k = 0; k < kDepth; k++) {
            const int64_t e = e0 + k * kMoveThreads + tid;
            if (e < all) {
                const int64_t row = e / width;
                v[k] = *piece_at(p, row & 1 ? p.values : p.keys, from, head, int(row >> 1), int(e - row * width));
            }
        }
#pragma unroll
        for (int k = 0; k < kDepth; k++) {
            const int64_t e = e0 + k * kMoveThreads + tid;
            if (e < all) {
                const int64_t row = e / width;
                *piece_at(p, row & 1 ? p.values : p.keys, to, head, int(row >> 1), int(e - row * width)) = v[k];
            }
        }
    }
    if (p.bounds) {
        const int D = p.head_dim;
        const int64_t f = int64_t(from) * p.kv_heads + head, t = int64_t(to) * p.kv_heads + head;
        for (int d = tid; d < 2 * D; d += kMoveThreads)
            p.bounds[t * 2 * D + d] = p.bounds[f * 2 * D + d];
        if (tid == 0)
            p.bound_scales[t] = p.bound_scales[f];
    }
}

/* Rows move to lower places in ascending order, and a row's place is at or
 * below its source: a round may write what it and earlier ones have read. */
__global__ void __launch_bounds__(kMoveThreads) compact_kernel(const __grid_constant__ PagedCompact a) {
    __shared__ int list[kTreeMost], from_page[kTreeMost], to_page[kTreeMost];
    __shared__ int counted[kMoveThreads / 32];
    begin_kernel();
    const PagedPool &p = a.p;
    const int s = blockIdx.x, head = blockIdx.y, tid = threadIdx.x, lane = tid & 31;
    const int stored = p.lengths[s];
    const int row0 = a.starts[s], row1 = a.starts[s + 1];
    const int length = stored < 0 || stored > p.capacity ? -1 : stored;
    const int64_t n = int64_t(row1) - row0;
    bool fine = true;
    if (length < 0) {
        fine = false;
        if (tid == 0)
            paged_fail(p, kPagedBadLength);
    } else if (row0 < 0 || n < 0 || n > length) {
        fine = false;
        if (tid == 0)
            paged_fail(p, kPagedBadStarts);
    }
    /* the list ends with its first -1 */
    int end = a.n_accepted;
    for (int i = tid; i < a.n_accepted; i += kMoveThreads) {
        const int v = a.accepted[int64_t(s) * a.n_accepted + i];
        list[i] = v;
        if (v < 0)
            end = min(end, i);
    }
    end = __reduce_min_sync(0xffffffffu, end);
    if (lane == 0)
        counted[tid >> 5] = end;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kMoveThreads / 32; w++)
        end = min(end, counted[w]);
    const int first = int(length - n);
    bool bad_list = false, bad_page = false;
    if (fine)
        for (int i = tid; i < a.n_accepted; i += kMoveThreads) {
            const int v = list[i];
            if (i >= end) {
                bad_list |= v != -1 && i == end;
                continue;
            }
            if (v >= n || (i > 0 && v <= list[i - 1])) {
                bad_list = true;
                continue;
            }
            if (v != i) {
                from_page[i] = lookup(p, s, (first + v) / p.page_size);
                to_page[i] = lookup(p, s, (first + i) / p.page_size);
                bad_page |= from_page[i] < 0 || to_page[i] < 0;
            }
        }
    if (__syncthreads_or(bad_list)) {
        fine = false;
        if (tid == 0)
            paged_fail(p, kPagedBadStarts);
    }
    if (__syncthreads_or(bad_page)) {
        fine = false;
        if (tid == 0)
            paged_fail(p, kPagedBadPage);
    }
    if (fine) {
        const int width = row_pieces(p), rows = kPieces / (2 * width);
        for (int r0 = 0; r0 < end; r0 += rows) {
            int4 v[kDepth];
            const int all = min(rows, end - r0) * width * 2;
#pragma unroll
            for (int k = 0; k < kDepth; k++) {
                const int e = k * kMoveThreads + tid, row = e / width, i = r0 + (row >> 1);
                if (e < all && list[i] != i)
                    v[k] = *piece_at(p, row & 1 ? p.values : p.keys, from_page[i], head, (first + list[i]) % p.page_size,
                                     e - row * width);
            }
            __syncthreads();
#pragma unroll
            for (int k = 0; k < kDepth; k++) {
                const int e = k * kMoveThreads + tid, row = e / width, i = r0 + (row >> 1);
                if (e < all && list[i] != i)
                    *piece_at(p, row & 1 ? p.values : p.keys, to_page[i], head, (first + i) % p.page_size, e - row * width) =
                        v[k];
            }
        }
        const int64_t at = (int64_t(s) * p.kv_heads + head) * p.capacity + first;
        for (int r0 = 0; r0 < end && (a.positions || a.weights); r0 += kMoveThreads) {
            const int i = r0 + tid;
            const bool moves = i < end && list[i] != i;
            const int position = moves && a.positions ? a.positions[at + list[i]] : 0;
            const float weight = moves && a.weights ? a.weights[at + list[i]] : 0.0f;
            __syncthreads();
            if (moves && a.positions)
                a.positions[at + i] = position;
            if (moves && a.weights)
                a.weights[at + i] = weight;
        }
    }
    /* new_lengths may be the lengths that the other heads' blocks still read */
    if (tid == 0) {
        __threadfence();
        if (atomicAdd(a.order + s, 1) == p.kv_heads - 1) {
            a.order[s] = 0;
            a.new_lengths[s] = fine ? first + end : stored;
        }
    }
}

} // namespace

cudaError_t paged_copy(const PagedCopy &a, cudaStream_t s) {
    return launch_kernel(copy_kernel, dim3(a.count, a.p.kv_heads), kMoveThreads, 0, s, 1, a);
}

cudaError_t paged_compact(const PagedCompact &a, cudaStream_t s) {
    return launch_kernel(compact_kernel, dim3(a.p.sequences, a.p.kv_heads), kMoveThreads, 0, s, 1, a);
}

} // namespace nut
