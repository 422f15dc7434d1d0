/* Pages of branching sequences (nut_pages_update).
 *
 * One cluster of blocks does all of an update in three steps, with a
 * barrier of the cluster between them:
 *   1  each sequence's kept pages are staged; every entry of the table that
 *      changes takes a holder from its old page and gives one to its new
 *      page (`delta`), and a partly kept page that is to be written counts
 *      its writers and notes the first of them
 *   2  who gets a copy follows from those; a prefix sum over the sequences
 *      says which free pages each takes
 *   3  unless something was out of range: the table, lengths, copy lists and
 *      holders are written, pages without a holder are counted, and after
 *      another barrier given back in order of their numbers.
 * Sums of whole numbers do not depend on the order of the atomics, and
 * places come from prefix sums, so results do not depend on timing.
 *
 * It is a chain of round trips to L2, not bytes: in a graph, with the copies
 * behind it, 64 sequences of 1,003 slots take 16 us, 512 of 16,000 slots, a
 * table of half a million entries, 27 us.
 */
#include <climits>
#include <cooperative_groups.h>
#include <cstdint>
#include <cuda_runtime.h>

#include "branch.h"
#include "paged.cuh"

namespace nut {
namespace {

namespace cg = cooperative_groups;

/* Loads that a lane has in flight: with one, a table of 512 rows of 1,000 pages
 * took 125 us. */
constexpr int kFlight = 8;

__device__ __forceinline__ int pages_of(int slots, int page_size) { return int((unsigned(slots) + page_size - 1) / page_size); }

/* Exclusive sum over the block's threads, and the total. */
template <int kWarpsABlock> __device__ __forceinline__ int64_t before_in_block(int64_t v, int64_t *sums, int64_t &total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int64_t upto = v;
#pragma unroll
    for (int x = 1; x < 32; x <<= 1) {
        const int64_t w = __shfl_up_sync(0xffffffffu, upto, x);
        upto += lane >= x ? w : 0;
    }
    __syncthreads();
    if (lane == 31)
        sums[warp] = upto;
    __syncthreads();
    total = 0;
    int64_t before = upto - v;
#pragma unroll
    for (int w = 0; w < kWarpsABlock; w++) {
        before += w < warp ? sums[w] : 0;
        total += sums[w];
    }
    return before;
}

template <int kThreads, int kBlocks> __global__ void __launch_bounds__(kThreads, 1) update_kernel(const __grid_constant__ PagesUpdate a) {
    constexpr int kWarpsABlock = kThreads / 32, kWarps = kBlocks * kWarpsABlock;
    __shared__ int64_t sums[kWarpsABlock];
    __shared__ int places[kThreads];
    __shared__ uint8_t copied[kThreads];
    begin_kernel();
    cg::cluster_group cluster = cg::this_cluster();
    const int tid = threadIdx.x, lane = tid & 31;
    const int warp = int(blockIdx.x) * kWarpsABlock + (tid >> 5); /* of the cluster */
    const int S = a.sequences, P = a.n_pages, ps = a.page_size;
    const int64_t capacity = int64_t(a.max_pages) * ps;
    int met = 0;

    /* 1 */
    for (int s = warp; s < S; s += kWarps) {
        const int p = a.parent ? a.parent[s] : s, length = a.lengths[s], more = a.add ? a.add[s] : 0;
        const int wish = a.keep ? a.keep[s] : INT_MAX;
        const bool fine = p >= -1 && p < S && more >= 0 && wish >= 0;
        const int from = !fine || p < 0 ? 0 : a.lengths[p];
        int bad = fine ? 0 : kPagesBadArgument;
        const int kept = min(wish, from);
        if (length < 0 || length > capacity || from < 0 || from > capacity || int64_t(kept) + more > capacity)
            bad |= kPagesBadLength;
        met |= bad;
        if (bad) {
            if (lane == 0)
                a.plan[s] = make_int4(0, 0, -1, -1);
            continue;
        }
        const int had = pages_of(length, ps), keeps = pages_of(kept, ps);
        const int32_t *mine = a.table + int64_t(s) * a.max_pages, *its = a.table + int64_t(p) * a.max_pages;
        int32_t *to = a.staged + int64_t(s) * a.max_pages;
        /* a sequence that continues itself keeps its entries as they are */
        const int ends = max(had, keeps);
        int changes = -1; /* entries from here on are staged: those before stay */
        for (int i0 = (p == s ? keeps : 0) + lane; i0 - lane < ends; i0 += 32 * kFlight) {
            int old[kFlight], next[kFlight];
            bool differ = false;
#pragma unroll
            for (int k = 0; k < kFlight; k++) {
                const int i = i0 + k * 32;
                old[k] = i < had ? mine[i] : -1;
                next[k] = i < keeps ? its[i] : -1;
                differ |= old[k] != next[k];
            }
            if (changes < 0 && __any_sync(0xffffffffu, differ))
                changes = i0 - lane;
#pragma unroll
            for (int k = 0; k < kFlight; k++) {
                const int i = i0 + k * 32;
                if (i >= ends)
                    break;
                if ((i < had && unsigned(old[k]) >= unsigned(P)) || (i < keeps && unsigned(next[k]) >= unsigned(P))) {
                    met |= kPagesBadPage;
                    continue;
                }
                if (old[k] != next[k]) {
                    if (i < had)
                        atomicAdd(a.delta + old[k], -1);
                    if (i < keeps)
                        atomicAdd(a.delta + next[k], 1);
                }
                if (i < keeps && changes >= 0)
                    to[i] = next[k];
            }
        }
        if (lane == 0) {
            int tail = more > 0 && kept % ps != 0 ? its[keeps - 1] : -1;
            if (unsigned(tail) >= unsigned(P))
                tail = -1;
            if (tail >= 0) {
                atomicAdd(a.writers + tail, 1);
                atomicMax(a.first + tail, S - s); /* the first writer has the greatest */
            }
            a.plan[s] = make_int4(kept, kept + more, tail, p);
            a.changes[s] = changes < 0 ? keeps : min(changes, keeps);
        }
    }
    cluster.sync();

    /* 2 */
    const int count = __ldcg(a.free_count);
    int64_t total = 0;
    if (count < 0 || count > P)
        met |= kPagesBadPage;
    else
        for (int s0 = 0; s0 < S; s0 += kThreads) {
            const int s = s0 + tid;
            int need = 0;
            bool copy = false;
            if (s < S) {
                const int4 plan = __ldcg(a.plan + s);
                if (plan.z >= 0) {
                    const int holders = a.refs[plan.z] + __ldcg(a.delta + plan.z);
                    copy = holders > 1 &&
                           !(__ldcg(a.writers + plan.z) == holders && __ldcg(a.first + plan.z) == S - s);
                }
                need = pages_of(plan.y, ps) - pages_of(plan.x, ps) + (copy ? 1 : 0);
            }
            int64_t all;
            const int64_t before = total + before_in_block<kWarpsABlock>(need, sums, all);
            total += all;
            if (total > count) /* the same in every block */
                break;
            places[tid] = int(before);
            copied[tid] = copy;
            __syncthreads();
            /* the block's warps stage the pages that the chunk's sequences take */
            for (int i = warp; i < min(kThreads, S - s0); i += kWarps) {
                const int4 plan = __ldcg(a.plan + s0 + i);
                const int keeps = pages_of(plan.x, ps), ends = pages_of(plan.y, ps), begin = keeps - copied[i];
                int32_t *to = a.staged + int64_t(s0 + i) * a.max_pages;
                for (int j = begin + lane; j < ends; j += 32) {
                    const int page = a.free_pages[count - 1 - (places[i] + j - begin)];
                    /* a page without a holder, and listed once */
                    if (unsigned(page) >= unsigned(P) || a.refs[page] != 0 || __ldcg(a.delta + page) != 0 ||
                        atomicAdd(a.writers + page, 1) != 0)
                        met |= kPagesBadPage;
                    else
                        to[j] = page;
                }
                if (lane == 0 && copied[i])
                    a.plan[s0 + i].w = -2 - plan.w; /* below -1: it gets a copy */
            }
            __syncthreads();
        }
    if (total > count)
        met |= kPagesNoneFree;
    met = __reduce_or_sync(0xffffffffu, met);
    if (lane == 0 && met)
        atomicOr(a.met, met);
    cluster.sync();

    /* 3 */
    const int wrong = __ldcg(a.met);
    for (int s = warp; s < S; s += kWarps) {
        if (wrong) {
            if (lane == 0 && a.copy_from) {
                a.copy_from[s] = a.copy_to[s] = -1;
                a.copy_slots[s] = 0;
            }
            continue;
        }
        const int4 plan = __ldcg(a.plan + s);
        const int keeps = pages_of(plan.x, ps), ends = pages_of(plan.y, ps);
        const bool copy = plan.w < -1;
        const int32_t *next = a.staged + int64_t(s) * a.max_pages;
        int32_t *row = a.table + int64_t(s) * a.max_pages;
        const int taken = keeps - (copy ? 1 : 0);
        for (int i0 = min(__ldcg(a.changes + s), taken) + lane; i0 < ends; i0 += 32 * kFlight) {
            int page[kFlight];
#pragma unroll
            for (int k = 0; k < kFlight; k++)
                page[k] = i0 + k * 32 < ends ? __ldcg(next + i0 + k * 32) : -1;
#pragma unroll
            for (int k = 0; k < kFlight; k++) {
                const int i = i0 + k * 32;
                if (page[k] >= 0)
                    row[i] = page[k];
                if (page[k] >= 0 && i >= taken)
                    a.refs[page[k]] = 1;
            }
        }
        if (lane == 0) {
            a.lengths[s] = plan.y;
            if (a.copy_from) {
                a.copy_from[s] = copy ? plan.z : -1;
                a.copy_to[s] = copy ? __ldcg(next + keeps - 1) : -1;
                a.copy_slots[s] = copy ? plan.x % ps : 0;
            }
        }
    }
    /* a run of pages for each warp: what their holders come to */
    const int run = (P + kWarps - 1) / kWarps;
    const int p0 = min(int64_t(warp) * run, int64_t(P)), p1 = min(p0 + run, P);
    int gone = 0, late = 0;
    for (int i0 = p0 + lane; i0 < p1; i0 += 32 * kFlight) {
        int d[kFlight], w[kFlight], held[kFlight];
#pragma unroll
        for (int k = 0; k < kFlight; k++) {
            const int i = i0 + k * 32;
            d[k] = i < p1 ? __ldcg(a.delta + i) : 0;
            w[k] = i < p1 ? __ldcg(a.writers + i) : 0;
            held[k] = i < p1 ? __ldcg(a.refs + i) : 0;
        }
#pragma unroll
        for (int k = 0; k < kFlight; k++) {
            const int i = i0 + k * 32;
            if (!d[k] && !w[k])
                continue;
            if (w[k]) {
                a.first[i] = 0;
                a.writers[i] = 0;
            }
            int next = held[k] + d[k];
            /* copies take the place of writers, but where the first keeps the page; a page
             * taken from the list has one holder at most */
            if (w[k] && next > 1)
                next -= w[k] == next ? w[k] - 1 : w[k];
            if (next < 0) { /* fewer holders than the table shows */
                next = 0;
                late |= kPagesBadPage;
            }
            const bool freed = !wrong && held[k] > 0 && next == 0;
            if (!wrong && next != held[k])
                a.refs[i] = next;
            a.delta[i] = freed ? INT_MIN : 0;
            gone += freed;
        }
    }
    gone = __reduce_add_sync(0xffffffffu, gone);
    if (lane == 0)
        a.freed[warp] = gone;
    cluster.sync();
    int before = 0, all = 0;
    for (int w = lane; w < kWarps; w += 32) {
        const int n = __ldcg(a.freed + w);
        all += n;
        before += w < warp ? n : 0;
    }
    all = __reduce_add_sync(0xffffffffu, all);
    before = __reduce_add_sync(0xffffffffu, before);
    if (gone) {
        int64_t at = count - total + before;
        for (int i = p0; i < p1; i += 32) {
            const bool freed = i + lane < p1 && a.delta[i + lane] == INT_MIN;
            const unsigned who = __ballot_sync(0xffffffffu, freed);
            if (freed) {
                const int64_t place = at + __popc(who & ((1u << lane) - 1u));
                if (place < P)
                    a.free_pages[place] = i + lane;
                else /* a page that had holders was listed as free */
                    late |= kPagesBadPage;
                a.delta[i + lane] = 0;
            }
            at += __popc(who);
        }
    }
    if (!wrong && late)
        atomicOr(a.error, late);
    if (warp == 0 && lane == 0) {
        if (wrong) {
            atomicOr(a.error, wrong);
            *a.met = 0;
        } else {
            *a.free_count = int(min(count - total + all, int64_t(P)));
        }
    }
}

} // namespace

cudaError_t pages_update(const PagesUpdate &a, cudaStream_t s) {
    /* A small book is a chain of barriers, which few threads pass sooner; a large one needs loads in
     * flight, and takes the most blocks that a cluster can have.  With 8 blocks of 256, 8 of 1,024 and
     * 16 of 1,024 threads, us in a graph, with copies of one small head behind it: 32 sequences of 1,000 slots
     * 13.3, 17.5, 19.8; 64 of 1,003 14.2, 19.1, 21.8; 128 of 1,000 17.5, 18.1, 19.7; 128 of 8,000 20.9, 19.3,
     * 20.6; 256 of 1,000 23.9, 18.4, 20.2; 1,024 of 2,000 67, 31.1, 24.6; 512 of 16,000 72, 34.9, 26.2. */
    const bool small = a.sequences <= 128 && a.n_pages <= 16384 && int64_t(a.sequences) * a.max_pages <= 65536;
    if (small)
        return launch_kernel(update_kernel<256, 8>, dim3(8), 256, 0, s, 8, a);
    const auto kernel = update_kernel<1024, 16>;
    static bool set[kMaxDevices] = {};
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess)
        return e;
    if (!set[device % kMaxDevices]) {
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (e != cudaSuccess)
            return e;
        set[device % kMaxDevices] = true;
    }
    return launch_kernel(kernel, dim3(16), 1024, 0, s, 16, a);
}

} // namespace nut
