#pragma once
/* Choosing the largest of many 32-bit keys, ties to the lowest index: page
 * selection and slot eviction of the paged KV cache.
 *
 * search_largest: few keys, in the registers of a warp or of four; the
 * threshold is found between the least and the greatest of them, a quarter
 * of what is left at a time, by counting the keys at or above three
 * candidates: no atomics, no scans.
 * choose_largest: any number of keys, by histograms of 11, 11 and 10 bits
 * from the top; one block, or the blocks of a cluster that each hold a run
 * of the keys and add their histograms over distributed shared memory. */
#include <cooperative_groups.h>

#include "common.cuh"

namespace nut {

constexpr int kChooseThreads = 512;
constexpr int kChooseWarps = kChooseThreads / 32;
constexpr int kOwn = 8; /* neighbouring keys a thread holds of a chunk */
constexpr int kChooseChunk = kOwn * kChooseThreads;
constexpr int kBins = 2048;

struct ChooseScratch {
    int hist[kBins], sums[kBins];
    int warp[2][kChooseWarps];
    uint32_t prefix;
    int left, all;
    int shared[4]; /* read by the cluster's other blocks */
};

/* Exclusive rank of each thread's count within the block, and the total.
 * Two of these in a row need different `turn`s. */
__device__ __forceinline__ int block_before(int count, ChooseScratch &s, int turn, int &total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int upto = count;
#pragma unroll
    for (int x = 1; x < 32; x <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, upto, x);
        upto += lane >= x ? v : 0;
    }
    if (lane == 31)
        s.warp[turn][warp] = upto;
    __syncthreads();
    int t = lane < kChooseWarps ? s.warp[turn][lane] : 0;
    total = __reduce_add_sync(0xffffffffu, t);
    const int before = __reduce_add_sync(0xffffffffu, lane < warp ? t : 0);
    return before + upto - count;
}

/* N neighbouring words from x, zeros behind the first `there`; aligned:
 * 16-byte loads. */
template <int N, typename T> __device__ __forceinline__ void load_own(const T *x, int there, T (&v)[N]) {
    static_assert(sizeof(T) == 4 && N % 4 == 0, "16-byte loads");
    if (there >= N && (reinterpret_cast<uintptr_t>(x) & 15) == 0) {
#pragma unroll
        for (int e = 0; e < N; e += 4)
            *reinterpret_cast<uint4 *>(v + e) = *reinterpret_cast<const uint4 *>(x + e);
    } else {
#pragma unroll
        for (int e = 0; e < N; e++)
            v[e] = e < there ? x[e] : T(0);
    }
}

constexpr int kFewWarps = 4;

/* Sums of two counts (below 2^16 each) over kFewWarps warps, and the least
 * and greatest of two keys, for every thread. */
struct FewSums {
    int2 (*scratch)[kFewWarps]; /* [2] */
    int turn = 0;
    __device__ __forceinline__ const int2 *all(int a, int b) {
        if ((threadIdx.x & 31) == 0)
            scratch[turn][threadIdx.x >> 5] = make_int2(a, b);
        __syncthreads();
        const int2 *of = scratch[turn];
        turn ^= 1;
        return of;
    }
    __device__ __forceinline__ void operator()(int &a, int &b) {
        const int2 *of = all(__reduce_add_sync(0xffffffffu, a), __reduce_add_sync(0xffffffffu, b));
        a = b = 0;
#pragma unroll
        for (int w = 0; w < kFewWarps; w++) {
            a += of[w].x;
            b += of[w].y;
        }
    }
    __device__ __forceinline__ void range(uint32_t &lo, uint32_t &hi) {
        const int2 *of = all(int(__reduce_min_sync(0xffffffffu, lo)), int(__reduce_max_sync(0xffffffffu, hi)));
#pragma unroll
        for (int w = 0; w < kFewWarps; w++) {
            lo = min(lo, uint32_t(of[w].x));
            hi = max(hi, uint32_t(of[w].y));
        }
    }
};

/* The same over a warp. */
struct WarpSums {
    __device__ __forceinline__ void operator()(int &a, int &b) {
        a = __reduce_add_sync(0xffffffffu, a);
        b = __reduce_add_sync(0xffffffffu, b);
    }
    __device__ __forceinline__ void range(uint32_t &lo, uint32_t &hi) {
        lo = __reduce_min_sync(0xffffffffu, lo);
        hi = __reduce_max_sync(0xffffffffu, hi);
    }
};

/* The `want` (1 .. number of keys - 1) largest of the group's keys, N a
 * thread, 0 where a thread has fewer: a key is chosen when it is above
 * `threshold`, or equal to it and one of the first `quota` such.  Keys of
 * +inf stand outside the range that is searched: a few of them (pages that
 * are always read) would stretch it.  (From the top bit down, two bits a
 * round, 256 choices among 1024 pages took 6.4 us; so, 5.8.)  Invariant: at least `want` keys are
 * >= lo; `above` of them, fewer than `want`, are >= hi. */
template <int N, typename Sum>
__device__ __forceinline__ void search_largest(const uint32_t (&k)[N], int want, Sum &sum, uint32_t &threshold,
                                               int &quota) {
    constexpr uint32_t kTop = 0xff800000u; /* ordered_bits(+inf) */
    uint32_t lo = ~0u, hi = 0;
    int above = 0, here = 0;
#pragma unroll
    for (int e = 0; e < N; e++) {
        above += k[e] >= kTop;
        here += k[e] != 0;
        lo = min(lo, k[e] != 0 ? k[e] : ~0u);
        hi = max(hi, k[e] < kTop ? k[e] : 0u);
    }
    sum.range(lo, hi);
    sum(above, here);
    if (here < want) { /* keys of 0, too, are chosen */
        threshold = 0;
        quota = want - here;
        return;
    }
    if (above >= want) {
        int last = 0, none = 0; /* some NaN have all bits set */
#pragma unroll
        for (int e = 0; e < N; e++)
            last += k[e] == ~0u;
        sum(last, none);
        if (last >= want) {
            threshold = ~0u;
            quota = want;
            return;
        }
        lo = kTop;
        hi = ~0u;
        here = above;
        above = last;
    } else {
        hi++;
    }
    while (here != want) { /* otherwise no key is left to tell apart */
        if (hi - lo == 1) {
            threshold = lo;
            quota = want - above;
            return;
        }
        const uint32_t left = hi - lo, step = max(left / 4, 1u); /* lo < c1 <= c2 <= c3 < hi */
        const uint32_t c1 = lo + step, c2 = lo + left / 2, c3 = hi - step;
        int n1 = 0, n2 = 0, n3 = 0;
#pragma unroll
        for (int e = 0; e < N; e++) {
            n1 += k[e] >= c1;
            n2 += k[e] >= c2;
            n3 += k[e] >= c3;
        }
        n1 |= n2 << 16;
        sum(n1, n3);
        n2 = int(uint32_t(n1) >> 16);
        n1 &= 0xffff;
        if (n3 >= want) {
            lo = c3;
            here = n3;
        } else if (n2 >= want) {
            lo = c2;
            here = n2;
            hi = c3;
            above = n3;
        } else if (n1 >= want) {
            lo = c1;
            here = n1;
            hi = c2;
            above = n2;
        } else {
            hi = c1;
            above = n1;
        }
    }
    threshold = lo - 1u;
    quota = 0;
}

/* The keys of this thread in the chunk that starts at `base`; 0 beyond n.
 * key.own(i, there, k) makes the first `there` of keys i .. i + N - 1. */
template <int N, typename Key>
__device__ __forceinline__ void own_keys(const Key &key, int base, int n, uint32_t (&k)[N]) {
    const int i0 = base + int(threadIdx.x) * N;
    key.own(i0, max(0, min(N, n - i0)), k);
}

/* Adds `value` of every block of the cluster, for blocks of lower rank only
 * (before) and for all. */
template <int kBlocks>
__device__ __forceinline__ void cluster_before(int value, ChooseScratch &s, int place, int &before, int &all) {
    if constexpr (kBlocks == 1) {
        before = 0;
        all = value;
    } else {
        auto cluster = cooperative_groups::this_cluster();
        if (threadIdx.x == 0)
            s.shared[place] = value;
        cluster.sync();
        const int rank = int(cluster.block_rank());
        before = all = 0;
#pragma unroll
        for (int b = 0; b < kBlocks; b++) {
            const int v = *cluster.map_shared_rank(&s.shared[place], b);
            all += v;
            before += b < rank ? v : 0;
        }
    }
}

/* The `want` largest of all keys of the cluster (key(0) .. key(n - 1) in
 * this block, `all` in the cluster): a key is chosen when it is above
 * `threshold`, or equal to it and one of the first `quota` such.  `first`
 * holds the block's first chunk, N keys a thread. */
template <int kBlocks, int N, typename Key>
__device__ void choose_largest(const Key &key, int n, int all, int want, const uint32_t (&first)[N],
                               ChooseScratch &s, uint32_t &threshold, int &quota) {
    if (want <= 0 || want >= all) {
        threshold = want <= 0 ? 0xffffffffu : 0u;
        quota = want <= 0 ? 0 : all;
        return;
    }
    const int tid = threadIdx.x;
    uint32_t prefix = 0;
    int left = want;
    for (int pass = 0; pass < 3; pass++) {
        const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
        for (int i = tid; i < kBins; i += kChooseThreads)
            s.hist[i] = 0;
        __syncthreads();
        for (int base = 0; base < n; base += N * kChooseThreads) {
            uint32_t k[N];
            if (base == 0) {
#pragma unroll
                for (int e = 0; e < N; e++)
                    k[e] = first[e];
            } else {
                own_keys(key, base, n, k);
            }
#pragma unroll
            for (int e = 0; e < N; e++)
                if (base + tid * N + e < n &&
                    (pass == 0 || (k[e] >> (shift + bits)) == (prefix >> (shift + bits))))
                    atomicAdd(&s.hist[(k[e] >> shift) & ((1u << bits) - 1u)], 1);
        }
        __syncthreads();
        const int *hist = s.hist;
        if constexpr (kBlocks > 1) {
            auto cluster = cooperative_groups::this_cluster();
            cluster.sync();
            for (int i = tid; i < kBins; i += kChooseThreads) {
                int v = 0;
#pragma unroll
                for (int b = 0; b < kBlocks; b++)
                    v += *cluster.map_shared_rank(&s.hist[i], b);
                s.sums[i] = v;
            }
            cluster.sync(); /* the others' histograms have been read */
            hist = s.sums;
        }
        /* bins from the top: thread t has four of them */
        constexpr int kEach = kBins / kChooseThreads;
        int c[kEach], sum = 0;
#pragma unroll
        for (int i = 0; i < kEach; i++)
            sum += c[i] = hist[kBins - 1 - (tid * kEach + i)];
        int total;
        int before = block_before(sum, s, pass & 1, total);
        if (before < left && left <= before + sum) {
#pragma unroll
            for (int i = 0; i < kEach; i++) {
                if (left > before && left <= before + c[i]) {
                    s.prefix = prefix | (uint32_t(kBins - 1 - (tid * kEach + i)) << shift);
                    s.left = left - before;
                    s.all = c[i];
                }
                before += c[i];
            }
        }
        __syncthreads();
        prefix = s.prefix;
        left = s.left;
        if (left == s.all && prefix != 0u) { /* the whole bin: no key is left to tell apart */
            threshold = prefix - 1u;
            quota = 0;
            return;
        }
    }
    threshold = prefix;
    quota = left;
}

} // namespace nut
