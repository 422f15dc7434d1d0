/* Appending to the paged KV cache (nut_paged_append, nut_paged_summarise).
 *
 * New token at position t with cos/sin row c, z: for every pair (2i, 2i+1)
 *   x'[2i] = x[2i] c_i - x[2i+1] z_i,  x'[2i+1] = x[2i] z_i + x[2i+1] c_i
 * on the queries and the keys, in fp32 with unfused products (the
 * reference's order, src/quant_model.cpp:26-37).  A CTA takes one page that
 * receives tokens and one kv head: the group's queries, the key and the
 * value of each of the page's new tokens, then the page's key bounds over
 * all of its used slots.  Bytes bound it: the rows are read and written
 * once, the bounds re-read at most one page of keys from L2.  12 prompts of
 * up to 1,000 tokens, 32/8 heads of 128, fp32 rows to an fp16 cache with
 * bounds (297 MB): 56 us, 5.3 TB/s of those bytes, waiting for DRAM with all
 * the rows in flight that fit.  One token of one sequence: 2.5 us.  The bounds
 * of all pages anew (1.1 GB of keys): 460 us, 2.4 TB/s.
 */
#include <algorithm>
#include <cstdint>
#include <cuda_runtime.h>

#include "paged.cuh"

namespace nut {
namespace {


/* 4 neighbouring elements as floats; kVec: in one access. */
template <bool kVec> __device__ __forceinline__ void load4(const float *x, float *v) {
    if constexpr (kVec) {
        *reinterpret_cast<float4 *>(v) = *reinterpret_cast<const float4 *>(x);
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++)
            v[i] = x[i];
    }
}
template <bool kVec, typename T> __device__ __forceinline__ void load4(const T *x, float *v) {
    if constexpr (kVec) {
        const uint2 a = *reinterpret_cast<const uint2 *>(x);
        const T *e = reinterpret_cast<const T *>(&a);
#pragma unroll
        for (int i = 0; i < 4; i++)
            v[i] = to_float(e[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++)
            v[i] = to_float(x[i]);
    }
}
template <bool kVec> __device__ __forceinline__ void store4(float *x, const float *v) {
    if constexpr (kVec) {
        *reinterpret_cast<float4 *>(x) = make_float4(v[0], v[1], v[2], v[3]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++)
            x[i] = v[i];
    }
}
template <bool kVec, typename T> __device__ __forceinline__ void store4(T *x, const float *v) {
    if constexpr (kVec) {
        uint2 a;
        T *e = reinterpret_cast<T *>(&a);
#pragma unroll
        for (int i = 0; i < 4; i++)
            e[i] = from_float<T>(v[i]);
        *reinterpret_cast<uint2 *>(x) = a;
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++)
            x[i] = from_float<T>(v[i]);
    }
}
template <bool kVec> __device__ __forceinline__ void load2(const float *x, float *v) {
    if constexpr (kVec) {
        *reinterpret_cast<float2 *>(v) = *reinterpret_cast<const float2 *>(x);
    } else {
        v[0] = x[0];
        v[1] = x[1];
    }
}

/* Greatest and least key of each dimension over `used` slots, in 8 bits
 * (the bounds of nut_paged_view); every thread of the block takes part.  A
 * thread takes 8 dims of every `groups`-th slot, then the groups meet in
 * shared memory. */
template <int kThreads, typename T>
__device__ void page_bounds(const PagedPool &p, int page, int head, int used) {
    __shared__ float most_of[kThreads * 8], least_of[kThreads * 8], tops[kThreads / 32];
    const T *keys = static_cast<const T *>(p.keys) + int64_t(page) * p.page_stride +
                    int64_t(head) * p.head_stride;
    const int D = p.head_dim, octets = D / 8, groups = kThreads / octets;
    const int o = threadIdx.x % octets, group = threadIdx.x / octets;
    float most[8], least[8];
#pragma unroll
    for (int i = 0; i < 8; i++) {
        most[i] = -INFINITY;
        least[i] = INFINITY;
    }
    if (group < groups) {
        for (int t = group; t < used; t += groups) {
            float k[8];
            load4<true>(keys + int64_t(t) * p.slot_stride + o * 8, k);
            load4<true>(keys + int64_t(t) * p.slot_stride + o * 8 + 4, k + 4);
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float v = finite_key(k[i]);
                most[i] = fmaxf(most[i], v);
                least[i] = fminf(least[i], v);
            }
        }
#pragma unroll
        for (int i = 0; i < 8; i++) {
            most_of[group * D + o * 8 + i] = most[i];
            least_of[group * D + o * 8 + i] = least[i];
        }
    }
    __syncthreads();
    constexpr int kEach = (256 + kThreads - 1) / kThreads; /* dims of a thread */
    const int filled = min(groups, used);
    float hi[kEach], lo[kEach], top = 0.0f;
#pragma unroll
    for (int k = 0; k < kEach; k++) {
        const int d = threadIdx.x + k * kThreads;
        hi[k] = -INFINITY;
        lo[k] = INFINITY;
        if (d < D) {
            for (int i = 0; i < filled; i++) {
                hi[k] = fmaxf(hi[k], most_of[i * D + d]);
                lo[k] = fminf(lo[k], least_of[i * D + d]);
            }
            top = fmaxf(top, fmaxf(fabsf(hi[k]), fabsf(lo[k])));
        }
    }
    top = warp_max(top);
    if ((threadIdx.x & 31) == 0)
        tops[threadIdx.x >> 5] = top;
    __syncthreads();
    float all = 0.0f;
#pragma unroll
    for (int w = 0; w < kThreads / 32; w++)
        all = fmaxf(all, tops[w]);
    const float u = unit_of(all), inv = u > 0.0f ? 1.0f / u : 0.0f; /* exact: u is a power of two */
    const int64_t at = int64_t(page) * p.kv_heads + head;
#pragma unroll
    for (int k = 0; k < kEach; k++) {
        const int d = threadIdx.x + k * kThreads;
        if (d < D) {
            /* a key below 2^-149 of the unit is not a whole 0 of it */
            const float most_units = hi[k] > 0.0f ? fmaxf(ceilf(hi[k] * inv), 1.0f) : ceilf(hi[k] * inv);
            const float least_units = lo[k] < 0.0f ? fminf(floorf(lo[k] * inv), -1.0f) : floorf(lo[k] * inv);
            p.bounds[at * 2 * D + d] = int8_t(most_units);
            p.bounds[at * 2 * D + D + d] = int8_t(least_units);
        }
    }
    if (threadIdx.x == 0)
        p.bound_scales[at] = u;
}

/* A thread keeps 4 dims of each half of a row (neighbouring threads then read
 * and write neighbouring 16 bytes) and walks the page's new
 * (token, unit) rows, a unit being one of the group's query heads, the key or
 * the value.  1536 threads on an SM: registers for 1280 and 2048 took 61 and
 * 65 us where this takes 56 (12 prompts, 297 MB). */
template <int kThreads, typename R, typename T, bool kVec>
__global__ void __launch_bounds__(kThreads, 1536 / kThreads)
    append_kernel(const __grid_constant__ PagedAppend a) {
    begin_kernel();
    const PagedPool &p = a.p;
    const int head = blockIdx.y, s = blockIdx.z;
    const int row0 = a.starts[s], row1 = a.starts[s + 1];
    const int n = row1 - row0, length = checked_length(p, p.lengths[s]);
    if (n == 0)
        return;
    if (row0 < 0 || n < 0 || row1 > a.rows || n > a.max_new || n > length) {
        paged_fail(p, kPagedBadStarts);
        return;
    }
    const int first = length - n, ps = p.page_size; /* first new slot */
    const int j = first / ps + int(blockIdx.x);     /* logical page */
    const int t0 = max(first, j * ps), t1 = min(length, (j + 1) * ps);
    if (t0 >= t1)
        return;
    const int page = checked_page(p, s, j);
    if (page < 0)
        return;
    const int ahead = a.seen ? a.seen[s] - length : 0; /* position less slot */
    const int D = p.head_dim, half = D / 2, octets = D / 8, groups = kThreads / octets;
    const int o = threadIdx.x % octets * 4, group = threadIdx.x / octets;
    const int64_t base = int64_t(page) * p.page_stride + int64_t(head) * p.head_stride + o;
    T *keys = static_cast<T *>(p.keys) + base, *values = static_cast<T *>(p.values) + base;
    const int heads = a.q ? p.group : 0, units = heads + 2;
    /* whether slot t's position has a rotation, where there are any: rows without one are skipped */
    const auto turns = [&](int t) {
        const int64_t pos = int64_t(t) + ahead;
        return !a.cos || (pos >= 0 && pos < a.rope_rows);
    };
    if (group < groups)
        for (int e = group; e < (t1 - t0) * units; e += groups) {
            const int t = t0 + e / units, unit = e % units;
            const int64_t row = row0 + (t - first), column = int64_t(head * p.group + unit) * D + o;
            float v[8], c[4], z[4];
            if (!turns(t)) {
                paged_fail(p, kPagedBadPosition);
                continue;
            }
            const R *x = unit < heads    ? static_cast<const R *>(a.q) + row * a.q_stride + column
                         : unit == heads ? static_cast<const R *>(a.k) + row * a.k_stride + head * D + o
                                         : static_cast<const R *>(a.v) + row * a.v_stride + head * D + o;
            load4<kVec>(x, v);
            load4<kVec>(x + half, v + 4);
            if (a.cos && unit <= heads) {
                const int64_t turn = (int64_t(t) + ahead) * half + o / 2;
                load2<kVec>(a.cos + turn, c);
                load2<kVec>(a.cos + turn + half / 2, c + 2);
                load2<kVec>(a.sin + turn, z);
                load2<kVec>(a.sin + turn + half / 2, z + 2);
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float x0 = v[2 * i], x1 = v[2 * i + 1];
                    v[2 * i] = __fsub_rn(__fmul_rn(x0, c[i]), __fmul_rn(x1, z[i]));
                    v[2 * i + 1] = __fadd_rn(__fmul_rn(x0, z[i]), __fmul_rn(x1, c[i]));
                }
            }
            if (unit >= heads) {
                T *to = (unit > heads ? values : keys) + int64_t(t - j * ps) * p.slot_stride;
                store4<true>(to, v);
                store4<true>(to + half, v + 4);
            } else {
                R *to = static_cast<R *>(a.q_out) + row * a.q_out_stride + column;
                store4<kVec>(to, v);
                store4<kVec>(to + half, v + 4);
            }
        }
    if (a.positions || a.weights) {
        const int64_t at = (int64_t(s) * p.kv_heads + head) * p.capacity;
        for (int t = t0 + threadIdx.x; t < t1; t += kThreads) {
            if (!turns(t))
                continue;
            if (a.positions)
                a.positions[at + t] = t + ahead;
            if (a.weights)
                a.weights[at + t] = 0.0f;
        }
    }
    if (p.bounds) {
        __syncthreads(); /* the block's own key writes, read back below */
        page_bounds<kThreads, T>(p, page, head, t1 - j * ps);
    }
}

constexpr int kSummaryThreads = 128;

template <typename T>
__global__ void __launch_bounds__(kSummaryThreads) summarise_kernel(const __grid_constant__ PagedPool p) {
    begin_kernel();
    const int j = blockIdx.x, head = blockIdx.y, s = blockIdx.z;
    const int used = min(checked_length(p, p.lengths[s]) - j * p.page_size, p.page_size);
    if (used <= 0)
        return;
    const int page = checked_page(p, s, j);
    if (page >= 0)
        page_bounds<kSummaryThreads, T>(p, page, head, used);
}

template <typename R, typename T> cudaError_t launch_append(const PagedAppend &a, cudaStream_t s) {
    const PagedPool &p = a.p;
    /* pages that max_new consecutive slots can touch */
    const dim3 grid((a.max_new + p.page_size - 2) / p.page_size + 1, p.kv_heads, p.sequences);
    uintptr_t bits = 0;
    for (const void *x : {a.q, a.k, a.v, static_cast<const void *>(a.q_out), static_cast<const void *>(a.cos),
                          static_cast<const void *>(a.sin)})
        bits |= reinterpret_cast<uintptr_t>(x);
    for (int64_t stride : {a.q_stride, a.k_stride, a.v_stride, a.q_out_stride})
        bits |= uintptr_t(stride) * sizeof(R);
    const bool vec = (bits & 15) == 0;
    /* a block has a page's new rows of one kv head: where they are few (one
     * token of 3 rows: 4.2 against 5.7 us for 2048 pages), two warps */
    const int64_t octets = int64_t(std::min(a.max_new, p.page_size)) * ((a.q ? p.group : 0) + 2) * (p.head_dim / 8);
    if (octets <= 64)
        return launch_kernel(vec ? append_kernel<64, R, T, true> : append_kernel<64, R, T, false>, grid, 64, 0, s, 1, a);
    return launch_kernel(vec ? append_kernel<128, R, T, true> : append_kernel<128, R, T, false>, grid, 128, 0, s, 1, a);
}

} // namespace

cudaError_t paged_append(const PagedAppend &a, cudaStream_t s) {
    const bool wide = a.type == 0;
    if (a.p.type == 0)
        return launch_append<float, float>(a, s);
    if (a.p.type == 1)
        return wide ? launch_append<float, __half>(a, s) : launch_append<__half, __half>(a, s);
    return wide ? launch_append<float, __nv_bfloat16>(a, s) : launch_append<__nv_bfloat16, __nv_bfloat16>(a, s);
}

cudaError_t paged_summarise(const PagedPool &p, cudaStream_t s) {
    const dim3 grid(p.max_pages, p.kv_heads, p.sequences);
    const auto kernel = p.type == 0   ? summarise_kernel<float>
                        : p.type == 1 ? summarise_kernel<__half>
                                      : summarise_kernel<__nv_bfloat16>;
    return launch_kernel(kernel, grid, kSummaryThreads, 0, s, 1, p);
}

} // namespace nut
