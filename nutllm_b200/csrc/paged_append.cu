/* Appending to the paged KV cache (nut_paged_append, nut_paged_summarise).
 *
 * New token at position t with cos/sin row c, z: for every pair (2i, 2i+1)
 *   x'[2i] = x[2i] c_i - x[2i+1] z_i,  x'[2i+1] = x[2i] z_i + x[2i+1] c_i
 * on the queries and the keys, in fp32 with unfused products (the
 * reference's order, src/quant_model.cpp:26-37).  A CTA takes one page that
 * receives tokens and one kv head: the group's queries, the key and the
 * value of each of the page's new tokens, then the page's key bounds over
 * all of its used slots.  Bytes bound it: the rows are read and written
 * once, the bounds re-read at most one page of keys from L2.
 */
#include <cstdint>
#include <cuda_runtime.h>

#include "kernels.h"
#include "paged.cuh"

namespace nut {
namespace {

/* Greatest and least key of each dimension over `used` slots, in 8 bits
 * (the bounds of nut_paged_view); every thread of the block takes part. */
template <typename T>
__device__ void page_bounds(const PagedPool &p, int page, int head, int used) {
    __shared__ float tops[8];
    const T *keys = static_cast<const T *>(p.keys) + int64_t(page) * p.page_stride +
                    int64_t(head) * p.head_stride;
    const int D = p.head_dim, d = threadIdx.x;
    float most = 0.0f, least = 0.0f;
    if (d < D) {
        most = -INFINITY;
        least = INFINITY;
        for (int t = 0; t < used; t++) {
            const float k = finite_key(to_float(keys[int64_t(t) * p.slot_stride + d]));
            most = fmaxf(most, k);
            least = fminf(least, k);
        }
    }
    const float top = warp_max(fmaxf(fabsf(most), fabsf(least)));
    if ((threadIdx.x & 31) == 0)
        tops[threadIdx.x >> 5] = top;
    __syncthreads();
    float all = 0.0f;
    for (int w = 0; w < int(blockDim.x >> 5); w++)
        all = fmaxf(all, tops[w]);
    const float u = unit_of(all);
    const int64_t at = int64_t(page) * p.kv_heads + head;
    if (d < D) {
        const float inv = u > 0.0f ? 1.0f / u : 0.0f; /* exact: u is a power of two */
        p.bounds[at * 2 * D + d] = int8_t(ceilf(most * inv));
        p.bounds[at * 2 * D + D + d] = int8_t(floorf(least * inv));
    }
    if (threadIdx.x == 0)
        p.bound_scales[at] = u;
    __syncthreads();
}

template <typename R, typename T>
__global__ void __launch_bounds__(256) append_kernel(const __grid_constant__ PagedAppend a) {
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
    const int seen = a.seen ? a.seen[s] : length;
    const int D = p.head_dim, half = D / 2;
    const int64_t base = int64_t(page) * p.page_stride + int64_t(head) * p.head_stride;
    T *keys = static_cast<T *>(p.keys) + base, *values = static_cast<T *>(p.values) + base;
    const int units = (a.q ? p.group : 0) + 2; /* query heads, key, value */
    for (int e = threadIdx.x; e < (t1 - t0) * units * half; e += blockDim.x) {
        const int t = t0 + e / (units * half), rest = e % (units * half);
        const int unit = rest / half, i = rest % half;
        const int row = row0 + (t - first);
        if (unit == units - 1) {
            const R *v = static_cast<const R *>(a.v) + row * a.v_stride + head * D + 2 * i;
            T *to = values + int64_t(t - j * ps) * p.slot_stride + 2 * i;
            to[0] = from_float<T>(to_float(v[0]));
            to[1] = from_float<T>(to_float(v[1]));
            continue;
        }
        const bool is_key = unit == units - 2;
        const R *x = is_key ? static_cast<const R *>(a.k) + row * a.k_stride + head * D
                            : static_cast<const R *>(a.q) + row * a.q_stride +
                                  (head * p.group + unit) * D;
        float x0 = to_float(x[2 * i]), x1 = to_float(x[2 * i + 1]);
        if (a.cos) {
            const int64_t pos = int64_t(t) + (seen - length);
            if (pos < 0 || pos >= a.rope_rows) {
                paged_fail(p, kPagedBadPosition);
            } else {
                const float c = a.cos[pos * half + i], z = a.sin[pos * half + i];
                const float y0 = __fsub_rn(__fmul_rn(x0, c), __fmul_rn(x1, z));
                x1 = __fadd_rn(__fmul_rn(x0, z), __fmul_rn(x1, c));
                x0 = y0;
            }
        }
        if (is_key) {
            T *to = keys + int64_t(t - j * ps) * p.slot_stride + 2 * i;
            to[0] = from_float<T>(x0);
            to[1] = from_float<T>(x1);
        } else {
            R *to = static_cast<R *>(a.q_out) + row * a.q_out_stride +
                    (head * p.group + unit) * D + 2 * i;
            to[0] = from_float<R>(x0);
            to[1] = from_float<R>(x1);
        }
    }
    if (a.positions || a.weights) {
        const int64_t at = (int64_t(s) * p.kv_heads + head) * p.capacity;
        for (int t = t0 + threadIdx.x; t < t1; t += blockDim.x) {
            if (a.positions)
                a.positions[at + t] = t + (seen - length);
            if (a.weights)
                a.weights[at + t] = 0.0f;
        }
    }
    if (p.bounds) {
        __syncthreads(); /* the block's own key writes, read back below */
        page_bounds<T>(p, page, head, t1 - j * ps);
    }
}

template <typename T>
__global__ void __launch_bounds__(256) summarise_kernel(const __grid_constant__ PagedPool p) {
    const int j = blockIdx.x, head = blockIdx.y, s = blockIdx.z;
    const int used = min(checked_length(p, p.lengths[s]) - j * p.page_size, p.page_size);
    if (used <= 0)
        return;
    const int page = checked_page(p, s, j);
    if (page >= 0)
        page_bounds<T>(p, page, head, used);
}

} // namespace

cudaError_t paged_append(const PagedAppend &a, cudaStream_t s) {
    const PagedPool &p = a.p;
    /* pages that max_new consecutive slots can touch */
    const dim3 grid((a.max_new + p.page_size - 2) / p.page_size + 1, p.kv_heads, p.sequences);
    const bool wide = a.type == 0;
    if (p.type == 0)
        append_kernel<float, float><<<grid, 256, 0, s>>>(a);
    else if (p.type == 1 && wide)
        append_kernel<float, __half><<<grid, 256, 0, s>>>(a);
    else if (p.type == 1)
        append_kernel<__half, __half><<<grid, 256, 0, s>>>(a);
    else if (wide)
        append_kernel<float, __nv_bfloat16><<<grid, 256, 0, s>>>(a);
    else
        append_kernel<__nv_bfloat16, __nv_bfloat16><<<grid, 256, 0, s>>>(a);
    count_launches(1);
    return cudaGetLastError();
}

cudaError_t paged_summarise(const PagedPool &p, cudaStream_t s) {
    const dim3 grid(p.max_pages, p.kv_heads, p.sequences);
    if (p.type == 0)
        summarise_kernel<float><<<grid, 256, 0, s>>>(p);
    else if (p.type == 1)
        summarise_kernel<__half><<<grid, 256, 0, s>>>(p);
    else
        summarise_kernel<__nv_bfloat16><<<grid, 256, 0, s>>>(p);
    count_launches(1);
    return cudaGetLastError();
}

} // namespace nut
