/* Attention of one token per row over the paged KV cache
 * (nut_paged_attention).
 *
 *   z_t = scale q . k_t,  m = max z,  l = sum exp(z_t - m),
 *   out = sum exp(z_t - m) v_t / l,   lse = m + log l
 * in one pass over the keys and values with a running maximum and sum.
 * A CTA takes one row and kv head, its warps every fourth slot.
 */
#include <cstdint>
#include <cuda_runtime.h>

#include "kernels.h"
#include "paged.cuh"

namespace nut {
namespace {

constexpr int kWarps = 4;
constexpr int kMaxDim = 256;

template <typename R, typename T>
__global__ void __launch_bounds__(kWarps * 32)
    attention_simple_kernel(const __grid_constant__ PagedAttention a) {
    __shared__ float part[kWarps][kMaxDim], maxima[kWarps], sums[kWarps];
    const PagedPool &p = a.p;
    const int head = blockIdx.x, r = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int D = p.head_dim, ps = p.page_size;
    int length;
    const int s = row_span(p, a.row_sequence, a.row_length, r, length);
    const int span = a.selected ? a.n_selected * ps : length;
    const int32_t *list =
        a.selected ? a.selected + (int64_t(r) * p.kv_heads + head) * a.n_selected : nullptr;
    for (int g = 0; g < p.group; g++) {
        const int h = head * p.group + g;
        const R *q = static_cast<const R *>(a.q) + r * a.q_stride + int64_t(h) * D;
        float x[8], acc[8], m = -INFINITY, l = 0.0f;
        for (int i = 0; i < 8; i++) {
            x[i] = lane + 32 * i < D ? to_float(q[lane + 32 * i]) : 0.0f;
            acc[i] = 0.0f;
        }
        for (int v = warp; v < span; v += kWarps) {
            const int j = list ? list[v / ps] : v / ps, t = j * ps + v % ps;
            if (j < 0 || j >= p.max_pages || t >= length)
                continue;
            const int page = checked_page(p, s, j);
            if (page < 0)
                continue;
            const int64_t at = int64_t(page) * p.page_stride + int64_t(head) * p.head_stride +
                               int64_t(v % ps) * p.slot_stride;
            const T *k = static_cast<const T *>(p.keys) + at,
                    *val = static_cast<const T *>(p.values) + at;
            float dot = 0.0f;
            for (int i = 0; i < 8; i++)
                if (lane + 32 * i < D)
                    dot = fmaf(x[i], to_float(k[lane + 32 * i]), dot);
            const float z = warp_sum(dot) * a.scale;
            if (a.weights && lane == 0)
                a.logits[(int64_t(r) * p.heads + h) * p.capacity + t] = z;
            const float top = fmaxf(m, z), keep = m == top ? 1.0f : expf(m - top);
            const float w = z == -INFINITY ? 0.0f : expf(z - top);
            l = l * keep + w;
            for (int i = 0; i < 8; i++)
                if (lane + 32 * i < D)
                    acc[i] = fmaf(acc[i], keep, w * to_float(val[lane + 32 * i]));
            m = top;
        }
        for (int i = 0; i < 8; i++)
            if (lane + 32 * i < D)
                part[warp][lane + 32 * i] = acc[i];
        if (lane == 0) {
            maxima[warp] = m;
            sums[warp] = l;
        }
        __syncthreads();
        float top = -INFINITY, total = 0.0f;
        for (int w = 0; w < kWarps; w++)
            top = fmaxf(top, maxima[w]);
        for (int w = 0; w < kWarps; w++)
            total += maxima[w] == -INFINITY ? 0.0f : sums[w] * expf(maxima[w] - top);
        const float lse = top + logf(total);
        for (int d = threadIdx.x; d < D; d += blockDim.x) {
            float o = 0.0f;
            for (int w = 0; w < kWarps; w++)
                if (maxima[w] != -INFINITY)
                    o = fmaf(part[w][d], expf(maxima[w] - top), o);
            static_cast<R *>(a.out)[r * a.out_stride + int64_t(h) * D + d] =
                from_float<R>(total == 0.0f ? 0.0f : o / total);
        }
        if (a.lse && threadIdx.x == 0)
            a.lse[int64_t(r) * p.heads + h] = total == 0.0f ? -INFINITY : lse;
        if (a.weights) {
            const int64_t to = (int64_t(r) * p.kv_heads + head) * p.capacity;
            const float *z = a.logits + (int64_t(r) * p.heads + h) * p.capacity;
            const float *from = g == 0 ? a.weights : a.weights_out;
            for (int t = threadIdx.x; t < length; t += blockDim.x)
                a.weights_out[to + t] = from[to + t] + expf(z[t] - lse);
        }
        __syncthreads();
    }
}

} // namespace

cudaError_t paged_attention(const PagedAttention &a, cudaStream_t s) {
    const PagedPool &p = a.p;
    const dim3 grid(p.kv_heads, a.rows);
    const int n = kWarps * 32;
    if (p.type == 0)
        attention_simple_kernel<float, float><<<grid, n, 0, s>>>(a);
    else if (p.type == 1 && a.type == 0)
        attention_simple_kernel<float, __half><<<grid, n, 0, s>>>(a);
    else if (p.type == 1)
        attention_simple_kernel<__half, __half><<<grid, n, 0, s>>>(a);
    else if (a.type == 0)
        attention_simple_kernel<float, __nv_bfloat16><<<grid, n, 0, s>>>(a);
    else
        attention_simple_kernel<__nv_bfloat16, __nv_bfloat16><<<grid, n, 0, s>>>(a);
    count_launches(1);
    return cudaGetLastError();
}

} // namespace nut
