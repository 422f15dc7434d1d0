/* Choosing pages by their key bounds (nut_paged_select).
 *
 * score(page) = max_g u_g U sum_d max(x_gd M_d, x_gd L_d), with x the query
 * head in 8 bits, M and L the page's greatest and least key in 8 bits, u and
 * U powers of two.  The sum is at most 256 * 127 * 128 < 2^24 in size, so
 * it is exact in an int and in fp32, whatever its order.
 */
#include <cstdint>
#include <cuda_runtime.h>

#include "kernels.h"
#include "paged.cuh"

namespace nut {
namespace {

/* Warp per page: its score for one row and kv head. */
template <typename R>
__global__ void __launch_bounds__(256) score_kernel(const __grid_constant__ PagedSelect a) {
    const PagedPool &p = a.p;
    const int head = blockIdx.y, r = blockIdx.z, lane = threadIdx.x & 31;
    const int j = int(blockIdx.x) * 8 + int(threadIdx.x >> 5);
    int length;
    const int s = row_span(p, a.row_sequence, a.row_length, r, length);
    const int pages = (length + p.page_size - 1) / p.page_size, D = p.head_dim;
    if (j >= pages)
        return;
    float best = -INFINITY;
    if (j < a.sink_pages || j >= pages - a.recent_pages) {
        best = INFINITY;
    } else {
        const int page = checked_page(p, s, j);
        if (page >= 0) {
            const int64_t at = int64_t(page) * p.kv_heads + head;
            const int8_t *b = p.bounds + at * 2 * D;
            for (int g = 0; g < p.group; g++) {
                const R *q = static_cast<const R *>(a.q) + r * a.q_stride +
                             int64_t(head * p.group + g) * D;
                float top = 0.0f;
                for (int d = lane; d < D; d += 32)
                    top = fmaxf(top, fabsf(finite_key(to_float(q[d]))));
                const float u = unit_of(warp_max(top)), inv = u > 0.0f ? 1.0f / u : 0.0f;
                int sum = 0;
                for (int d = lane; d < D; d += 32) {
                    const int x = int(rintf(finite_key(to_float(q[d])) * inv));
                    sum += max(x * b[d], x * b[D + d]);
                }
                sum = __reduce_add_sync(0xffffffffu, sum);
                best = fmaxf(best, float(sum) * u);
            }
            best *= p.bound_scales[at];
        }
    }
    if (lane == 0)
        a.scores[(int64_t(r) * p.kv_heads + head) * p.max_pages + j] = best;
}

__global__ void __launch_bounds__(kChooseThreads)
    choose_pages_kernel(const __grid_constant__ PagedSelect a) {
    __shared__ ChooseScratch scratch;
    const PagedPool &p = a.p;
    const int head = blockIdx.x, r = blockIdx.y;
    int length;
    row_span(p, a.row_sequence, a.row_length, r, length);
    const int pages = (length + p.page_size - 1) / p.page_size;
    const int64_t at = int64_t(r) * p.kv_heads + head;
    const float *score = a.scores + at * p.max_pages;
    int32_t *out = a.selected + at * a.n_selected;
    uint32_t threshold;
    int quota;
    choose_largest([=](int i) { return ordered_bits(score[i]); }, pages, a.n_selected, scratch,
                   threshold, quota);
    int ties = 0, n = 0;
    for (int i0 = 0; i0 < pages; i0 += blockDim.x) {
        const int i = i0 + threadIdx.x;
        const uint32_t k = i < pages ? ordered_bits(score[i]) : 0u;
        const bool tie = i < pages && k == threshold;
        int total;
        const int rank = ties + block_rank(tie, scratch.warp[0], total);
        ties += total;
        const bool chosen = i < pages && (k > threshold || (tie && rank < quota));
        const int to = n + block_rank(chosen, scratch.warp[1], total);
        n += total;
        if (chosen)
            out[to] = i;
    }
    for (int i = n + threadIdx.x; i < a.n_selected; i += blockDim.x)
        out[i] = -1;
}

} // namespace

cudaError_t paged_select(const PagedSelect &a, cudaStream_t s) {
    const PagedPool &p = a.p;
    const dim3 grid((p.max_pages + 7) / 8, p.kv_heads, a.rows);
    if (a.type == 0)
        score_kernel<float><<<grid, 256, 0, s>>>(a);
    else if (a.type == 1)
        score_kernel<__half><<<grid, 256, 0, s>>>(a);
    else
        score_kernel<__nv_bfloat16><<<grid, 256, 0, s>>>(a);
    choose_pages_kernel<<<dim3(p.kv_heads, a.rows), kChooseThreads, 0, s>>>(a);
    count_launches(2);
    return cudaGetLastError();
}

} // namespace nut
